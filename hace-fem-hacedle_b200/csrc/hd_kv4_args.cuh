// hd_kv4_args.cuh -- what the attention kernels over the 4-bit cache are given.
#pragma once
#include <cstdint>

struct hd_ctx;

constexpr int MAXREP4 = 16;   // query heads per kv head

struct Kv4Args {
    const float *q;
    int64_t q_ld;
    const uint8_t *cache;
    int64_t pages;
    int shift;                    // log2 of the page size
    const int32_t *tables;
    int max_pages;
    const int32_t *lens, *row0;   // row0: prefill; null: row r is request r's last position
    int seqs;
    int64_t rows;
    int n_heads, n_kv, window, sinks;
    float scale;
    float *out;
    float scale_m;                // scale * log2(e) = scale_m * 2^scale_e, scale_m in [0.72, 1.45)
    int scale_e;
};

// Refuses what the kernels do not take, and fills in shift and the defaults of
// q_ld and scale (hd_kv4_attention.cu).
int hd_kv4_attention_check(hd_ctx *ctx, const char *name, Kv4Args &A, int page_size, int head_dim);
