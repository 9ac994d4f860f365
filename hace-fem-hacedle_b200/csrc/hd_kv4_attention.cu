// hd_kv4_attention.cu -- GQA attention over a paged 4-bit KV cache, decode
// and ragged prefill, with a sliding window and first tokens (sinks) that
// stay visible.
//
// The query at position i of its request sees position j when j <= i and
// (window == 0 or j > i - window or j < sinks); its output is
// sum_j softmax_j(scale q . k_j) v_j over those, and zeros when it sees
// none (no length, or only table entries that name no page).  One pass over
// the positions with the running maximum and sum of the softmax.
#include <cmath>

#include "hd_internal.cuh"
#include "hd_kv4.cuh"
#include "hd_kv4_args.cuh"

namespace {

// One CTA per query row and head, a warp per position.
template <int HD>
__global__ void __launch_bounds__(128) k_kv4_attention(Kv4Args A) {
    constexpr int E = HD / 32;
    pdl_wait();
    pdl_trigger();
    const int64_t row = blockIdx.x;
    const int head = blockIdx.y, kvh = head / (A.n_heads / A.n_kv);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int seq = (int)row, back = 1;
    if (A.row0) {
        if (row >= A.row0[A.seqs]) return;
        int lo = 0, hi = A.seqs;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (A.row0[mid] <= row) lo = mid;
            else hi = mid;
        }
        seq = lo;
        back = A.row0[seq + 1] - (int)row;
    }
    const int64_t cap = (int64_t)A.max_pages << A.shift;
    int64_t len = A.lens[seq];
    len = len < 0 ? 0 : len > cap ? cap : len;
    const int64_t i = len - back;
    const int64_t first = A.window && i + 1 > A.window ? i + 1 - A.window : 0;
    const float *q = A.q + row * A.q_ld + head * HD;
    float qv[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        qv[e] = q[32 * e + lane] * A.scale;
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int64_t j = warp; j <= i; j += 4) {
        if (j < first && j >= A.sinks) continue;
        const int64_t page = A.tables[(int64_t)seq * A.max_pages + (j >> A.shift)];
        if (page < 0 || page >= A.pages) continue;
        const int off = (int)(j & ((1 << A.shift) - 1)), p = off & 15;
        const uint8_t *tile = A.cache + (((page * A.n_kv + kvh) << A.shift) / 16 + off / 16) * kv4_tile_bytes(HD);
        auto value = [&](int v, int e) {
            const uint32_t b = tile[v * 8 * HD + p * (HD / 2) + 16 * e + (lane & 15)];
            const float d = __half2float(*(const __half *)(tile + (16 + v) * HD + 2 * (p * E + e)));
            return (float)((int)(lane < 16 ? b & 15u : b >> 4) - 8) * d;
        };
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) s = fmaf(qv[e], value(0, e), s);
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        const float mn = fmaxf(m, s), a = m == -INFINITY ? 0.f : expf(m - mn), pj = expf(s - mn);
        l = l * a + pj;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(pj, value(1, e), o[e] * a);
        m = mn;
    }
    __shared__ float sm[4][HD + 2];
#pragma unroll
    for (int e = 0; e < E; e++) sm[warp][32 * e + lane] = o[e];
    if (lane == 0) {
        sm[warp][HD] = m;
        sm[warp][HD + 1] = l;
    }
    __syncthreads();
    const float M = fmaxf(fmaxf(sm[0][HD], sm[1][HD]), fmaxf(sm[2][HD], sm[3][HD]));
    for (int d = threadIdx.x; d < HD; d += 128) {
        float O = 0.f, L = 0.f;
        for (int w = 0; w < 4; w++) {
            const float a = sm[w][HD] == -INFINITY ? 0.f : expf(sm[w][HD] - M);
            O = fmaf(sm[w][d], a, O);
            L = fmaf(sm[w][HD + 1], a, L);
        }
        A.out[(row * A.n_heads + head) * HD + d] = L == 0.f ? 0.f : O / L;
    }
}

int run(hd_ctx *ctx, const Kv4Args &A, int hd, const char *name) {
    cudaError_t e;
    const dim3 grid((unsigned)A.rows, A.n_heads);
    if (hd == 128) e = hd_launch(ctx, k_kv4_attention<128>, grid, dim3(128), 0, A);
    else if (hd == 64) e = hd_launch(ctx, k_kv4_attention<64>, grid, dim3(128), 0, A);
    else e = hd_launch(ctx, k_kv4_attention<32>, grid, dim3(128), 0, A);
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
    return HD_OK;
}

}  // namespace

int hd_kv4_attention_check(hd_ctx *ctx, const char *name, Kv4Args &A, int page_size, int hd) {
    if ((A.rows > 0 && (!A.q || !A.out)) || (A.seqs > 0 && (!A.tables || !A.lens)) || (A.pages > 0 && !A.cache))
        return hd_fail(ctx, HD_E_ARG, "%s: null argument", name);
    int rc = hd_kv4_check(ctx, name, A.cache, A.pages, page_size, A.n_kv, hd);
    if (rc) return rc;
    HD_REQUIRE(ctx, A.n_heads > 0 && A.n_heads % A.n_kv == 0 && A.n_heads / A.n_kv <= MAXREP4, HD_E_SHAPE,
               "%s: n_heads %d must be a multiple of n_kv %d, at most %d per kv head", name, A.n_heads, A.n_kv, MAXREP4);
    HD_REQUIRE(ctx, A.seqs >= 0 && A.rows >= 0 && A.rows < ((int64_t)1 << 31) && A.max_pages > 0 &&
                        (int64_t)A.max_pages * page_size < ((int64_t)1 << 31),
               HD_E_SHAPE, "%s: bad shape (requests %d, rows %lld, table width %d)", name, A.seqs, (long long)A.rows,
               A.max_pages);
    HD_REQUIRE(ctx, A.window >= 0 && A.sinks >= 0 && A.scale >= 0.f && std::isfinite(A.scale), HD_E_ARG,
               "%s: window %d, sinks %d and scale %g must not be negative", name, A.window, A.sinks, (double)A.scale);
    if (A.q_ld == 0) A.q_ld = (int64_t)A.n_heads * hd;
    HD_REQUIRE(ctx, A.q_ld >= (int64_t)A.n_heads * hd, HD_E_SHAPE, "%s: row stride %lld of q", name, (long long)A.q_ld);
    HD_REQUIRE(ctx, A.q_ld % 4 == 0 && (((uintptr_t)A.q | (uintptr_t)A.out) & 15) == 0, HD_E_ARG,
               "%s: rows must be 16-byte aligned", name);
    if (!ctx) return HD_E_ARG;
    if (A.scale == 0.f) A.scale = 1.0f / sqrtf((float)hd);
    A.shift = 4;
    while ((1 << A.shift) < page_size) A.shift++;
    return HD_OK;
}

extern "C" int hd_kv4_attention_prefill(hd_ctx *ctx, const float *q, int64_t q_ld, const uint8_t *cache, int64_t pages,
                                        int page_size, const int32_t *tables, int max_pages, const int32_t *lens,
                                        const int32_t *row0, int seqs, int64_t rows, int n_heads, int n_kv, int head_dim,
                                        int window, int sinks, float scale, float *out) {
    Kv4Args A{q, q_ld, cache, pages, 0, tables, max_pages, lens, row0, seqs, rows, n_heads, n_kv, window, sinks, scale, out};
    if (seqs > 0 && !row0) return hd_fail(ctx, HD_E_ARG, "hd_kv4_attention_prefill: null argument");
    int rc = hd_kv4_attention_check(ctx, "hd_kv4_attention_prefill", A, page_size, head_dim);
    if (rc || seqs == 0 || rows == 0) return rc;
    HdDevice on(ctx);
    return run(ctx, A, head_dim, "hd_kv4_attention_prefill");
}
