// hd_kv4.cuh -- the 4-bit KV cache: layout and the rule that quantizes a
// group of 32 values.
//
// One layer's cache is bytes [pages][n_kv][P / 16] of tiles, a tile 16
// positions of one kv head, 18 * head_dim bytes:
//   K quants [16][head_dim / 2] | V quants [16][head_dim / 2]
//   | K scales f16 [16][head_dim / 32] | V scales f16 [16][head_dim / 32]
// Byte j of a group of 32 values holds value j in its low and value j + 16 in
// its high nibble, GGUF's order.  4.5 bits a value; a tile is a multiple of
// 64 bytes and the tiles of a page and head are consecutive, so what a warp
// needs of 16 positions is one contiguous bulk copy.
//
// value = (nibble - 8) * d with d = f16(clamp(bf16(-x_max / 8), +-8160)),
// x_max the first value of largest magnitude (the largest value meets the
// nibble 0, as in GGUF's Q4_0).  d is rounded to bf16's 8 significant bits on
// purpose: |nibble - 8| is at most 3 bits times a power of two, so
// (nibble - 8) * d needs at most 11 significant bits, is a multiple of 2^-24
// and at most 65280 in magnitude: it is exact in f16, and the tensor cores
// multiply the cache's own values.  The rounding moves a value by at most
// 2^-9 of itself, against the 4-bit grid's 2^-4.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

namespace {

constexpr int KV4_TILE = 16;   // positions per tile
__host__ __device__ constexpr int kv4_tile_bytes(int hd) { return 18 * hd; }

inline bool kv4_page_ok(int page) { return page >= 16 && page <= 1024 && (page & (page - 1)) == 0; }

// The scale of a group whose first value of largest magnitude is x.
__device__ __forceinline__ __half kv4_scale(float x) {
    const float d = __bfloat162float(__float2bfloat16_rn(__fmul_rn(x, -0.125f)));
    if (d != d) return __float2half_rn(d);
    return __float2half_rn(fminf(fmaxf(d, -8160.f), 8160.f));
}

// clamp(rint(x / d), -8, 7) + 8 as the division in 64 bits gives it, without
// one: n = rint(x * (1/d)) is at most one off, n * d has at most 12
// significant bits, so r = x - n d is exact where n counts (|x| <= 9 |d|),
// and the exact comparison of |r| with |d| / 2 settles the step and the tie.
__device__ __forceinline__ uint32_t kv4_quant(float x, float d, float inv) {
    if (!(d != 0.f) || d != d) return 8u;
    float n = rintf(fminf(fmaxf(__fmul_rn(x, inv), -9.f), 9.f));
    const float r = __fmaf_rn(-n, d, x), h = __fmul_rn(0.5f, fabsf(d));
    const float step = (r < 0.f) == (d < 0.f) ? 1.f : -1.f;
    if (fabsf(r) > h || (fabsf(r) == h && ((int)n & 1))) n += step;
    return (uint32_t)((int)fminf(fmaxf(n, -8.f), 7.f) + 8);
}

}  // namespace
