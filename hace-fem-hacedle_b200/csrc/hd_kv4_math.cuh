// hd_kv4_math.cuh -- arithmetic that the attention kernels over the 4-bit
// cache share: nibbles to exact f16 values, f32 values in two f16 parts, and
// which tiles of a request a range of queries sees.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>

#include "hd_kv4.cuh"
#include "hd_kv4_args.cuh"

namespace {

constexpr uint32_t KV4_MAGIC = 0x64006400u;   // (1024, 1024) in f16

__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<const uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b),
                              *reinterpret_cast<const __half2 *>(&c));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// (nibble - 8) * d for two nibbles of a word 16 bits apart: bits 0-3 and
// 16-19, or bits 4-7 and 20-23.  A nibble under the exponent of 1024 is
// 1024 + n (or 1024 + 16 n); every step is exact.  `magic` is KV4_MAGIC from a
// register that the compiler cannot see through: as a constant, mask and magic
// are two immediates and take two instructions.
__device__ __forceinline__ uint32_t and_or(uint32_t w, uint32_t mask, uint32_t magic) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "r"(mask), "r"(magic));
    return r;
}
__device__ __forceinline__ uint32_t nib_lo(uint32_t w, uint32_t d2, uint32_t magic) {
    return h2_mul(h2_sub(and_or(w, 0x000F000Fu, magic), 0x64086408u), d2);                // 1024 + n - 1032
}
__device__ __forceinline__ uint32_t nib_hi(uint32_t w, uint32_t d2, uint32_t magic) {
    return h2_mul(h2_fma(and_or(w, 0x00F000F0u, magic), 0x2C002C00u, 0xD480D480u), d2);   // (1024 + 16 n) / 16 - 72
}

// (a, b) in two f16 parts: 22 significant bits.
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A row of q whose largest magnitude is mx is multiplied by `up` for its f16
// parts, which takes that to between 2^13 and 2^16 (at most 47500); kappa, a
// power of two, then takes its scores to base-2 exponents: the significant bits
// of scale * log2(e) are in `up`, so s * kappa is exact.  |s| < 2^39 (128
// products with cache values below 2^16), and kappa is held to 2^-120 .. 2^88,
// so s * kappa is finite and -infinity * kappa is -infinity; at those ends
// scores that differ at all are too far apart, or all too close, for kappa to
// matter.
__device__ __forceinline__ void q_scales(const Kv4Args &A, float mx, float &up, float &kappa) {
    int e = (int)(__float_as_uint(mx) >> 23) - 127;
    e = e < -100 ? -100 : e;                // the factor stays a normal number
    up = A.scale_m * __uint_as_float((uint32_t)(127 + 14 - e) << 23);
    const int k = A.scale_e + e - 14;
    kappa = __uint_as_float((uint32_t)(127 + (k < -120 ? -120 : k > 88 ? 88 : k)) << 23);
}
// Weights are 2^(s kappa - ref) with ref = m kappa - 15 rounded up, m the
// largest score so far: the largest weight lies at 2^15 for its f16 parts, and
// never above it, whatever the size of the scores.  (Rounded to nearest, from
// |m kappa| = 2^24 on it came to 2^16, infinite in f16.)  Where a step of the
// scores is 2 or more, weights are whole powers of two and their largest is at
// least 1, so nothing is lost there either.
__device__ __forceinline__ float weight_ref(float m, float kappa) {
    return m == -INFINITY ? 0.f : __fmaf_ru(m, kappa, -15.f);
}

// The tiles that queries at positions i0 .. last of a request see: `sink`
// first ones, then those from `from` on, `units` in all.
struct Seen {
    int last, first;   // the last query's position, the first query's first one in the window
    int sink, from, units;
    __device__ __forceinline__ int tile(int u) const { return u < sink ? u : from + u - sink; }
    // whether any of the queries sees position p
    __device__ __forceinline__ bool any(int p, int sinks) const { return p <= last && (p >= first || p < sinks); }
};
__device__ __forceinline__ Seen seen_tiles(int window, int sinks, int i0, int last) {
    Seen s;
    s.last = last;
    s.first = window && i0 >= window ? i0 - window + 1 : 0;
    s.from = s.first / KV4_TILE;
    s.sink = min((min(sinks, s.first) + KV4_TILE - 1) / KV4_TILE, s.from);
    s.units = last < 0 ? 0 : s.sink + last / KV4_TILE - s.from + 1;
    return s;
}
// A request's length, within what its table can hold.
__device__ __forceinline__ int held_length(const Kv4Args &A, int len) {
    const int cap = A.max_pages << A.shift;
    return len < 0 ? 0 : len > cap ? cap : len;
}

}  // namespace
