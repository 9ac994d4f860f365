// hd_kv4.cu -- a paged KV cache held in 4 bits: rows quantized into their
// slots, and read back.  Layout and rounding: hd_kv4.cuh.
#include "hd_internal.cuh"
#include "hd_kv4.cuh"

namespace {

// hr / n_kv, by a multiplication where that is exact (recip = 2^32 / n_kv rounded up; 0: not).
__device__ __forceinline__ uint32_t row_of(uint32_t hr, uint32_t n_kv, uint32_t recip) {
    return recip ? __umulhi(hr, recip) : hr / n_kv;
}

// Four nibbles by the exact rule (a call, so that it costs only those that take it).
__device__ __noinline__ uint32_t quant4_exact(float a, float b, float c, float e, float d, float inv) {
    return kv4_quant(a, d, inv) | kv4_quant(b, d, inv) << 8 | kv4_quant(c, d, inv) << 16 | kv4_quant(e, d, inv) << 24;
}

// Four threads a group of 32 values, eight values each, blockIdx.y choosing
// keys or values: the group's largest magnitude by two shuffles, the first
// value that has it by a vote, the nibbles of the upper half passed to the
// threads that hold the lower half, and 16 bytes written by two threads.
//
// 16383 rows of 2 x 4 x 128 values take 22 us a call among others of its kind,
// 25 with cold caches (76 MB; 11.7 us at the measured copy rate): instruction
// issue, 72% of its slots busy, bounds it before the rows read do (4 bytes a
// value against 0.56 written).  The first form (four
// values a thread, 64-bit indices, the exact rounding of every value) took 337
// instructions a thread and 53 us; here the exact comparison is left to values
// within 10^-5 of a tie.
__global__ void __launch_bounds__(256) k_kv4_append(const float *__restrict__ k, const float *__restrict__ v, int64_t k_ld,
                                                    int64_t v_ld, const int32_t *__restrict__ slots, uint32_t rows,
                                                    uint32_t n_kv, uint32_t recip, int lhd, int shift, int64_t n_slots,
                                                    uint8_t *cache) {
    pdl_wait();
    pdl_trigger();
    const int hd = 1 << lhd, per_head = lhd - 3;                  // log2 of a head's threads
    const uint32_t i = blockIdx.x * 256u + threadIdx.x, hr = i >> per_head, r = row_of(hr, n_kv, recip), h = hr - r * n_kv;
    const bool is_v = blockIdx.y != 0;
    const int e = (int)(i & ((1u << per_head) - 1)), g4 = threadIdx.x & 3, group = e >> 2;
    const int64_t slot = r < rows ? slots[r] : -1;
    const bool on = slot >= 0 && slot < n_slots;                  // the same for the whole group
    float4 x0 = {0.f, 0.f, 0.f, 0.f}, x1 = x0;
    if (on) {
        const float4 *src = (const float4 *)((is_v ? v + r * v_ld : k + r * k_ld) + (h << lhd) + 8 * e);
        x0 = __ldcs(src);
        x1 = __ldcs(src + 1);
    }
    // (every lane takes part in the shuffles: with a mask per group the warp ran them group by group, 400
    // instructions a thread instead of 150)
    constexpr unsigned ALL = 0xffffffffu;
    const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
    uint32_t top = 0;                                             // magnitudes as integers: a NaN is above infinity
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
    const uint32_t mine = top;
    top = max(top, __shfl_xor_sync(ALL, top, 1));
    top = max(top, __shfl_xor_sync(ALL, top, 2));
    float xc = x[7];
#pragma unroll
    for (int j = 6; j >= 0; j--) xc = (__float_as_uint(x[j]) & 0x7fffffffu) == top ? x[j] : xc;
    const int holder = __ffs(__ballot_sync(ALL, mine == top) & (0xfu << (threadIdx.x & 28))) - 1;
    const __half dh = kv4_scale(__shfl_sync(ALL, xc, holder));
    const float d = __half2float(dh);
    const bool none = !(fabsf(d) > 0.f);                          // 0 or NaN: every nibble 8
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(d));
    uint32_t n[8];
    float far = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        // x / d to within 10^-5, rounded by an addition whose last bit is 1: the low byte is the nibble
        const float t = fminf(fmaxf(x[j] * inv, -8.f), 7.f), m = t + 12582920.f;
        n[j] = __float_as_uint(m);
        far = fmaxf(far, fabsf(t - (m - 12582920.f)));
    }
    uint32_t w0 = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    uint32_t w1 = __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410);
    if (far > 0.49999f) {                                         // near a tie: exactly
        w0 = quant4_exact(x[0], x[1], x[2], x[3], d, inv);
        w1 = quant4_exact(x[4], x[5], x[6], x[7], d, inv);
    }
    if (none) w0 = w1 = 0x08080808u;
    const uint32_t h0 = __shfl_down_sync(ALL, w0, 2, 4), h1 = __shfl_down_sync(ALL, w1, 2, 4);
    if (!on) return;
    const int off = (int)(slot & ((1 << shift) - 1)), p = off & (KV4_TILE - 1);
    uint8_t *tile = cache + ((((slot >> shift) * n_kv + h) << shift) / KV4_TILE + off / KV4_TILE) * kv4_tile_bytes(hd);
    if (g4 < 2) *(uint2 *)(tile + (is_v ? 8 * hd : 0) + p * (hd / 2) + 16 * group + 8 * g4) = make_uint2(w0 | (h0 << 4), w1 | (h1 << 4));
    if (g4 == 2) *(__half *)(tile + 16 * hd + (is_v ? hd : 0) + 2 * (p * (hd / 32) + group)) = dh;
}

// Eight values a thread: four bytes of quants give the values 4t..4t+3 of
// both halves of a group, and four threads write 64 bytes in a row (16 values
// a thread, 32 bytes in a row: 23 us against 17 for 16383 x 2 x 4 x 128).
// Bound by the rows written.
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t *__restrict__ cache, const int32_t *__restrict__ slots,
                                                  uint32_t rows, uint32_t n_kv, uint32_t recip, int lhd, int shift,
                                                  int64_t n_slots, float *__restrict__ k, float *__restrict__ v) {
    pdl_wait();
    pdl_trigger();
    const int hd = 1 << lhd, per_head = lhd - 3;
    const uint32_t i = blockIdx.x * 256u + threadIdx.x, hr = i >> per_head, r = row_of(hr, n_kv, recip), h = hr - r * n_kv;
    if (r >= rows) return;
    const bool is_v = blockIdx.y != 0;
    const int u = (int)(i & ((1u << per_head) - 1)), group = u / 4, t = u & 3;
    float *out = (is_v ? v : k) + (((int64_t)hr << lhd) + 32 * group + 4 * t);
    const int64_t slot = slots[r];
    uint32_t w = 0x88888888u;
    float d = 0.f;
    if (slot >= 0 && slot < n_slots) {
        const int off = (int)(slot & ((1 << shift) - 1)), p = off & (KV4_TILE - 1);
        const uint8_t *tile = cache + ((((slot >> shift) * n_kv + h) << shift) / KV4_TILE + off / KV4_TILE) * kv4_tile_bytes(hd);
        w = *(const uint32_t *)(tile + (is_v ? 8 * hd : 0) + p * (hd / 2) + 16 * group + 4 * t);
        d = __half2float(*(const __half *)(tile + 16 * hd + (is_v ? hd : 0) + 2 * (p * (hd / 32) + group)));
    }
    // a nibble under the exponent of 2^23 is 2^23 + n; less 2^23 + 8, times d: exact
    auto val = [&](uint32_t b, int c) { return __fmul_rn(__uint_as_float(__byte_perm(b, 0x4B000000u, 0x7440 + c)) - 8388616.f, d); };
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    __stcs((float4 *)out, make_float4(val(lo, 0), val(lo, 1), val(lo, 2), val(lo, 3)));
    __stcs((float4 *)(out + 16), make_float4(val(hi, 0), val(hi, 1), val(hi, 2), val(hi, 3)));
}

// What row_of takes: hr < 2^32 / n_kv makes the multiplication exact.
uint32_t recip_of(int64_t rows, int64_t n_kv) {
    return n_kv > 1 && rows < (((int64_t)1 << 32) / n_kv) / n_kv - 256 ? (uint32_t)(((uint64_t)1 << 32) / (uint64_t)n_kv + 1) : 0u;
}

int log2_of(int v) {
    int s = 0;
    while ((1 << s) < v) s++;
    return s;
}

}  // namespace

int hd_kv4_check(hd_ctx *ctx, const char *name, const void *cache, int64_t pages, int page_size, int n_kv, int head_dim) {
    HD_REQUIRE(ctx, pages >= 0 && n_kv > 0 && kv4_page_ok(page_size), HD_E_SHAPE,
               "%s: bad shape (pages %lld, n_kv %d, page size %d: a power of two, 16 to 1024)", name, (long long)pages, n_kv,
               page_size);
    HD_REQUIRE(ctx, head_dim == 32 || head_dim == 64 || head_dim == 128, HD_E_UNSUPPORTED,
               "%s: head_dim %d (32, 64 or 128)", name, head_dim);
    HD_REQUIRE(ctx, pages < ((int64_t)1 << 31) / page_size, HD_E_SHAPE, "%s: %lld pages of %d: 2^31 slots or more", name,
               (long long)pages, page_size);
    HD_REQUIRE(ctx, (int64_t)n_kv * head_dim < ((int64_t)1 << 31), HD_E_SHAPE, "%s: %d kv heads of %d", name, n_kv, head_dim);
    HD_REQUIRE(ctx, ((uintptr_t)cache & 15) == 0, HD_E_ARG, "%s: the cache must be 16-byte aligned", name);
    return HD_OK;
}

extern "C" uint64_t hd_kv4_cache_bytes(int64_t pages, int page_size, int n_kv, int head_dim) {
    if (pages < 0 || n_kv <= 0 || !kv4_page_ok(page_size) || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
    return (uint64_t)pages * n_kv * (page_size / KV4_TILE) * kv4_tile_bytes(head_dim);
}

extern "C" int hd_kv4_append(hd_ctx *ctx, const float *k, const float *v, int64_t k_ld, int64_t v_ld,
                             const int32_t *slots, int64_t rows, int n_kv, int head_dim, uint8_t *cache, int64_t pages,
                             int page_size) {
    if ((rows > 0 && (!k || !v || !slots)) || (pages > 0 && !cache))
        return hd_fail(ctx, HD_E_ARG, "hd_kv4_append: null argument");
    int rc = hd_kv4_check(ctx, "hd_kv4_append", cache, pages, page_size, n_kv, head_dim);
    if (rc) return rc;
    const int64_t width = (int64_t)n_kv * head_dim;
    if (k_ld == 0) k_ld = width;
    if (v_ld == 0) v_ld = width;
    HD_REQUIRE(ctx, rows >= 0 && k_ld >= width && v_ld >= width && rows < ((int64_t)1 << 33) / width, HD_E_SHAPE,
               "hd_kv4_append: bad shape (rows %lld, row strides %lld and %lld for %lld values; fewer than 2^33 in all)",
               (long long)rows, (long long)k_ld, (long long)v_ld, (long long)width);
    HD_REQUIRE(ctx, k_ld % 4 == 0 && v_ld % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, HD_E_ARG,
               "hd_kv4_append: rows must be 16-byte aligned");
    if (!ctx) return HD_E_ARG;
    if (rows == 0 || pages == 0) return HD_OK;
    HdDevice on(ctx);
    const int64_t threads = rows * (width / 8);
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_kv4_append, dim3((unsigned)((threads + 255) / 256), 2), dim3(256), 0, k, v, k_ld, v_ld,
                               slots, (uint32_t)rows, (uint32_t)n_kv, recip_of(rows, n_kv), log2_of(head_dim),
                               log2_of(page_size), pages * page_size, cache));
    return HD_OK;
}

extern "C" int hd_kv4_read(hd_ctx *ctx, const uint8_t *cache, int64_t pages, int page_size, const int32_t *slots,
                           int64_t rows, int n_kv, int head_dim, float *k, float *v) {
    if ((rows > 0 && (!k || !v || !slots)) || (pages > 0 && !cache))
        return hd_fail(ctx, HD_E_ARG, "hd_kv4_read: null argument");
    int rc = hd_kv4_check(ctx, "hd_kv4_read", cache, pages, page_size, n_kv, head_dim);
    if (rc) return rc;
    const int64_t width = (int64_t)n_kv * head_dim;
    HD_REQUIRE(ctx, rows >= 0 && rows < ((int64_t)1 << 33) / width, HD_E_SHAPE,
               "hd_kv4_read: bad shape (rows %lld of %lld values: fewer than 2^33 in all)", (long long)rows, (long long)width);
    HD_REQUIRE(ctx, (((uintptr_t)k | (uintptr_t)v) & 15) == 0, HD_E_ARG, "hd_kv4_read: rows must be 16-byte aligned");
    if (!ctx) return HD_E_ARG;
    if (rows == 0) return HD_OK;
    HdDevice on(ctx);
    const int64_t threads = rows * (width / 8);
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_kv4_read, dim3((unsigned)((threads + 255) / 256), 2), dim3(256), 0, cache, slots,
                               (uint32_t)rows, (uint32_t)n_kv, recip_of(rows, n_kv), log2_of(head_dim), log2_of(page_size),
                               pages * page_size, k, v));
    return HD_OK;
}
