// hd_kv4.cu -- a paged KV cache held in 4 bits: rows quantized into their
// slots, and read back.  Layout and rounding: hd_kv4.cuh.
#include "hd_internal.cuh"
#include "hd_kv4.cuh"

namespace {

// Eight threads a group of 32 values, four values each, blockIdx.y choosing
// keys or values: the group's largest magnitude by three shuffles, the first
// value that has it by a vote, the nibbles of the upper half passed to the
// thread that holds the lower half, and 16 bytes written by four threads.
// Bound by the rows read (4 bytes a value against 0.56 written) once indices
// are 32 bits wide: with 64-bit divisions a row of 16383 x 4 x 128 keys and
// values took 38 us, as many as three times its bytes.
__global__ void __launch_bounds__(256) k_kv4_append(const float *__restrict__ k, const float *__restrict__ v, int64_t k_ld,
                                                    int64_t v_ld, const int32_t *__restrict__ slots, uint32_t rows,
                                                    uint32_t n_kv, int lhd, int shift, int64_t n_slots, uint8_t *cache) {
    pdl_wait();
    pdl_trigger();
    const int hd = 1 << lhd, per_head = lhd - 2;                  // log2 of a head's threads
    const uint32_t i = blockIdx.x * 256u + threadIdx.x, hr = i >> per_head, r = hr / n_kv, h = hr - r * n_kv;
    if (r >= rows) return;                                        // whole groups of 8 threads
    const bool is_v = blockIdx.y != 0;
    const int e = (int)(i & ((1u << per_head) - 1)), g8 = threadIdx.x & 7, group = e >> 3;
    const unsigned first = threadIdx.x & 24, mask = 0xffu << first;
    const int64_t slot = slots[r];
    if (slot < 0 || slot >= n_slots) return;                      // the same for the whole group
    const float4 x = *(const float4 *)((is_v ? v + r * v_ld : k + r * k_ld) + (h << lhd) + 4 * e);
    const float xs[4] = {x.x, x.y, x.z, x.w};
    uint32_t a[4], top = 0;                                       // magnitudes as integers: a NaN is above infinity
#pragma unroll
    for (int j = 0; j < 4; j++) {
        a[j] = __float_as_uint(xs[j]) & 0x7fffffffu;
        top = max(top, a[j]);
    }
    const uint32_t mine = top;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, __shfl_xor_sync(mask, top, o));
    const float xc = a[0] == top ? x.x : a[1] == top ? x.y : a[2] == top ? x.z : x.w;
    const int holder = __ffs(__ballot_sync(mask, mine == top) & mask) - 1;
    const __half dh = kv4_scale(__shfl_sync(mask, xc, holder));
    const float d = __half2float(dh), inv = __fdiv_rn(1.f, d);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= kv4_quant(xs[j], d, inv) << (8 * j);
    const uint32_t hi = __shfl_down_sync(mask, w, 4, 8);
    const int off = (int)(slot & ((1 << shift) - 1)), p = off & (KV4_TILE - 1);
    uint8_t *tile = cache + ((((slot >> shift) * n_kv + h) << shift) / KV4_TILE + off / KV4_TILE) * kv4_tile_bytes(hd);
    if (g8 < 4) *(uint32_t *)(tile + (is_v ? 8 * hd : 0) + p * (hd / 2) + 16 * group + 4 * g8) = w | (hi << 4);
    if (g8 == 4) *(__half *)(tile + 16 * hd + (is_v ? hd : 0) + 2 * (p * (hd / 32) + group)) = dh;
}

// Eight values a thread: four bytes of quants give the values 4t..4t+3 of
// both halves of a group.
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t *__restrict__ cache, const int32_t *__restrict__ slots,
                                                  uint32_t rows, uint32_t n_kv, int lhd, int shift, int64_t n_slots,
                                                  float *__restrict__ k, float *__restrict__ v) {
    pdl_wait();
    pdl_trigger();
    const int hd = 1 << lhd, per_head = lhd - 3;
    const uint32_t i = blockIdx.x * 256u + threadIdx.x, hr = i >> per_head, r = hr / n_kv, h = hr - r * n_kv;
    if (r >= rows) return;
    const bool is_v = blockIdx.y != 0;
    const int u = (int)(i & ((1u << per_head) - 1)), group = u / 4, t = u & 3;
    float *out = (is_v ? v : k) + (((int64_t)hr << lhd) + 32 * group + 4 * t);
    const int64_t slot = slots[r];
    float4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    if (slot >= 0 && slot < n_slots) {
        const int off = (int)(slot & ((1 << shift) - 1)), p = off & (KV4_TILE - 1);
        const uint8_t *tile = cache + ((((slot >> shift) * n_kv + h) << shift) / KV4_TILE + off / KV4_TILE) * kv4_tile_bytes(hd);
        const uint32_t w = *(const uint32_t *)(tile + (is_v ? 8 * hd : 0) + p * (hd / 2) + 16 * group + 4 * t);
        const float d = __half2float(*(const __half *)(tile + 16 * hd + (is_v ? hd : 0) + 2 * (p * (hd / 32) + group)));
        auto val = [&](int s) { return __fmul_rn((float)((int)((w >> s) & 15u) - 8), d); };
        lo = make_float4(val(0), val(8), val(16), val(24));
        hi = make_float4(val(4), val(12), val(20), val(28));
    }
    __stcs((float4 *)out, lo);
    __stcs((float4 *)(out + 16), hi);
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
    const int64_t threads = rows * (width / 4);
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_kv4_append, dim3((unsigned)((threads + 255) / 256), 2), dim3(256), 0, k, v, k_ld, v_ld,
                               slots, (uint32_t)rows, (uint32_t)n_kv, log2_of(head_dim), log2_of(page_size),
                               pages * page_size, cache));
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
                               (uint32_t)rows, (uint32_t)n_kv, log2_of(head_dim), log2_of(page_size), pages * page_size, k, v));
    return HD_OK;
}
