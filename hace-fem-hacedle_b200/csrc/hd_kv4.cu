// hd_kv4.cu -- a paged KV cache held in 4 bits: rows quantized into their
// slots, and read back.  Layout and rounding: hd_kv4.cuh.
#include "hd_internal.cuh"
#include "hd_kv4.cuh"

namespace {

// Eight threads a group of 32 values, four values each: the group's scale
// comes from its first value of largest magnitude (three shuffles over a key
// of magnitude and index), the nibbles of the upper half go to the thread
// that holds the lower half, and four threads write 16 bytes.
__global__ void __launch_bounds__(256) k_kv4_append(const float *__restrict__ k, const float *__restrict__ v, int64_t k_ld,
                                                    int64_t v_ld, const int32_t *__restrict__ slots, int64_t rows,
                                                    int n_kv, int hd, int shift, int64_t n_slots, uint8_t *cache) {
    pdl_wait();
    pdl_trigger();
    const int per_head = hd / 4, per_row = n_kv * per_head;       // threads of a row's keys
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= 2 * rows * per_row) return;                          // whole groups of 8 threads
    const int64_t kr = i / per_row;
    const int e = (int)(i - kr * per_row);
    const bool is_v = kr >= rows;
    const int64_t r = is_v ? kr - rows : kr;
    const unsigned mask = 0xffu << (threadIdx.x & 24);
    const int64_t slot = slots[r];
    if (slot < 0 || slot >= n_slots) return;                      // the same for the whole group
    const float4 x = *(const float4 *)((is_v ? v + r * v_ld : k + r * k_ld) + 4 * e);
    const int g8 = threadIdx.x & 7;
    const uint32_t a[4] = {__float_as_uint(x.x) & 0x7fffffffu, __float_as_uint(x.y) & 0x7fffffffu,
                           __float_as_uint(x.z) & 0x7fffffffu, __float_as_uint(x.w) & 0x7fffffffu};
    const float xs[4] = {x.x, x.y, x.z, x.w};
    int c = 0;
#pragma unroll
    for (int j = 1; j < 4; j++)
        if (a[j] > a[c]) c = j;
    const float xc = c == 0 ? x.x : c == 1 ? x.y : c == 2 ? x.z : x.w;
    const uint32_t ac = __float_as_uint(xc) & 0x7fffffffu;
    // magnitude (a NaN is above infinity), then the lowest index, with the value's sign behind them
    uint64_t key = ((uint64_t)ac << 32) | ((uint32_t)(31 - (4 * g8 + c)) << 1) | (__float_as_uint(xc) >> 31);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        const uint64_t other = __shfl_xor_sync(mask, key, o);
        key = other > key ? other : key;
    }
    const float top = __uint_as_float((uint32_t)(key >> 32) | ((uint32_t)key << 31));
    const __half dh = kv4_scale(top);
    const float d = __half2float(dh), inv = __fdiv_rn(1.f, d);
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= kv4_quant(xs[j], d, inv) << (8 * j);
    const uint32_t hi = __shfl_down_sync(mask, w, 4, 8);
    const int h = e / per_head, group = (e - h * per_head) / 8;
    const int64_t page = slot >> shift;
    const int off = (int)(slot & ((1 << shift) - 1)), p = off & (KV4_TILE - 1);
    uint8_t *tile = cache + (((page * n_kv + h) << shift) / KV4_TILE + off / KV4_TILE) * kv4_tile_bytes(hd);
    if (g8 < 4) *(uint32_t *)(tile + (is_v ? 8 * hd : 0) + p * (hd / 2) + 16 * group + 4 * g8) = w | (hi << 4);
    if (g8 == 4) *(__half *)(tile + 16 * hd + (is_v ? hd : 0) + 2 * (p * (hd / 32) + group)) = dh;
}

// Eight values a thread: four bytes of quants give the values 4t..4t+3 of
// both halves of a group.
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t *__restrict__ cache, const int32_t *__restrict__ slots,
                                                  int64_t rows, int n_kv, int hd, int shift, int64_t n_slots,
                                                  float *__restrict__ k, float *__restrict__ v) {
    pdl_wait();
    pdl_trigger();
    const int per_head = hd / 8, per_row = n_kv * per_head;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= 2 * rows * per_row) return;
    const int64_t kr = i / per_row;
    const int e = (int)(i - kr * per_row);
    const bool is_v = kr >= rows;
    const int64_t r = is_v ? kr - rows : kr;
    const int h = e / per_head, u = e - h * per_head, group = u / 4, t = u & 3;
    float *out = (is_v ? v : k) + (r * n_kv + h) * hd + 32 * group + 4 * t;
    const int64_t slot = slots[r];
    float4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
    if (slot >= 0 && slot < n_slots) {
        const int64_t page = slot >> shift;
        const int off = (int)(slot & ((1 << shift) - 1)), p = off & (KV4_TILE - 1);
        const uint8_t *tile = cache + (((page * n_kv + h) << shift) / KV4_TILE + off / KV4_TILE) * kv4_tile_bytes(hd);
        const uint32_t w = *(const uint32_t *)(tile + (is_v ? 8 * hd : 0) + p * (hd / 2) + 16 * group + 4 * t);
        const float d = __half2float(*(const __half *)(tile + 16 * hd + (is_v ? hd : 0) + 2 * (p * (hd / 32) + group)));
        auto val = [&](int s) { return __fmul_rn((float)((int)((w >> s) & 15u) - 8), d); };
        lo = make_float4(val(0), val(8), val(16), val(24));
        hi = make_float4(val(4), val(12), val(20), val(28));
    }
    *(float4 *)out = lo;
    *(float4 *)(out + 16) = hi;
}

int shift_of(int page) {
    int s = 0;
    while ((1 << s) < page) s++;
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
    HD_REQUIRE(ctx, rows >= 0 && k_ld >= width && v_ld >= width && rows < ((int64_t)1 << 39) / width, HD_E_SHAPE,
               "hd_kv4_append: bad shape (rows %lld, row strides %lld and %lld for %lld values)", (long long)rows,
               (long long)k_ld, (long long)v_ld, (long long)width);
    HD_REQUIRE(ctx, k_ld % 4 == 0 && v_ld % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, HD_E_ARG,
               "hd_kv4_append: rows must be 16-byte aligned");
    if (!ctx) return HD_E_ARG;
    if (rows == 0 || pages == 0) return HD_OK;
    HdDevice on(ctx);
    const int64_t threads = 2 * rows * (width / 4);
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_kv4_append, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, k, v, k_ld, v_ld,
                               slots, rows, n_kv, head_dim, shift_of(page_size), pages * page_size, cache));
    return HD_OK;
}

extern "C" int hd_kv4_read(hd_ctx *ctx, const uint8_t *cache, int64_t pages, int page_size, const int32_t *slots,
                           int64_t rows, int n_kv, int head_dim, float *k, float *v) {
    if ((rows > 0 && (!k || !v || !slots)) || (pages > 0 && !cache))
        return hd_fail(ctx, HD_E_ARG, "hd_kv4_read: null argument");
    int rc = hd_kv4_check(ctx, "hd_kv4_read", cache, pages, page_size, n_kv, head_dim);
    if (rc) return rc;
    const int64_t width = (int64_t)n_kv * head_dim;
    HD_REQUIRE(ctx, rows >= 0 && rows < ((int64_t)1 << 39) / width, HD_E_SHAPE, "hd_kv4_read: bad shape (rows %lld)",
               (long long)rows);
    HD_REQUIRE(ctx, (((uintptr_t)k | (uintptr_t)v) & 15) == 0, HD_E_ARG, "hd_kv4_read: rows must be 16-byte aligned");
    if (!ctx) return HD_E_ARG;
    if (rows == 0) return HD_OK;
    HdDevice on(ctx);
    const int64_t threads = 2 * rows * (width / 8);
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_kv4_read, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, cache, slots, rows,
                               n_kv, head_dim, shift_of(page_size), pages * page_size, k, v));
    return HD_OK;
}
