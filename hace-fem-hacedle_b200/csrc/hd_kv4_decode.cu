// hd_kv4_decode.cu -- decode attention (one query per request) over the paged
// 4-bit cache.
//
// Mathematics.  A warp takes a tile of 16 positions of one kv head at a time
// and keeps the running maximum, sum and output of up to 8 query heads that
// share it.  Both products run on m16n8k16 MMAs: rows 0..7 of the A operand
// are the heads' high f16 parts and rows 8..15 their low parts, so one MMA
// multiplies both and adding accumulator rows g and g + 8 -- which the same
// thread holds -- gives 22 significant bits of q (scaled by a power of two per
// head) and of the softmax weights (scaled by 2^15), against cache values that
// are exact in f16 (hd_kv4.cuh).  The score accumulators are already in the
// layout the second product wants its A operand in.
//
// Operand layout.  The contraction's order is free, so each thread takes the
// bytes of a key that lie together (HD / 8 of them) and q is laid out to
// match; a value pair of the second product is two positions of one
// dimension, one byte permute away from the stored rows.  Nothing is
// transposed and nothing but raw tiles passes through shared memory: each warp
// has its own ring of tiles filled by cp.async, rows placed so that both
// products read without bank conflicts.
//
// Split.  A request's visible tiles (sinks and window) times its kv heads are
// units in one line over all requests; every CTA scans the lengths, takes an
// equal run of units, and so ragged lengths balance whatever they are, with
// nothing planned on the host.  A run that covers a head's units alone writes
// the output; pieces go to the workspace and the CTA that arrives last joins
// them in order, so results do not depend on the schedule.
#include <cmath>

#include "hd_internal.cuh"
#include "hd_kv4.cuh"
#include "hd_kv4_args.cuh"
#include "hd_mma.cuh"

namespace {

constexpr int DW = 4;           // warps per CTA
constexpr int DNT = 32 * DW;
constexpr int DSTAGES = 5;      // tiles in a warp's ring
constexpr int DMIN = 2 * DW;    // fewest tiles a CTA takes
constexpr int DHEADS = 8;       // query heads per unit

template <int HD>
constexpr int d_occ() { return HD == 128 ? 3 : 4; }   // CTAs per SM

template <int HD>
struct DShared {
    alignas(16) uint8_t ring[DW][DSTAGES][kv4_tile_bytes(HD)];
    float o[DW][DHEADS][HD + 4];
    float m[DW][DHEADS], l[DW][DHEADS];
    int64_t part[DW];
    int64_t start_off;
    int start_req, last;
};

// Where row p of a tile's quants lies in the ring: a permutation of the rows
// (and of a row's 16-byte pieces at HD 128) under which a quarter warp's keys
// (rows k and k + 4) and the rows t, t + 4 of the second product fall into
// different banks.
template <int HD>
__device__ __forceinline__ int d_slot(int p) {
    return HD == 128 ? p ^ ((p >> 2) & 1) : HD == 64 ? p ^ ((p >> 1) & 2) : p;
}
template <int HD>
__device__ __forceinline__ int d_piece(int slot, int c) { return HD == 128 ? c ^ (slot & 2) : c; }

// (nibble - 8) * d for the pairs of a word: nibbles 0 and 4, 2 and 6 (odd
// bytes), and 1 and 5, 3 and 7 (the bytes' high halves); exact.
__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t b) {
    __half2 r = __hmul2(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&b));
    return *reinterpret_cast<uint32_t *>(&r);
}
__device__ __forceinline__ uint32_t nib_lo(uint32_t w, uint32_t d2) {
    return hmul2u(hsub2u((w & 0x000F000Fu) | H_MAGIC, 0x64086408u), d2);             // 1024 + n - 1032
}
__device__ __forceinline__ uint32_t nib_hi(uint32_t w, uint32_t d2) {
    return hmul2u(hfma2u((w & 0x00F000F0u) | H_MAGIC, H_SIXTEENTH, 0xD480D480u), d2);  // (1024 + 16 n) / 16 - 72
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
}
// (a, b) in two f16 parts.
__device__ __forceinline__ void split2(float a, float b, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = pack2(a - f.x, b - f.y);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The tiles a request's last position sees: `sink` first ones, then those from
// `from` on, `units` in all.
struct Seen {
    int last, first;   // the query's position, the window's first one
    int sink, from, units;
};
__device__ __forceinline__ Seen seen_tiles(const Kv4Args &A, int len) {
    Seen s;
    const int cap = A.max_pages << A.shift;
    len = len < 0 ? 0 : len > cap ? cap : len;
    s.last = len - 1;
    s.first = A.window && len > A.window ? len - A.window : 0;
    s.from = s.first / KV4_TILE;
    const int sinks = min(A.sinks, s.first);
    s.sink = min((sinks + KV4_TILE - 1) / KV4_TILE, s.from);
    s.units = len == 0 ? 0 : s.sink + s.last / KV4_TILE - s.from + 1;
    return s;
}

template <int HD>
__global__ void __launch_bounds__(DNT, d_occ<HD>()) k_kv4_decode(Kv4Args A, int groups, int gh, int *tickets, float *parts) {
    constexpr int WPT = HD / 32;       // words of a key per thread
    constexpr int NT = HD / 8;         // column tiles of the output
    constexpr int W = HD + 2;          // floats of a partial per head
    extern __shared__ __align__(16) uint8_t smem_raw[];
    DShared<HD> &sm = *reinterpret_cast<DShared<HD> *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();
    const int items = A.n_kv * groups, rep = A.n_heads / A.n_kv;

    // ---- this CTA's run of units
    const int per_thread = (A.seqs + DNT - 1) / DNT, rb = min(A.seqs, tid * per_thread), re = min(A.seqs, rb + per_thread);
    int64_t mine = 0;
    for (int r = rb; r < re; r++) mine += seen_tiles(A, A.lens[r]).units;
    int64_t inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) sm.part[warp] = inc;
    __syncthreads();
    int64_t before = inc - mine, total = 0;
#pragma unroll
    for (int w = 0; w < DW; w++) {
        if (w < warp) before += sm.part[w];
        total += sm.part[w];
    }
    total *= items;
    before *= items;
    int64_t per = (total + gridDim.x - 1) / gridDim.x;
    per = per < DMIN ? DMIN : per;
    const int64_t c_begin = per * blockIdx.x, c_end = min(total, c_begin + per);
    // requests without any position
    for (int r = blockIdx.x; r < A.seqs; r += gridDim.x)
        if (seen_tiles(A, A.lens[r]).units == 0)
            for (int i = tid; i < A.n_heads * HD; i += DNT) A.out[(int64_t)r * A.n_heads * HD + i] = 0.f;
    if (c_begin >= c_end) return;
    if (before <= c_begin && c_begin < before + mine * items) {
        int r = rb;
        for (;; r++) {
            const int64_t u = (int64_t)seen_tiles(A, A.lens[r]).units * items;
            if (c_begin < before + u) break;
            before += u;
        }
        sm.start_req = r;
        sm.start_off = c_begin - before;
    }
    __syncthreads();
    int req = sm.start_req;
    int64_t off = sm.start_off;

    for (int64_t at = c_begin; at < c_end;) {
        const Seen S = seen_tiles(A, A.lens[req]);
        if (off >= (int64_t)S.units * items) {
            off -= (int64_t)S.units * items;
            req++;
            continue;
        }
        const int item = (int)(off / S.units), u0 = (int)(off - (int64_t)item * S.units);
        const int u1 = (int)min((int64_t)S.units, u0 + (c_end - at));
        const int kvh = item / groups, h0 = (item - kvh * groups) * gh, nh = min(gh, rep - h0);
        const int32_t *table = A.tables + (int64_t)req * A.max_pages;

        // ---- tiles into the warp's ring
        auto tile_of = [&](int u) { return u < S.sink ? u : S.from + u - S.sink; };
        auto fetch = [&](int u, int stage) {
            const int tile = tile_of(u), pos = tile * KV4_TILE;
            const int64_t page = table[pos >> A.shift];
            const bool ok = page >= 0 && page < A.pages;
            if (ok) {
                const uint8_t *src = A.cache + ((((page * A.n_kv + kvh) << A.shift) + (pos & ((1 << A.shift) - 1))) / KV4_TILE) *
                                                   kv4_tile_bytes(HD);
                const uint32_t dst = smem_u32(sm.ring[warp][stage]);
                constexpr int PR = HD / 32, N = kv4_tile_bytes(HD) / 16;
#pragma unroll
                for (int i0 = 0; i0 < N; i0 += 32) {
                    const int i = i0 + lane;
                    if (i < N) {
                        int to = i;
                        if (i < 2 * 16 * PR) {           // quants: K rows 0..15, then V rows 0..15
                            const int row = i / PR, slot = d_slot<HD>(row);
                            to = slot * PR + d_piece<HD>(slot, i % PR);
                        }
                        cp16(dst + 16 * to, src + 16 * i);
                    }
                }
            }
            return ok;
        };

        // ---- q of the heads, in two f16 parts scaled to 2^14
        uint32_t qa[WPT][2][4];
        float kappa;                    // scores to base-2 exponents
        {
            float x[WPT][8];
            const float *q = A.q + (int64_t)req * A.q_ld + (int64_t)(kvh * rep + h0 + g) * HD;
            float mx = 0.f;
#pragma unroll
            for (int w = 0; w < WPT; w++) {
                const int b = t * (HD / 8) + 4 * w, d = b / 16 * 32 + b % 16;
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (g < nh) v = *(const float4 *)(q + d + 16 * hf);
                    x[w][4 * hf] = v.x;
                    x[w][4 * hf + 1] = v.y;
                    x[w][4 * hf + 2] = v.z;
                    x[w][4 * hf + 3] = v.w;
                    mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                }
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // 2^(14 - exponent of mx), a normal number as its inverse is
            int e = (int)(__float_as_uint(mx) >> 23) - 127;
            e = e < -100 ? -100 : e;
            const float up = __uint_as_float((uint32_t)(127 + 14 - e) << 23);
            kappa = A.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 - 14 + e) << 23);
#pragma unroll
            for (int w = 0; w < WPT; w++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float *v = x[w] + 4 * hf;
                    split2(v[0] * up, v[2] * up, qa[w][hf][0], qa[w][hf][1]);
                    split2(v[1] * up, v[3] * up, qa[w][hf][2], qa[w][hf][3]);
                }
        }
        float o[NT][4], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[i][c] = 0.f;

        uint32_t named = 0;             // bit s: the page of ring stage s exists
        const int n = u1 - u0 > warp ? (u1 - u0 - warp + DW - 1) / DW : 0;   // this warp's tiles
#pragma unroll
        for (int s = 0; s < DSTAGES - 1; s++) {
            if (s < n && fetch(u0 + warp + s * DW, s)) named |= 1u << s;
            cp_commit();
        }
        int stage = 0;
        for (int k = 0; k < n; k++) {
            {
                const int ahead = k + DSTAGES - 1, to = stage == 0 ? DSTAGES - 1 : stage - 1;
                __syncwarp();           // all lanes have read the stage that is refilled
                named &= ~(1u << to);
                if (ahead < n && fetch(u0 + warp + ahead * DW, to)) named |= 1u << to;
                cp_commit();
            }
            cp_wait<DSTAGES - 1>();
            __syncwarp();
            const int pos = tile_of(u0 + warp + k * DW) * KV4_TILE;
            const uint8_t *tile = sm.ring[warp][stage];
            const bool ok = named >> stage & 1;
            stage = stage == DSTAGES - 1 ? 0 : stage + 1;
            if (!ok) continue;
            const bool whole = pos + KV4_TILE - 1 <= S.last && (pos >= S.first || pos + KV4_TILE <= A.sinks);
            auto sees = [&](int p) { return pos + p <= S.last && (pos + p >= S.first || pos + p < A.sinks); };

            // ---- scores of positions t, t + 4 (first MMA) and t + 8, t + 12 (second)
            float s[2][4];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int p = 8 * j + (g >> 1) + 4 * (g & 1), slot = d_slot<HD>(p);
                uint32_t w[WPT];
                const uint8_t *row = tile + slot * (HD / 2);
                if constexpr (HD == 128) {
                    const uint4 v = *(const uint4 *)(row + 16 * d_piece<HD>(slot, t));
                    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                } else if constexpr (HD == 64) {
                    const uint2 v = *(const uint2 *)(row + 8 * t);
                    w[0] = v.x; w[1] = v.y;
                } else {
                    w[0] = *(const uint32_t *)(row + 4 * t);
                }
                uint32_t d = *(const uint16_t *)(tile + 16 * HD + 2 * (p * (HD / 32) + t * (HD / 8) / 16));
                if (!whole && !sees(p)) d = 0;
                d |= d << 16;
#pragma unroll
                for (int c = 0; c < 4; c++) s[j][c] = 0.f;
#pragma unroll
                for (int i = 0; i < WPT; i++) {
                    const uint32_t w8 = w[i] >> 8;
                    mma16816(s[j], qa[i][0][0], qa[i][0][1], qa[i][0][2], qa[i][0][3], nib_lo(w[i], d), nib_lo(w8, d), s[j]);
                    mma16816(s[j], qa[i][1][0], qa[i][1][1], qa[i][1][2], qa[i][1][3], nib_hi(w[i], d), nib_hi(w8, d), s[j]);
                }
            }
            float e[4] = {(s[0][0] + s[0][2]) * kappa, (s[0][1] + s[0][3]) * kappa, (s[1][0] + s[1][2]) * kappa,
                          (s[1][1] + s[1][3]) * kappa};
            if (!whole) {
#pragma unroll
                for (int c = 0; c < 4; c++)
                    if (!sees(t + 4 * c)) e[c] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m)) {
                const float mn = fmaxf(m, mx), a = m == -INFINITY ? 0.f : exp2_approx(m - mn);
                m = mn;
                l *= a;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[i][c] *= a;
            }
            const float ref = m == -INFINITY ? 0.f : m - 15.f;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                e[c] = exp2_approx(e[c] - ref);
                l += e[c];
            }
            uint32_t pa[4];
            split2(e[0], e[1], pa[0], pa[1]);
            split2(e[2], e[3], pa[2], pa[3]);

            // ---- output: value pairs (t, t + 4) and (t + 8, t + 12) of HD / 16 bytes of each row
            constexpr int NX = HD >= 64 ? HD / 32 : 1;    // half words of a row's bytes
            uint32_t x[2][NX], dd[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                uint32_t d[2];
                if constexpr (HD == 32) {
                    const int r0 = d_slot<HD>(8 * j + t), r1 = d_slot<HD>(8 * j + t + 4);
                    const uint32_t a = *(const uint16_t *)(tile + 8 * HD + r0 * 16 + 2 * g);
                    const uint32_t b = *(const uint16_t *)(tile + 8 * HD + r1 * 16 + 2 * g);
                    x[j][0] = a | b << 16;
                } else {
                    uint32_t w[2][HD / 64];
#pragma unroll
                    for (int y = 0; y < 2; y++) {
                        const int slot = d_slot<HD>(8 * j + t + 4 * y);
                        const uint8_t *row = tile + 8 * HD + slot * (HD / 2);
                        if constexpr (HD == 128) {
                            const uint2 v = *(const uint2 *)(row + 16 * d_piece<HD>(slot, g >> 1) + 8 * (g & 1));
                            w[y][0] = v.x;
                            w[y][1] = v.y;
                        } else {
                            w[y][0] = *(const uint32_t *)(row + 4 * g);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < HD / 64; i++) {
                        x[j][2 * i] = __byte_perm(w[0][i], w[1][i], 0x5410);
                        x[j][2 * i + 1] = __byte_perm(w[0][i], w[1][i], 0x7632);
                    }
                }
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int p = 8 * j + t + 4 * y;
                    d[y] = *(const uint16_t *)(tile + 17 * HD + 2 * (p * (HD / 32) + g * (HD / 16) / 16));
                    if (!whole && !sees(p)) d[y] = 0;
                }
                dd[j] = d[0] | d[1] << 16;
            }
#pragma unroll
            for (int i = 0; i < NX; i++) {
                const uint32_t y0 = x[0][i] >> 8, y1 = x[1][i] >> 8;
                mma16816(o[4 * i], pa[0], pa[1], pa[2], pa[3], nib_lo(x[0][i], dd[0]), nib_lo(x[1][i], dd[1]), o[4 * i]);
                mma16816(o[4 * i + 1], pa[0], pa[1], pa[2], pa[3], nib_hi(x[0][i], dd[0]), nib_hi(x[1][i], dd[1]), o[4 * i + 1]);
                mma16816(o[4 * i + 2], pa[0], pa[1], pa[2], pa[3], nib_lo(y0, dd[0]), nib_lo(y1, dd[1]), o[4 * i + 2]);
                mma16816(o[4 * i + 3], pa[0], pa[1], pa[2], pa[3], nib_hi(y0, dd[0]), nib_hi(y1, dd[1]), o[4 * i + 3]);
            }
        }
        cp_wait<0>();

        // ---- join the warps
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
            sm.m[warp][g] = m;
            sm.l[warp][g] = l;
        }
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int b = (2 * t + c) * (HD / 16) + 2 * (i >> 2) + ((i >> 1) & 1);
                sm.o[warp][g][b / 16 * 32 + b % 16 + 16 * (i & 1)] = o[i][c] + o[i][c + 2];
            }
        __syncthreads();
        const bool alone = u0 == 0 && u1 == S.units;
        // CTAs that share the item: from the one that holds its first unit
        const int64_t a0 = at - u0;
        const int first_cta = (int)(a0 / per), last_cta = (int)((a0 + S.units - 1) / per);
        float *mypart = parts + ((int64_t)blockIdx.x * 2 + (first_cta == (int)blockIdx.x ? 1 : 0)) * DHEADS * W;
        float *out = A.out + ((int64_t)req * A.n_heads + kvh * rep + h0) * HD;
        for (int i = tid; i < nh * HD; i += DNT) {
            const int h = i / HD, d = i % HD;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < DW; w++) M = fmaxf(M, sm.m[w][h]);
            const float ref = M == -INFINITY ? 0.f : M;
            float O = 0.f, L = 0.f;
#pragma unroll
            for (int w = 0; w < DW; w++) {
                const float a = exp2_approx(sm.m[w][h] - ref);
                O = fmaf(sm.o[w][h][d], a, O);
                L = fmaf(sm.l[w][h], a, L);
            }
            if (alone) {
                out[i] = L == 0.f ? 0.f : O / L;
            } else {
                __stcg(mypart + h * W + d, O);
                if (d == 0) {
                    __stcg(mypart + h * W + HD, M);
                    __stcg(mypart + h * W + HD + 1, L);
                }
            }
        }
        if (!alone) {
            __threadfence();
            __syncthreads();
            if (tid == 0) sm.last = atomicAdd(tickets + first_cta, 1) == last_cta - first_cta;
            __syncthreads();
            if (sm.last) {
                __threadfence();
                for (int i = tid; i < nh * HD; i += DNT) {
                    const int h = i / HD, d = i % HD;
                    float M = -INFINITY, O = 0.f, L = 0.f;
                    for (int c = first_cta; c <= last_cta; c++) {
                        const float *p = parts + ((int64_t)c * 2 + (c == first_cta ? 1 : 0)) * DHEADS * W + h * W;
                        const float pm = __ldcg(p + HD), mn = fmaxf(M, pm);
                        if (__ldcg(p + HD + 1) != 0.f) {
                            const float a = exp2_approx(M - mn), b = exp2_approx(pm - mn);
                            O = O * a + __ldcg(p + d) * b;
                            L = L * a + __ldcg(p + HD + 1) * b;
                            M = mn;
                        }
                    }
                    out[i] = L == 0.f ? 0.f : O / L;
                }
                if (tid == 0) tickets[first_cta] = 0;
            }
        }
        __syncthreads();
        at += u1 - u0;
        off += u1 - u0;
    }
}

// CTAs of the largest grid.
int max_ctas(const hd_ctx *ctx, int hd) { return ctx->sm_count * (hd == 128 ? d_occ<128>() : d_occ<64>()); }

template <int HD>
cudaError_t launch(hd_ctx *ctx, const Kv4Args &A, uint8_t *ws) {
    const int rep = A.n_heads / A.n_kv, groups = (rep + DHEADS - 1) / DHEADS, gh = (rep + groups - 1) / groups;
    const size_t smem = sizeof(DShared<HD>);
    cudaError_t e = cudaFuncSetAttribute(k_kv4_decode<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    // no more CTAs than the table's (or the window's) longest request can give work
    int64_t tiles = ((int64_t)A.max_pages << A.shift) / KV4_TILE;
    if (A.window) {
        const int64_t seen = ((int64_t)A.window + A.sinks) / KV4_TILE + 3;
        tiles = tiles < seen ? tiles : seen;
    }
    const int64_t units = tiles * A.seqs * A.n_kv * groups, most = max_ctas(ctx, HD);
    const int64_t want = (units + DMIN - 1) / DMIN;
    const int grid = (int)(want < most ? want : most);
    return hd_launch(ctx, k_kv4_decode<HD>, dim3(grid), dim3(DNT), smem, A, groups, gh, (int *)ws,
                     (float *)(ws + ((size_t)most * sizeof(int) + 255) / 256 * 256));
}

}  // namespace

extern "C" uint64_t hd_kv4_workspace_bytes(const hd_ctx *ctx, int n_heads, int n_kv, int head_dim) {
    if (!ctx || n_heads <= 0 || n_kv <= 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
    const uint64_t g = (uint64_t)max_ctas(ctx, head_dim);
    return (g * sizeof(int) + 255) / 256 * 256 + 2 * g * DHEADS * (head_dim + 2) * sizeof(float);
}

extern "C" int hd_kv4_attention_decode(hd_ctx *ctx, const float *q, int64_t q_ld, const uint8_t *cache, int64_t pages,
                                       int page_size, const int32_t *tables, int max_pages, const int32_t *lens, int seqs,
                                       int n_heads, int n_kv, int head_dim, int window, int sinks, float scale, float *out,
                                       void *ws, size_t ws_bytes) {
    Kv4Args A{q, q_ld, cache, pages, 0, tables, max_pages, lens, nullptr, seqs, seqs, n_heads, n_kv, window, sinks, scale, out};
    int rc = hd_kv4_attention_check(ctx, "hd_kv4_attention_decode", A, page_size, head_dim);
    if (rc || seqs == 0) return rc;
    const uint64_t need = hd_kv4_workspace_bytes(ctx, n_heads, n_kv, head_dim);
    HD_REQUIRE(ctx, !ws || ws_bytes >= need, HD_E_SHAPE, "hd_kv4_attention_decode: a workspace of %zu bytes (%llu needed)",
               ws_bytes, (unsigned long long)need);
    HD_REQUIRE(ctx, ((uintptr_t)ws & 15) == 0, HD_E_ARG, "hd_kv4_attention_decode: the workspace must be 16-byte aligned");
    HdDevice on(ctx);
    if (!ws) {
        if (!ctx->kv4_ws) {
            cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
            HD_CUDA_TRY(ctx, cudaStreamIsCapturing(ctx->stream, &capturing));
            HD_REQUIRE(ctx, capturing == cudaStreamCaptureStatusNone, HD_E_CUDA,
                       "hd_kv4_attention_decode: the context's workspace is made by the first call, which must not be "
                       "captured (or pass a workspace)");
            const size_t most = (size_t)hd_kv4_workspace_bytes(ctx, 1, 1, 128) + (size_t)hd_kv4_workspace_bytes(ctx, 1, 1, 64);
            void *p = nullptr;
            if (cudaMalloc(&p, most) != cudaSuccess) {
                cudaGetLastError();
                return hd_fail(ctx, HD_E_OOM, "hd_kv4_attention_decode: workspace of %zu bytes", most);
            }
            if (cudaMemsetAsync(p, 0, most, ctx->stream) != cudaSuccess || cudaStreamSynchronize(ctx->stream) != cudaSuccess) {
                cudaFree(p);
                return hd_fail(ctx, HD_E_CUDA, "hd_kv4_attention_decode: workspace: %s", cudaGetErrorString(cudaGetLastError()));
            }
            ctx->kv4_ws = (uint8_t *)p;
        }
        // the tickets of another head size's layout would meet this one's partials
        ws = ctx->kv4_ws + (head_dim == 128 ? 0 : (size_t)hd_kv4_workspace_bytes(ctx, 1, 1, 128));
    }
    cudaError_t e;
    if (head_dim == 128) e = launch<128>(ctx, A, (uint8_t *)ws);
    else if (head_dim == 64) e = launch<64>(ctx, A, (uint8_t *)ws);
    else e = launch<32>(ctx, A, (uint8_t *)ws);
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "hd_kv4_attention_decode: %s", cudaGetErrorString(e));
    return HD_OK;
}
