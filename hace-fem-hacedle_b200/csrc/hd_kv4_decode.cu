// hd_kv4_decode.cu -- decode attention (one query per request) over the paged
// 4-bit cache.
//
// Mathematics.  A warp takes a tile of 16 positions of one kv head at a time
// and keeps the running maximum, sum and output of up to 8 query heads that
// share it.  Both products run on m16n8k16 MMAs: rows 0..7 of the A operand
// are the heads' high f16 parts and rows 8..15 their low parts, so one MMA
// multiplies both and adding accumulator rows g and g + 8 -- which the same
// thread holds -- gives 22 significant bits of q (scaled per
// head) and of the softmax weights (the largest at 2^15), against cache values that
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
// them in order, so results do not depend on the schedule.  Many pieces of one
// head (a long request alone) join in groups of 16 CTAs first, so that no CTA
// walks hundreds of pieces alone; the groups count from the item's first CTA,
// so that up to 16 pieces join once (32 requests with a window of 2048, 14
// heads on 2 of 64: 12.6 us, 15.1 with groups of fixed CTAs).
//
// Measured, 28 heads on 4 kv heads of 128: 256 requests of 64 to 4096 tokens
// (152 MB of cache) 65 us, 2.3 TB/s; one request of 131001 tokens (75 MB) 38 us,
// 2.0 TB/s.  What bounds it is unpacking, not memory: about 440
// instructions per warp and 16 positions at HD 128, of which the f16 ones go
// at half rate, and the MMAs, together some 950 cycles a tile and SM sub-core
// where the bytes alone would take 400; and ~2.5 us per item that a CTA begins
// or joins.  Neither more warps (12 or 16 per SM: the same) nor the next
// step's scores computed beside this step's weights moved it.
#include <cmath>

#include "hd_internal.cuh"
#include "hd_kv4_math.cuh"
#include "hd_mma.cuh"

namespace {

constexpr int DW = 4;           // warps per CTA (2: 78 us against 66)
constexpr int DNT = 32 * DW;
constexpr int DPT = 2;          // tiles per step
template <int HD>
constexpr int d_stages() { return HD == 128 ? 2 : HD == 64 ? 3 : 4; }   // steps in a warp's ring
constexpr int DMIN = DPT * DW;  // fewest tiles a CTA takes (32: 10.2 us for one request of 700 tokens, 8.4 with 8)
constexpr int DHEADS = 8;       // query heads per unit
constexpr int DCOST = 16;       // what beginning an item costs, in tiles (24: 3% slower over ragged lengths)
constexpr int DJOIN = 16;       // CTAs whose partials are joined first
constexpr int DJOINS = 64;      // partials that one CTA joins at a time, at most

constexpr int D_OCC = 4;        // CTAs per SM (128 registers a thread)

template <int HD>
struct DShared {
    union {
        alignas(16) uint8_t ring[DW][d_stages<HD>()][DPT][kv4_tile_bytes(HD)];
        alignas(16) float o[DW][DHEADS][HD + 4];      // the warps' outputs, once the ring is drained
    };
    alignas(16) uint32_t q[HD / 16][32][4];
    float m[DW][DHEADS], l[DW][DHEADS];
    float ja[DJOINS * DHEADS], jl[DHEADS];
    float kappa[DHEADS];
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

// d += a b, m16n8k16, in place.
__device__ __forceinline__ void mma_add(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Shared memory by its 32-bit address, in the order written (the rings are
// filled behind the compiler's back).
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[N]) {
    static_assert(N == 1 || N == 2 || N == 4, "");
    if constexpr (N == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
    else if constexpr (N == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(a));
}

// What a request's last position sees.
__device__ __forceinline__ Seen last_sees(const Kv4Args &A, int len) {
    const int last = held_length(A, len) - 1;
    return seen_tiles(A.window, A.sinks, last, last);
}

// a / b, without the long division where 32 bits hold both.
__device__ __forceinline__ int64_t div_fast(int64_t a, int64_t b) {
    return (uint64_t)(a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}

// A CTA's run may begin with the end of one item and end with the beginning
// of another: two slots, the second for the item that begins in the run.
__device__ __forceinline__ int slot_of(int cta, int first_cta) { return 2 * cta + (cta == first_cta ? 1 : 0); }

// True in the CTA that arrives last of others + 1; the ticket is 0 again.
template <int HD>
__device__ bool arrive(DShared<HD> &sm, int *ticket, int others) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        sm.last = atomicAdd(ticket, 1) == others;
        if (sm.last) *ticket = 0;
    }
    __syncthreads();
    const bool last = sm.last;
    __threadfence();
    return last;
}

__device__ __forceinline__ void axpy4(float4 &y, float a, const float4 &x) {
    y.x = fmaf(a, x.x, y.x);
    y.y = fmaf(a, x.y, y.y);
    y.z = fmaf(a, x.z, y.z);
    y.w = fmaf(a, x.w, y.w);
}
__device__ __forceinline__ float4 over(const float4 &x, float l) {
    return l == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(x.x / l, x.y / l, x.z / l, x.w / l);
}

// Joins n <= DJOINS partials, the i-th in slot slot_at(i), in order: into slot
// `to` (a partial again; it may be one of them) or, for to < 0, the output.
template <int HD, typename SlotAt>
__device__ void join_parts(DShared<HD> &sm, float *parts, float2 *ml, int n, SlotAt slot_at, int nh, int to, float *out) {
    const int tid = threadIdx.x, lane = tid & 31;
    // half a warp per head
    for (int h = tid / 16; h < DHEADS; h += DNT / 16) {
        float M = -INFINITY, L = 0.f;
        for (int i = lane & 15; i < n; i += 16) M = fmaxf(M, __ldcg(ml + (int64_t)slot_at(i) * DHEADS + h).x);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float ref = M == -INFINITY ? 0.f : M;
        for (int i = lane & 15; i < n; i += 16) {
            const float2 v = __ldcg(ml + (int64_t)slot_at(i) * DHEADS + h);
            const float a = exp2_approx(v.x - ref);
            sm.ja[i * DHEADS + h] = a;
            L = fmaf(v.y, a, L);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        if ((lane & 15) == 0) {
            sm.jl[h] = L;
            if (to >= 0 && h < nh) sm.m[0][h] = M;
        }
    }
    __syncthreads();
    for (int i = tid; i < nh * (HD / 4); i += DNT) {
        const int h = i / (HD / 4);
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int c = 0; c < n; c++)
            axpy4(O, sm.ja[c * DHEADS + h], __ldcg((const float4 *)(parts + (int64_t)slot_at(c) * DHEADS * HD) + i));
        if (to < 0) *((float4 *)out + i) = over(O, sm.jl[h]);
        else __stcg((float4 *)(parts + (int64_t)to * DHEADS * HD) + i, O);   // each thread has read what it overwrites
    }
    if (to >= 0 && tid < nh) __stcg(ml + (int64_t)to * DHEADS + tid, make_float2(sm.m[0][tid], sm.jl[tid]));
}

// An item's length on the line that the CTAs share out: DCOST for its
// beginning, then its tiles.
__device__ __forceinline__ int cost_of(const Seen &s) { return s.units ? s.units + DCOST : 0; }

template <int HD>
__global__ void __launch_bounds__(DNT, D_OCC) k_kv4_decode(Kv4Args A, int groups, int gh, int *tickets, float2 *ml,
                                                               float *parts) {
    constexpr int NS = d_stages<HD>();
    constexpr int WPT = HD / 32;       // words of a key per thread
    constexpr int NT = HD / 8;         // column tiles of the output
    extern __shared__ __align__(16) uint8_t smem_raw[];
    DShared<HD> &sm = *reinterpret_cast<DShared<HD> *>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    pdl_wait();
    pdl_trigger();
    // this lane's place in a tile's copy: 16-byte piece `lane` of each 512 bytes, rows permuted
    const uint32_t ring0 = smem_u32(sm.ring[warp][0][0]);
    constexpr int PR = HD / 32;
    const int my_slot = (lane / PR & 8) | d_slot<HD>(lane / PR & 7);
    const uint32_t my_dst = HD == 32 ? 16u * lane : 16u * (my_slot * PR + d_piece<HD>(my_slot, lane % PR));
    // where this lane reads a tile (first column tile of a step, first half of the positions)
    const int kp = (g >> 1) + 4 * (g & 1), kslot = d_slot<HD>(kp);
    constexpr int ROW = HD / 2;                     // bytes of a row's quants
    const uint32_t k_at = kslot * ROW + (HD == 128 ? 16 * d_piece<HD>(kslot, t) : t * (HD / 8));
    const uint32_t kd_at = 16 * HD + 2 * (kp * (HD / 32) + t * (HD / 8) / 16);
    const int vslot = d_slot<HD>(t), vslot4 = d_slot<HD>(t + 4);
    const uint32_t v_in = HD == 128 ? 16 * d_piece<HD>(vslot, g >> 1) + 8 * (g & 1) : g * (HD / 16);
    const uint32_t v_at = 8 * HD + vslot * ROW + v_in, v4_at = 8 * HD + vslot4 * ROW + v_in;
    const uint32_t vd_at = 17 * HD + 2 * (t * (HD / 32) + g * (HD / 16) / 16);
    const uint32_t q_at = smem_u32(sm.q[0][lane]);
    const uint32_t magic = KV4_MAGIC + (uint32_t)(A.shift >> 8);   // the shift is at most 10
    const int items = A.n_kv * groups, rep = A.n_heads / A.n_kv;

    // ---- this CTA's run of units
    const int per_thread = (A.seqs + DNT - 1) / DNT, rb = min(A.seqs, tid * per_thread), re = min(A.seqs, rb + per_thread);
    int64_t mine = 0;
    for (int r = rb; r < re; r++) mine += cost_of(last_sees(A, A.lens[r]));
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
    int64_t per = div_fast(total + gridDim.x - 1, gridDim.x);
    per = per < DMIN ? DMIN : per;
    const int64_t c_begin = per * blockIdx.x, c_end = min(total, c_begin + per);
    // requests without any position
    for (int r = blockIdx.x; r < A.seqs; r += gridDim.x)
        if (last_sees(A, A.lens[r]).units == 0)
            for (int i = tid; i < A.n_heads * HD; i += DNT) A.out[(int64_t)r * A.n_heads * HD + i] = 0.f;
    if (c_begin >= c_end) return;
    if (before <= c_begin && c_begin < before + mine * items) {
        int r = rb;
        for (;; r++) {
            const int64_t u = (int64_t)cost_of(last_sees(A, A.lens[r])) * items;
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
        const Seen S = last_sees(A, A.lens[req]);
        const int cost = cost_of(S);
        if (off >= (int64_t)cost * items) {
            off -= (int64_t)cost * items;
            req++;
            continue;
        }
        const int item = (int)div_fast(off, cost), o0 = (int)(off - (int64_t)item * cost);
        const int o1 = (int)min((int64_t)cost, o0 + (c_end - at));
        const int u0 = max(0, o0 - DCOST), u1 = max(0, o1 - DCOST);
        const int64_t a0 = at - o0 + DCOST;         // where the item's tiles begin on the line
        at += o1 - o0;
        off += o1 - o0;
        if (u0 >= u1) continue;
        const int kvh = item / groups, h0 = (item - kvh * groups) * gh, nh = min(gh, rep - h0);
        const int32_t *table = A.tables + (int64_t)req * A.max_pages;

        // ---- q of the heads, scaled, in two f16 parts (one warp; the others wait below)
        if (warp == 0) {
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
            float up, kappa;
            q_scales(A, mx, up, kappa);
            if (t == 0) sm.kappa[g] = kappa;
#pragma unroll
            for (int w = 0; w < WPT; w++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const float *v = x[w] + 4 * hf;
                    uint4 f;
                    split2(v[0] * up, v[2] * up, f.x, f.y);
                    split2(v[1] * up, v[3] * up, f.z, f.w);
                    *(uint4 *)sm.q[2 * w + hf][lane] = f;
                }
        }

        // ---- this warp's steps of two tiles: step k is units first_u + DPT * DW * k ..
        const int first_u = u0 + DPT * warp;
        const int n = u1 > first_u ? (u1 - first_u + DPT * DW - 1) / (DPT * DW) : 0;
        // lane 2 i + j holds where tile j of step 16 * batch + i lies, or -1
        auto look = [&](int batch) {
            const int u = first_u + DPT * DW * (16 * batch + (lane >> 1)) + (lane & 1);
            if (u >= u1) return -1;
            const int tile = S.tile(u);
            const int64_t page = table[tile >> (A.shift - 4)];
            if (page < 0 || page >= A.pages) return -1;
            return (int)(((page * A.n_kv + kvh) << (A.shift - 4)) + (tile & ((1 << (A.shift - 4)) - 1)));
        };
        int ids = look(0), ids_next = n > 16 ? look(1) : -1;
        uint32_t named = 0;             // bits 2 s, 2 s + 1: the tiles of ring stage s exist
        auto fetch = [&](int k, int stage) {
            if (k < n) {
                if (k && (k & 15) == 0) {
                    ids = ids_next;
                    ids_next = look(k / 16 + 1);
                }
#pragma unroll
                for (int j = 0; j < DPT; j++) {
                    const int at = __shfl_sync(0xffffffffu, ids, 2 * (k & 15) + j);
                    named &= ~(1u << (DPT * stage + j));
                    if (at < 0) continue;
                    named |= 1u << (DPT * stage + j);
                    const uint8_t *src = A.cache + (uint64_t)(uint32_t)at * kv4_tile_bytes(HD) + 16 * lane;
                    const uint32_t dst = smem_u32(sm.ring[warp][stage][j]) + my_dst;
                    constexpr int N = kv4_tile_bytes(HD) / 16, FULL = N / 32;
#pragma unroll
                    for (int c = 0; c < FULL; c++) cp16(dst + 512 * c, src + 512 * c);
                    if (lane < N - 32 * FULL) cp16(ring0 + (uint32_t)(((stage * DPT) + j) * kv4_tile_bytes(HD)) + 512 * FULL + 16 * lane, src + 512 * FULL);
                }
            }
            cp_commit();
        };
#pragma unroll
        for (int s = 0; s < NS - 1; s++) fetch(s, s);
        __syncthreads();                // q is there
        const float kappa = sm.kappa[g];
        float o[NT][4], m = -INFINITY, ref = 0.f, l = 0.f;
#pragma unroll
        for (int i = 0; i < NT; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) o[i][c] = 0.f;

        // units whose 16 positions are all seen: from .. to - 1, and those below sinks
        const int whole_from = S.sink + ((S.first & (KV4_TILE - 1)) != 0), whole_to = S.units - ((S.last + 1) % KV4_TILE != 0);
        const int whole_sinks = min(A.sinks, S.first) / KV4_TILE;
        int stage = 0;
        for (int k = 0; k < n; k++) {
            __syncwarp();               // all lanes have read the stage that is refilled
            fetch(k + NS - 1, stage == 0 ? NS - 1 : stage - 1);
            cp_wait<NS - 1>();
            __syncwarp();
            const int u = first_u + DPT * DW * k;
            const int cur = stage;
            const uint32_t ok = named >> (DPT * stage) & 3;
            stage = stage == NS - 1 ? 0 : stage + 1;
            if (!ok) continue;
            const bool whole = ok == 3 && ((u >= whole_from && u + 1 < whole_to) || u + 1 < whole_sinks);
            // a tile that is seen in part: the scales of the other positions become 0, so that whatever
            // their slots hold counts for nothing (their scores are hidden below)
            uint32_t hidden = 0;        // bit 16 j + p: position p of tile j is not seen
            if (!whole) {
                const int j = lane >> 4, p = lane & 15;
                const bool sees = (ok >> j & 1) && S.any(S.tile(u + j) * KV4_TILE + p, A.sinks);
                if (!sees) {
                    uint8_t *d = sm.ring[warp][cur][j] + 16 * HD + p * (HD / 16);
#pragma unroll
                    for (int i = 0; i < HD / 32; i++) {
                        *(uint16_t *)(d + 2 * i) = 0;
                        *(uint16_t *)(d + HD + 2 * i) = 0;
                    }
                }
                hidden = __ballot_sync(0xffffffffu, !sees);
                __syncwarp();
            }

            // ---- scores of positions t, t + 4 (first column tile) and t + 8, t + 12 (second) of each tile
            const uint32_t base = ring0 + (uint32_t)(cur * DPT * kv4_tile_bytes(HD));
            float s[2 * DPT][4];
            uint32_t w[2 * DPT][WPT], dk[2 * DPT];
#pragma unroll
            for (int j = 0; j < 2 * DPT; j++) {
                const uint32_t tile = base + (j >> 1) * kv4_tile_bytes(HD);
                lds_words<WPT>(tile + k_at + (j & 1) * 8 * ROW, w[j]);
                const uint32_t d = lds16(tile + kd_at + (j & 1) * (HD / 2));
                dk[j] = __byte_perm(d, d, 0x1010);
#pragma unroll
                for (int c = 0; c < 4; c++) s[j][c] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < WPT; i++) {
                uint32_t q0[4], q1[4];
                lds_words<4>(q_at + 1024 * i, q0);
                lds_words<4>(q_at + 1024 * i + 512, q1);
#pragma unroll
                for (int j = 0; j < 2 * DPT; j++) {
                    const uint32_t w8 = w[j][i] >> 8;
                    mma_add(s[j], q0[0], q0[1], q0[2], q0[3], nib_lo(w[j][i], dk[j], magic), nib_lo(w8, dk[j], magic));
                    mma_add(s[j], q1[0], q1[1], q1[2], q1[3], nib_hi(w[j][i], dk[j], magic), nib_hi(w8, dk[j], magic));
                }
            }
            float e[DPT][4], mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < DPT; j++) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    e[j][c] = s[2 * j + (c >> 1)][c & 1] + s[2 * j + (c >> 1)][(c & 1) + 2];
                }
            }
            if (hidden) {
                const uint32_t mine_hidden = hidden >> t;
#pragma unroll
                for (int j = 0; j < DPT; j++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (mine_hidden >> (16 * j + 4 * c) & 1) e[j][c] = -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < DPT; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) mx = fmaxf(mx, e[j][c]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m)) {
                const float mn = fmaxf(m, mx), rn = weight_ref(mn, kappa), a = m == -INFINITY ? 0.f : exp2_approx(ref - rn);
                m = mn;
                ref = rn;
                l *= a;
#pragma unroll
                for (int i = 0; i < NT; i++)
#pragma unroll
                    for (int c = 0; c < 4; c++) o[i][c] *= a;
            }
            uint32_t pa[DPT][4];
#pragma unroll
            for (int j = 0; j < DPT; j++) {
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    e[j][c] = exp2_approx(fmaf(e[j][c], kappa, -ref));
                    l += e[j][c];
                }
                split2(e[j][0], e[j][1], pa[j][0], pa[j][1]);
                split2(e[j][2], e[j][3], pa[j][2], pa[j][3]);
            }

            // ---- output: value pairs (t, t + 4) and (t + 8, t + 12) of HD / 16 bytes of each row
#pragma unroll
            for (int jt = 0; jt < DPT; jt++) {
                const uint32_t tile = base + jt * kv4_tile_bytes(HD);
                constexpr int NX = HD >= 64 ? HD / 32 : 1;    // half words of a row's bytes
                uint32_t x[2][NX], dd[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    if constexpr (HD == 32) {
                        x[j][0] = __byte_perm(lds16(tile + v_at + j * 8 * ROW), lds16(tile + v4_at + j * 8 * ROW), 0x5410);
                    } else {
                        uint32_t v0[HD / 64], v4[HD / 64];
                        lds_words<HD / 64>(tile + v_at + j * 8 * ROW, v0);
                        lds_words<HD / 64>(tile + v4_at + j * 8 * ROW, v4);
#pragma unroll
                        for (int i = 0; i < HD / 64; i++) {
                            x[j][2 * i] = __byte_perm(v0[i], v4[i], 0x5410);
                            x[j][2 * i + 1] = __byte_perm(v0[i], v4[i], 0x7632);
                        }
                    }
                    dd[j] = __byte_perm(lds16(tile + vd_at + j * (HD / 2)), lds16(tile + vd_at + HD / 4 + j * (HD / 2)), 0x5410);
                }
                const uint32_t(&pj)[4] = pa[jt];
#pragma unroll
                for (int i = 0; i < NX; i++) {
                    const uint32_t y0 = x[0][i] >> 8, y1 = x[1][i] >> 8;
                    mma_add(o[4 * i], pj[0], pj[1], pj[2], pj[3], nib_lo(x[0][i], dd[0], magic), nib_lo(x[1][i], dd[1], magic));
                    mma_add(o[4 * i + 1], pj[0], pj[1], pj[2], pj[3], nib_hi(x[0][i], dd[0], magic), nib_hi(x[1][i], dd[1], magic));
                    mma_add(o[4 * i + 2], pj[0], pj[1], pj[2], pj[3], nib_lo(y0, dd[0], magic), nib_lo(y1, dd[1], magic));
                    mma_add(o[4 * i + 3], pj[0], pj[1], pj[2], pj[3], nib_hi(y0, dd[0], magic), nib_hi(y1, dd[1], magic));
                }
            }
        }
        cp_wait<0>();
        __syncthreads();                // every warp is done with the ring

        // ---- join the warps
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
            sm.m[warp][g] = m == -INFINITY ? m : ref;   // what the warp's l and o are in units of
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
        const int first_cta = alone ? (int)blockIdx.x : (int)div_fast(a0, per), last_cta = alone ? (int)blockIdx.x : (int)div_fast(a0 + S.units - 1, per);
        float *out = A.out + ((int64_t)req * A.n_heads + kvh * rep + h0) * HD;
        const int slot = slot_of((int)blockIdx.x, first_cta);
        for (int i = tid; i < nh * (HD / 4); i += DNT) {
            const int h = i / (HD / 4), d = 4 * (i % (HD / 4));
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < DW; w++) M = fmaxf(M, sm.m[w][h]);
            const float ref = M == -INFINITY ? 0.f : M;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
            float L = 0.f;
#pragma unroll
            for (int w = 0; w < DW; w++) {
                const float a = exp2_approx(sm.m[w][h] - ref);
                axpy4(O, a, *(const float4 *)&sm.o[w][h][d]);
                L = fmaf(sm.l[w][h], a, L);
            }
            if (alone) {
                *((float4 *)out + i) = over(O, L);
            } else {
                __stcg((float4 *)(parts + (int64_t)slot * DHEADS * HD) + i, O);
                if (d == 0) __stcg(ml + (int64_t)slot * DHEADS + h, make_float2(M, L));
            }
        }
        if (!alone) {
            // pieces join in groups of DJOIN CTAs first, whose sums then join, each by whoever comes last
            const int gb = first_cta + ((int)blockIdx.x - first_cta) / DJOIN * DJOIN, ge = min(last_cta, gb + DJOIN - 1);
            const int ng = (last_cta - first_cta) / DJOIN + 1;
            if (arrive(sm, tickets + slot_of(gb, first_cta), ge - gb)) {
                join_parts<HD>(sm, parts, ml, ge - gb + 1, [&](int i) { return slot_of(gb + i, first_cta); }, nh,
                               ng > 1 ? slot_of(gb, first_cta) : -1, out);
                if (ng > 1 && arrive(sm, tickets + 2 * gridDim.x + first_cta, ng - 1))
                    join_parts<HD>(sm, parts, ml, ng,
                                   [&](int i) { return slot_of(first_cta + i * DJOIN, first_cta); }, nh, -1, out);
            }
        }
        __syncthreads();
    }
}

// CTAs of the largest grid, the same for every head size: the workspace's tickets are then, too, and one
// workspace serves calls of several.
int max_ctas(const hd_ctx *ctx) { return min(ctx->sm_count * D_OCC, DJOIN * DJOINS); }

template <int HD>
cudaError_t launch(hd_ctx *ctx, const Kv4Args &A, uint8_t *ws) {
    const int rep = A.n_heads / A.n_kv, groups = (rep + DHEADS - 1) / DHEADS, gh = (rep + groups - 1) / groups;
    const size_t smem = sizeof(DShared<HD>);
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = hd_allow_smem(allowed, ctx, (const void *)k_kv4_decode<HD>, smem);
    if (e != cudaSuccess) return e;
    // no more CTAs than the table's (or the window's) longest request can give work
    int64_t tiles = ((int64_t)A.max_pages << A.shift) / KV4_TILE;
    if (A.window) {
        const int64_t seen = ((int64_t)A.window + A.sinks) / KV4_TILE + 3;
        tiles = tiles < seen ? tiles : seen;
    }
    const int64_t tiles_items = (int64_t)A.seqs * A.n_kv * groups, units = tiles * tiles_items;
    const int64_t most = max_ctas(ctx);
    const int64_t want = (units + tiles_items * DCOST + DMIN - 1) / DMIN;
    const int grid = (int)(want < most ? want : most);
    float2 *ml = (float2 *)(ws + ((size_t)3 * most * sizeof(int) + 255) / 256 * 256);
    return hd_launch(ctx, k_kv4_decode<HD>, dim3(grid), dim3(DNT), smem, A, groups, gh, (int *)ws, ml,
                     (float *)(ml + (size_t)2 * most * DHEADS));
}

}  // namespace

extern "C" uint64_t hd_kv4_workspace_bytes(const hd_ctx *ctx, int n_heads, int n_kv, int head_dim) {
    if (!ctx || n_heads <= 0 || n_kv <= 0 || (head_dim != 32 && head_dim != 64 && head_dim != 128)) return 0;
    const uint64_t g = (uint64_t)max_ctas(ctx);
    return (3 * g * sizeof(int) + 255) / 256 * 256 + 2 * g * DHEADS * (head_dim + 2) * sizeof(float);
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
            const size_t most = (size_t)hd_kv4_workspace_bytes(ctx, 1, 1, 128);
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
        ws = ctx->kv4_ws;
    }
    cudaError_t e;
    if (head_dim == 128) e = launch<128>(ctx, A, (uint8_t *)ws);
    else if (head_dim == 64) e = launch<64>(ctx, A, (uint8_t *)ws);
    else e = launch<32>(ctx, A, (uint8_t *)ws);
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "hd_kv4_attention_decode: %s", cudaGetErrorString(e));
    return HD_OK;
}
