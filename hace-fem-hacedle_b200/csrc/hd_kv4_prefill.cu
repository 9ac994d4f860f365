// hd_kv4_prefill.cu -- causal attention of prompt chunks over the paged 4-bit
// cache on the tcgen05 tensor cores.
//
// A CTA takes 128 query rows -- the heads of one kv head for as many
// consecutive tokens of a request as fit -- and walks the positions that any
// of them sees, 128 at a time.  Operands and accuracy are those of the decode
// kernel: cache values are exact in f16, q and the softmax weights enter in
// two f16 parts, so each product is two MMAs into the same f32 accumulator.
//   S = Qhi K^T + Qlo K^T      A = Q in shared memory, B = K [128][HD]
//   PV = Phi V + Plo V         A = P in tensor memory, B = V^T [HD][128]
// O itself is kept in registers and takes up a tile's PV with an addition: an
// accumulator that grew over the whole context lost low bits at every MMA
// (7e-6 of the result over 8192 positions, 4e-7 now), and the change of the
// running maximum is one multiplication on the way.
//
// Roles (15 warps, one CTA per SM; S, P and PV have two buffers each in tensor
// memory, K and V two stages in shared memory, so the roles work on different
// tiles at a time):
//   warps 0-7       softmax: a thread has a row and half of a tile's columns,
//            and half of the row's dimensions of O; the two threads of a row
//            exchange their maxima through shared memory.  P overwrites S in
//            place: CW scores become CW / 2 columns of high and CW / 2 of low
//            parts.  Two f32 operations an instruction where they pair.
//   warps 8-11      write K and V^T as f16 operands in SWIZZLE_128B from the
//            cache tiles.  K's dimensions keep the order in which nibbles unpack
//            and Q is stored to match; V is paired by byte permutes, so neither
//            is transposed through memory.
//   warp 12, 13     issue the MMAs of S and of PV: one thread for both was the
//            pace (an MMA costs its issuer 60 to 80 cycles, 32 of them a tile).
//   warp 14         fetches cache tiles by bulk copies, a position tile ahead
//            (by one of the unpacking warps, the barrier among them and the page
//            table's latency stood in each tile: 52 us against 46.6 below).
//
// A value that is not finite (a cache row quantized from a NaN) must reach the
// rows that see its position and no other, but 0 * NaN is NaN: such values
// enter V as 0 and are kept in a bit mask per position, which the rows that
// see it take over for their output dimensions.
//
// Measured: 4096 rows on 8192 positions, 28 heads on 4 of 128 (361 GFLOP
// counted once), 0.94 ms: 384 TFLOP/s, 769 of MMA work with the two parts of q
// and P, 46% of the measured bf16 rate.  What bounds that: an SM takes 299 steps
// of 128 positions, 6.2 thousand cycles each, where the softmax warps or the
// unpacking warps alone need about 4.5 thousand and the MMAs 2.2 thousand, so
// the roles wait for one another as well.  No pipe is full (issue slots 51%,
// tensor 36%): three warps per scheduler wait for their own latencies, tensor
// memory's and the instruction cache's (either role runs through its code once
// a tile).  Chunks of 1 to 500 rows of 12 requests, 14 heads on 2 of 64, take 37
// to 47 us by how long the chunks' prefixes are: 154 CTAs are about one wave,
// and the one with the longest walk (16 to 18 steps, 2.4 to 6 on average) sets
// the time, since a row tile's positions are not split.  Slower: 8 unpacking or
// 16 softmax warps (1.1 and 1.5 ms), registers moved from the issuing to the
// softmax warps (no spills, 1.1 ms), half of the scores kept in registers over
// the barrier (1.1 ms), the unpacking loops rolled (1.03 ms), a subtraction of
// the maximum before the multiplication with kappa (0.96 ms).
#include "hd_internal.cuh"
#include "hd_kv4_math.cuh"
#include "hd_tc.cuh"

namespace {

constexpr int PM = 128, PN = 128;               // rows, positions per tile
constexpr int P_SOFT = 256, P_DEQ = 128;        // threads of the softmax and of the unpacking warps
constexpr int P_THREADS = P_SOFT + P_DEQ + 96;
constexpr int PG = PN / KV4_TILE;               // cache tiles per position tile
constexpr int ABSENT = 0x7ffffff0;              // position of a cache tile that is not there

template <int HD>
struct PLayout {
    static constexpr int ATOMS = HD > 64 ? HD / 64 : 1;      // 128-byte columns of a row of K and Q
    static constexpr int Q = PM * 128 * ATOMS, K = PN * 128 * ATOMS, V = HD * 256;
    // a position tile's cache tiles as they are, 32 bytes apart from a multiple of 128, so that the same rows of
    // different ones lie in different banks
    static constexpr int RAW1 = kv4_tile_bytes(HD) + (kv4_tile_bytes(HD) % 128 ? 0 : 32), RAW = PG * RAW1;
    static constexpr int OPERANDS = 2 * Q + 2 * (K + V) + RAW;
    // at least half an SM's shared memory: a second CTA would wait for tensor memory
    static constexpr size_t BYTES = (OPERANDS > 120 * 1024 ? OPERANDS : 120 * 1024) + 1024;
};

struct PShared {
    unsigned long long k_full[2], v_full[2], s_full[2], p_full[2], pv_done[2], raw_full, raw_free, fin[2];
    uint32_t tmem;
    int pos[8][PG];               // first position of each cache tile of a position tile (read long after K is free)
    uint8_t nan_bits[4][4][PN / 8];   // which of 8 positions' values of a group are not finite
    alignas(16) int nan_any[4][4];    // whether an unpacking warp found any
    float mx[2][2][PM], l[2][PM];
    int64_t part[P_THREADS / 32];
    int req, tile, found;
};

__device__ __forceinline__ void tmem_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(a));
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; i++) asm volatile("" : "+r"(r[i])::"memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
        "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t (&r)[32]) { tmem_ld32(a, r); }
__device__ __forceinline__ void tmem_ld(uint32_t a, uint32_t (&r)[16]) {
    tmem_ld16_async(a, r);
    tmem_wait_ld();
    tmem_regs_ready(r);
}
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t (&r)[32]) { tmem_st32(a, r); }
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(a)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// Two f32 operations an instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// split2 of a pair.
__device__ __forceinline__ void split_pair(uint64_t x, uint32_t &hi, uint32_t &lo) {
    const float2 v = unpack2(x);
    const __half2 h = __floats2half2_rn(v.x, v.y);
    const float2 f = __half22float2(h), d = unpack2(fma2(pack2(f.x, f.y), pack2(-1.f, -1.f), x));
    const __half2 l = __floats2half2_rn(d.x, d.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ bool not_finite(uint32_t d) { return (d & 0x7fffu) >= 0x7c00u; }

template <int HD>
__global__ void __launch_bounds__(P_THREADS, 1) k_kv4_prefill(Kv4Args A, int tq, int *flag) {
    using L = PLayout<HD>;
    constexpr int KS = HD / 16;                            // k-steps of the first product
    // scores that a softmax thread takes at a time (16 for HD 64: 54 us for 12 short prompts, 46.5 with 32; 32 for HD
    // 128: 1.06 ms for 4096 rows, 0.95 with 16: its two rolled loops then stay in the instruction cache)
    constexpr int CW = HD == 128 ? 16 : 32;
    constexpr uint32_t S_COL = 0, PV_COL = 2 * PN;         // tensor memory: two buffers of S and P, then two of PV
    extern __shared__ uint8_t raw[];
    __shared__ PShared sm;
    uint8_t *base = (uint8_t *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const uint32_t q_hi = smem_u32(base), q_lo = q_hi + L::Q, kv0 = q_lo + L::Q;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();

    // ---- which rows: query tiles of all requests in one line, the last first (they see most)
    const int kvh = blockIdx.x % A.n_kv, index = blockIdx.x / A.n_kv, rep = A.n_heads / A.n_kv;
    {
        auto tiles_of = [&](int r) { return (max(0, A.row0[r + 1] - A.row0[r]) + tq - 1) / tq; };
        const int per = (A.seqs + P_THREADS - 1) / P_THREADS, b = min(A.seqs, tid * per), e = min(A.seqs, b + per);
        int64_t mine = 0;
        for (int r = b; r < e; r++) mine += tiles_of(r);
        int64_t inc = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) sm.part[warp] = inc;
        if (tid == 0) sm.found = 0;
        __syncthreads();
        int64_t at = inc - mine, total = 0;
        for (int w = 0; w < P_THREADS / 32; w++) {
            if (w < warp) at += sm.part[w];
            total += sm.part[w];
        }
        const int64_t want = total - 1 - index;
        if (want >= at && want < at + mine) {
            int r = b;
            for (;; r++) {
                const int t = tiles_of(r);
                if (want < at + t) break;
                at += t;
            }
            sm.req = r;
            sm.tile = (int)(want - at);
            sm.found = 1;
        }
        __syncthreads();
        if (!sm.found) return;
    }
    const int req = sm.req, r_begin = A.row0[req], n_new = A.row0[req + 1] - r_begin, t0 = sm.tile * tq;
    const int tokens = min(tq, n_new - t0), rows = tokens * rep;
    const int i0 = held_length(A, A.lens[req]) - n_new + t0;      // the first token's position (below 0: it sees nothing)
    const Seen S = seen_tiles(A.window, A.sinks, i0, i0 + tokens - 1);
    const int nj = (S.units + PG - 1) / PG;
    const int32_t *table = A.tables + (int64_t)req * A.max_pages;
    // (rows beyond the buffers, which row0 may name, are neither read nor written)
    auto row_ok = [&](int r) { return r < rows && r_begin >= 0 && (int64_t)r_begin + t0 + r / rep < A.rows; };

    if (tid == 0) {
        for (int s = 0; s < 2; s++) {
            mbar_init(smem_u32(&sm.k_full[s]), P_DEQ);
            mbar_init(smem_u32(&sm.v_full[s]), P_DEQ);
            mbar_init(smem_u32(&sm.s_full[s]), 2);         // the MMAs, and their issuer
            mbar_init(smem_u32(&sm.p_full[s]), P_SOFT);
            mbar_init(smem_u32(&sm.pv_done[s]), 2);        // likewise
            mbar_init(smem_u32(&sm.fin[s]), 1);
        }
        mbar_init(smem_u32(&sm.raw_full), 1);
        mbar_init(smem_u32(&sm.raw_free), P_DEQ / 32);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // ---- Q: rows of the first warps' threads, half of the 16-byte chunks each
    float kappa = 0.f;
    const int r = tid & (PM - 1), half = tid >> 7;
    if (tid < P_SOFT) {
        constexpr int CH = HD / 16;                        // chunks of 8 dimensions per thread
        float4 x[CH][2];
        const float *q = A.q + ((int64_t)r_begin + t0 + r / rep) * A.q_ld + (int64_t)(kvh * rep + r % rep) * HD;
        const bool ok = row_ok(r);
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int ch = half * CH + c, d = ch / 4 * 32 + 4 * (ch % 4);
#pragma unroll
            for (int y = 0; y < 2; y++) {
                x[c][y] = ok ? *(const float4 *)(q + d + 16 * y) : make_float4(0.f, 0.f, 0.f, 0.f);
                mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[c][y].x), fabsf(x[c][y].y)), fmaxf(fabsf(x[c][y].z), fabsf(x[c][y].w))));
            }
        }
        sm.mx[0][half][r] = mx;
        bar_sync(1, P_SOFT);
        float up;
        q_scales(A, fmaxf(sm.mx[0][0][r], sm.mx[0][1][r]), up, kappa);
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int ch = half * CH + c;
            uint4 hi, lo;
            split2(x[c][0].x * up, x[c][0].z * up, hi.x, lo.x);
            split2(x[c][0].y * up, x[c][0].w * up, hi.y, lo.y);
            split2(x[c][1].x * up, x[c][1].z * up, hi.z, lo.z);
            split2(x[c][1].y * up, x[c][1].w * up, hi.w, lo.w);
            const int at = (ch >> 3) * (PM * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
            *(uint4 *)(base + at) = hi;
            *(uint4 *)(base + L::Q + at) = lo;
        }
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem;
    // Only now: the GEMMs and GEMVs of this library allocate tensor memory before they wait for the kernel in front of
    // them, so one that came to lie on this SM first would hold what this CTA still asks for, and wait for it.
    pdl_trigger();

    if (warp < 8) {
        // ================= softmax
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const int i_row = i0 + r / rep, f_row = A.window && i_row >= A.window ? i_row - A.window + 1 : 0;
        constexpr int OD = HD / 2, OC = OD < 32 ? 16 : 32;     // this thread's dimensions, and how many it reads at once
        uint64_t o[OD / 2];                // pairs of dimensions
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int i = 0; i < OD / 2; i++) o[i] = 0;
        uint32_t nan_mine = 0;
        bool alive = true;
        // the groups of tile j's values that are not finite, of positions that the row sees
        auto take_nans = [&](int j) {
            const int4 odd = *(const int4 *)sm.nan_any[j & 3];
            if (!(odd.x | odd.y | odd.z | odd.w)) return;
            for (int i = 0; i < PN; i++) {
                const int p = sm.pos[j & 7][i / KV4_TILE] + i % KV4_TILE;
                if (!(p <= i_row && (p >= f_row || p < A.sinks))) continue;
                for (int g = 0; g < HD / 32; g++) nan_mine |= (uint32_t)(sm.nan_bits[j & 3][g][i / 8] >> (i % 8) & 1) << g;
            }
        };
        // o += the PV of tile j
        auto take = [&](int j) {
            alive = alive && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.pv_done[j & 1]), (j >> 1) & 1, flag));
            if (!alive) return;
            tc_fence_after();
            take_nans(j);
            const uint32_t at = tmem + lanes + PV_COL + (j & 1) * HD + half * OD;
#pragma unroll
            for (int c = 0; c < OD; c += OC) {
                {
                    uint32_t x[OC];
                    tmem_ld(at + c, x);
#pragma unroll
                    for (int i = 0; i < OC / 2; i++)
                        o[c / 2 + i] = add2(o[c / 2 + i], pack2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])));
                }
            }
        };
        for (int j = 0; j < nj; j++) {
            const int s = j & 1, k = j >> 1;
            const uint32_t t_s = tmem + lanes + S_COL + s * PN + half * (PN / 2);
            // (after a wait that ran out a warp goes on to meet the others at the barriers, and touches nothing)
            // k_full is not waited for here: K's stage may be filled twice before a slow warp comes by, and a parity
            // does not tell a phase from the one after the next.  S of tile j + 2 waits for this tile's weights, so
            // s_full cannot run ahead, and its issuer's own arrival hands on what the unpacking warps wrote.
            alive = alive && __all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.s_full[s]), k & 1, flag));
            tc_fence_after();
            // scores of CW columns, -infinity where the row does not see the position
            auto load = [&](int c, float (&v)[CW]) {
                tmem_ld(t_s + CW * c, reinterpret_cast<uint32_t (&)[CW]>(v));
#pragma unroll
                for (int h = 0; h < CW / KV4_TILE; h++) {
                    const int p0 = sm.pos[j & 7][PN / 2 / KV4_TILE * half + CW / KV4_TILE * c + h];
                    const bool all = p0 + KV4_TILE - 1 <= i_row && (p0 >= f_row || p0 <= A.sinks - KV4_TILE);
                    if (__all_sync(0xffffffffu, all)) continue;
#pragma unroll
                    for (int i = 0; i < KV4_TILE; i++) {
                        const int p = p0 + i;
                        if (!(p <= i_row && (p >= f_row || p < A.sinks))) v[16 * h + i] = -INFINITY;
                    }
                }
            };
            float mx = -INFINITY;
#pragma unroll 1
            for (int c = 0; c < PN / 2 / CW && alive; c++) {
                float v[CW];
                load(c, v);
                float a = v[0], b = v[1];
#pragma unroll
                for (int i = 2; i < CW - 2; i += 4) {
                    a = max3(a, v[i], v[i + 1]);
                    b = max3(b, v[i + 2], v[i + 3]);
                }
                mx = max3(mx, max3(a, b, v[CW - 2]), v[CW - 1]);
            }
            sm.mx[s][half][r] = mx;          // (the other buffer next time: one barrier a tile is enough)
            bar_sync(1, P_SOFT);
            if (!alive) continue;
            const float mn = fmaxf(m, fmaxf(mx, sm.mx[s][half ^ 1][r])), ref = weight_ref(mn, kappa);
            const float a = m == -INFINITY ? 0.f : exp2_approx(weight_ref(m, kappa) - ref);
            m = mn;
            const uint64_t kappa2 = pack2(kappa, kappa), ref2 = pack2(-ref, -ref);
            uint64_t sum = 0;
#pragma unroll 1
            for (int c = 0; c < PN / 2 / CW; c++) {
                float v[CW];
                load(c, v);
                uint32_t p[CW];
#pragma unroll
                for (int i = 0; i < CW / 2; i++) {
                    const float2 t = unpack2(fma2(pack2(v[2 * i], v[2 * i + 1]), kappa2, ref2));
                    const uint64_t x = pack2(exp2_approx(t.x), exp2_approx(t.y));
                    sum = add2(sum, x);
                    split_pair(x, p[i], p[CW / 2 + i]);
                }
                tmem_st(t_s + CW * c, p);
            }
            l = fmaf(l, a, unpack2(sum).x + unpack2(sum).y);
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&sm.p_full[s]));
            // the tile before, while this one's product runs; then both in units of the new maximum
            if (j > 0) take(j - 1);
            if (__any_sync(0xffffffffu, a != 1.f)) {
#pragma unroll
                for (int i = 0; i < OD / 2; i++) o[i] = mul2(o[i], pack2(a, a));
            }
        }
        if (alive && nj > 0) take(nj - 1);
        sm.l[half][r] = l;
        bar_sync(1, P_SOFT);
        const float total = sm.l[0][r] + sm.l[1][r], inv = 1.f / total;
        if (alive && row_ok(r)) {
            float *out = A.out + (((int64_t)r_begin + t0 + r / rep) * A.n_heads + kvh * rep + r % rep) * HD + half * OD;
#pragma unroll
            for (int i = 0; i < OD; i += 4) {
                const float2 u = unpack2(o[i / 2]), w = unpack2(o[i / 2 + 1]);
                const bool bad = nan_mine >> ((half * OD + i) / 32) & 1;
                *(float4 *)(out + i) = i_row < 0 || total == 0.f ? make_float4(0.f, 0.f, 0.f, 0.f)
                                       : bad ? make_float4(NAN, NAN, NAN, NAN)
                                             : make_float4(u.x * inv, u.y * inv, w.x * inv, w.y * inv);
            }
        }
    } else if (warp < 12) {
        // ================= cache tiles to operands
        const int w4 = warp - 8;
        const uint32_t magic = KV4_MAGIC + (uint32_t)(A.shift >> 8);   // the shift is at most 10
        constexpr int PIECES = HD / 32, KROWS = 32 / PIECES, KI = PN / (4 * KROWS);
        const int k_piece = lane % PIECES, k_row = w4 * KROWS + lane / PIECES;
        // V: 8 positions x VW words of one 16-byte piece
        constexpr int VW = HD == 128 ? 2 : 1;
        const int vr = w4 * 4 + (lane >> 3), v_atom = vr & 1, v_chunk = (lane & 7) | (v_atom << 3);
        const int v_piece = HD == 32 ? 0 : (vr >> 1) & (PIECES - 1);
        const int v_word = HD == 128 ? 2 * (vr >> 3) : HD == 64 ? vr >> 2 : (vr >> 1) & 3;
        const bool v_on = HD != 32 || vr < 8;
        const uint8_t *raw0 = base + 2 * L::Q + 2 * (L::K + L::V);
        for (int j = 0; j < nj; j++) {
            const int s = j & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.raw_full), j & 1, flag))) break;
            const int pos = sm.pos[j & 7][lane & (PG - 1)];
            // whether every position is seen by some row (else the scales of the others count as 0)
            const bool whole = __all_sync(0xffffffffu, pos + KV4_TILE - 1 <= S.last && (pos >= S.first || pos <= A.sinks - KV4_TILE));
            uint4 kw[KI];
            uint32_t kd[KI], vw[8][VW], vd[8];
#pragma unroll
            for (int i = 0; i < KI; i++) {
                const int row = i * 4 * KROWS + k_row, in = row % KV4_TILE;
                const uint8_t *src = raw0 + row / KV4_TILE * L::RAW1;
                kw[i] = *(const uint4 *)(src + in * (HD / 2) + 16 * k_piece);
                kd[i] = *((const uint16_t *)(src + 16 * HD) + in * PIECES + k_piece);
            }
            {
                const uint8_t *src = raw0 + (v_chunk >> 1) * L::RAW1;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int in = 8 * (v_chunk & 1) + i;
                    const uint32_t *q = (const uint32_t *)(src + 8 * HD + in * (HD / 2) + 16 * v_piece) + v_word;
                    if constexpr (VW == 2) {
                        const uint2 x = *(const uint2 *)q;
                        vw[i][0] = x.x;
                        vw[i][1] = x.y;
                    } else {
                        vw[i][0] = *q;
                    }
                    vd[i] = *((const uint16_t *)(src + 17 * HD) + in * PIECES + v_piece);
                }
            }
            if (!whole) {
#pragma unroll
                for (int i = 0; i < KI; i++) {
                    const int row = i * 4 * KROWS + k_row;
                    if (!S.any(__shfl_sync(0xffffffffu, pos, row / KV4_TILE) + row % KV4_TILE, A.sinks)) kd[i] = 0;
                }
                const int p0 = __shfl_sync(0xffffffffu, pos, v_chunk >> 1) + 8 * (v_chunk & 1);
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (!S.any(p0 + i, A.sinks)) vd[i] = 0;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&sm.raw_free));   // this warp has read the raw tiles
            // K's stage is free once the S that read it is there, V's once the PV is
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.s_full[s]), ((j >> 1) & 1) ^ 1, flag))) break;
            uint8_t *K = base + 2 * L::Q + s * (L::K + L::V), *V = K + L::K;
#pragma unroll
            for (int i = 0; i < KI; i++) {
                const int row = i * 4 * KROWS + k_row;
                const uint32_t d = __byte_perm(kd[i], kd[i], 0x1010);
                const uint32_t w[4] = {kw[i].x, kw[i].y, kw[i].z, kw[i].w};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const uint32_t w8 = w[c] >> 8;
                    const int ch = 4 * k_piece + c;
                    *(uint4 *)(K + (ch >> 3) * (PN * 128) + row * 128 + (((ch & 7) ^ (row & 7)) << 4)) =
                        make_uint4(nib_lo(w[c], d, magic), nib_lo(w8, d, magic), nib_hi(w[c], d, magic), nib_hi(w8, d, magic));
                }
            }
            fence_async_smem();
            mbar_arrive(smem_u32(&sm.k_full[s]));
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.pv_done[s]), ((j >> 1) & 1) ^ 1, flag))) break;
            {
                uint32_t odd = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) odd |= not_finite(vd[i]) ? 1u << i : 0u;
                if (!v_on) odd = 0;
                if (v_on && v_word == 0) sm.nan_bits[j & 3][v_piece][v_chunk] = (uint8_t)odd;   // one lane's per group and 8 positions
                const int any = __any_sync(0xffffffffu, odd);
                if (lane == 0) sm.nan_any[j & 3][w4] = any;
                if (odd) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (odd >> i & 1) vd[i] = 0;
                }
            }
            if (v_on) {
                uint32_t dd[4];
#pragma unroll
                for (int i = 0; i < 4; i++) dd[i] = __byte_perm(vd[2 * i], vd[2 * i + 1], 0x5410);
                const uint32_t chunk = lane & 7;
#pragma unroll
                for (int w = 0; w < VW; w++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {          // bytes 2 h, 2 h + 1 of the word
                        uint32_t x[4], y[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            x[i] = __byte_perm(vw[2 * i][w], vw[2 * i + 1][w], h ? 0x7632 : 0x5410);
                            y[i] = x[i] >> 8;
                        }
                        const uint32_t dim = 32 * v_piece + 4 * (v_word + w) + 2 * h;
                        auto put = [&](uint32_t row, uint4 v) {
                            *(uint4 *)(V + v_atom * (HD * 128) + row * 128 + ((chunk ^ (row & 7)) << 4)) = v;
                        };
                        put(dim, make_uint4(nib_lo(x[0], dd[0], magic), nib_lo(x[1], dd[1], magic), nib_lo(x[2], dd[2], magic), nib_lo(x[3], dd[3], magic)));
                        put(dim + 1, make_uint4(nib_lo(y[0], dd[0], magic), nib_lo(y[1], dd[1], magic), nib_lo(y[2], dd[2], magic), nib_lo(y[3], dd[3], magic)));
                        put(dim + 16, make_uint4(nib_hi(x[0], dd[0], magic), nib_hi(x[1], dd[1], magic), nib_hi(x[2], dd[2], magic), nib_hi(x[3], dd[3], magic)));
                        put(dim + 17, make_uint4(nib_hi(y[0], dd[0], magic), nib_hi(y[1], dd[1], magic), nib_hi(y[2], dd[2], magic), nib_hi(y[3], dd[3], magic)));
                    }
            }
            fence_async_smem();
            mbar_arrive(smem_u32(&sm.v_full[s]));
        }
    } else if (warp == 14) {
        // ================= copies of the cache tiles
        const int page_tiles = 1 << (A.shift - 4);
        const uint32_t raw0 = smem_u32(base + 2 * L::Q + 2 * (L::K + L::V)), bar = smem_u32(&sm.raw_full);
        // lane i < 8: cache tile i of position tile j and the page it lies on, used a position tile later (worked
        // on at once, the load's latency stood in every tile)
        int tile_next, page_next;
        auto look = [&](int j) {
            const int u = PG * j + (lane & 7);
            tile_next = u < S.units ? S.tile(u) : 0;
            page_next = u < S.units ? table[tile_next >> (A.shift - 4)] : -1;
        };
        // where it lies, or -1; and its first position
        auto place = [&](int &pos) {
            const bool there = page_next >= 0 && page_next < A.pages;
            pos = there ? tile_next * KV4_TILE : ABSENT;
            return there ? (int)(((int64_t)page_next * A.n_kv + kvh) * page_tiles + (tile_next & (page_tiles - 1))) : -1;
        };
        look(0);
        int issued = 0;
        for (; issued < nj; issued++) {
            if (issued > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&sm.raw_free), (issued - 1) & 1, flag))) break;
            int pos;
            const int at = place(pos);
            // (the positions of eight tiles ago: the warps that read the raw tiles just now waited for their PV)
            if (lane < PG) sm.pos[issued & 7][lane] = pos;
            __syncwarp();
            const int n = __popc(__ballot_sync(0xffffffffu, lane < PG && at >= 0));
            if (lane == 0)
                asm volatile("{\n .reg .b64 st;\n mbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n}\n" ::"r"(bar),
                             "r"(n * kv4_tile_bytes(HD))
                             : "memory");
            __syncwarp();
            if (lane < PG && at >= 0)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                 raw0 + lane * L::RAW1),
                             "l"(A.cache + (uint64_t)(uint32_t)at * kv4_tile_bytes(HD)), "r"(kv4_tile_bytes(HD)), "r"(bar)
                             : "memory");
            look(issued + 1);
        }
        // the last copy ends before the CTA does, also after a wait that ran out
        if (issued > 0) mbar_wait_quiet(bar, (issued - 1) & 1);
    } else if (lane == 0) {
        // ================= MMAs: warp 12 S, warp 13 PV
        constexpr uint32_t id_s = idesc_f16(PN), id_o = idesc_f16(HD);
        if (warp == 12) {
            const uint64_t qh = sw128_desc(q_hi), ql = sw128_desc(q_lo);
            for (int j = 0; j < nj; j++) {
                const int s = j & 1;
                // the PV that read this buffer's P is done
                if (!mbar_wait(smem_u32(&sm.pv_done[s]), ((j >> 1) & 1) ^ 1, flag) ||
                    !mbar_wait(smem_u32(&sm.k_full[s]), (j >> 1) & 1, flag))
                    break;
                tc_fence_after();
                const uint64_t kd = sw128_desc(kv0 + s * (L::K + L::V));
                const uint32_t d = tmem + S_COL + s * PN;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    const uint32_t off = ((ks >> 2) * (PM * 128) + (ks & 3) * 32) >> 4;   // descriptors count 16 bytes
                    mma_ss(d, qh + off, kd + off, id_s, ks > 0);
                    mma_ss(d, ql + off, kd + off, id_s, 1);
                }
                commit(smem_u32(&sm.s_full[s]));
                mbar_arrive(smem_u32(&sm.s_full[s]));
            }
        } else {
            for (int j = 0; j < nj; j++) {
                const int s = j & 1;
                if (!mbar_wait(smem_u32(&sm.v_full[s]), (j >> 1) & 1, flag) || !mbar_wait(smem_u32(&sm.p_full[s]), (j >> 1) & 1, flag)) break;
                tc_fence_after();
                const uint64_t vdesc = sw128_desc(kv0 + s * (L::K + L::V) + L::K);
                const uint32_t p0 = tmem + S_COL + s * PN, d = tmem + PV_COL + s * HD;
#pragma unroll
                for (int ks = 0; ks < PN / 16; ks++) {
                    const uint64_t bd = vdesc + (((ks >> 2) * (HD * 128) + (ks & 3) * 32) >> 4);
                    const uint32_t a = p0 + (CW == 32 ? 32 * (ks >> 1) + 8 * (ks & 1) : 16 * ks);
                    mma_ts(d, a, bd, id_o, ks > 0);
                    mma_ts(d, a + CW / 2, bd, id_o, 1);
                }
                commit(smem_u32(&sm.pv_done[s]));
                mbar_arrive(smem_u32(&sm.pv_done[s]));         // (hands on the bit masks of the unpacking warps)
            }
        }
        // what was issued ends before tensor memory is freed, also after a wait that ran out
        commit(smem_u32(&sm.fin[warp - 12]));
        mbar_wait_quiet(smem_u32(&sm.fin[warp - 12]), 0);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

template <int HD>
cudaError_t launch(hd_ctx *ctx, const Kv4Args &A) {
    constexpr size_t smem = PLayout<HD>::BYTES;
    static std::atomic<uint64_t> allowed{0};
    cudaError_t e = hd_allow_smem(allowed, ctx, (const void *)k_kv4_prefill<HD>, smem);
    if (e != cudaSuccess) return e;
    const int rep = A.n_heads / A.n_kv, tq = PM / rep;
    // a request's last tile may be short: at most one more tile each, and no more than rows
    int64_t tiles = A.rows / tq + A.seqs;
    tiles = tiles < A.rows ? tiles : A.rows;
    return hd_launch(ctx, k_kv4_prefill<HD>, dim3((unsigned)(tiles * A.n_kv)), dim3(P_THREADS), smem, A, tq, ctx->flag);
}

}  // namespace

extern "C" int hd_kv4_attention_prefill(hd_ctx *ctx, const float *q, int64_t q_ld, const uint8_t *cache, int64_t pages,
                                        int page_size, const int32_t *tables, int max_pages, const int32_t *lens,
                                        const int32_t *row0, int seqs, int64_t rows, int n_heads, int n_kv, int head_dim,
                                        int window, int sinks, float scale, float *out) {
    Kv4Args A{q, q_ld, cache, pages, 0, tables, max_pages, lens, row0, seqs, rows, n_heads, n_kv, window, sinks, scale, out};
    if (seqs > 0 && !row0) return hd_fail(ctx, HD_E_ARG, "hd_kv4_attention_prefill: null argument");
    int rc = hd_kv4_attention_check(ctx, "hd_kv4_attention_prefill", A, page_size, head_dim);
    if (rc || seqs == 0 || rows == 0) return rc;
    HD_REQUIRE(ctx, (rows + seqs) * n_kv < ((int64_t)1 << 31), HD_E_SHAPE, "hd_kv4_attention_prefill: %lld rows of %d kv heads",
               (long long)rows, n_kv);
    HdDevice on(ctx);
    cudaError_t e = head_dim == 128 ? launch<128>(ctx, A) : head_dim == 64 ? launch<64>(ctx, A) : launch<32>(ctx, A);
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "hd_kv4_attention_prefill: %s", cudaGetErrorString(e));
    return HD_OK;
}
