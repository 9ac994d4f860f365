// hd_sample_filtered.cu -- one index per row from given random numbers, after
// temperature, top-k, top-p and min-p with each row's own settings.
//
// With m the row's largest logit and w_i = exp((x_i - m) / T):
//   top-k   the k largest logits stay (equal ones: the lowest index first);
//   top-p   of those in descending order the shortest prefix whose mass is at
//           least p times theirs;
//   min-p   of those the ones with w_i >= min_p;
// and the draw is the first index, in the vocabulary's order, at which the
// running sum of the kept weights exceeds u times their sum.
//
// All three filters keep a prefix of the descending order, so a row's kept
// set is "key above tau, or one of the first c elements equal to tau", found
// without a sort.  A row lies in the shared memory of a thread-block cluster
// (read from memory once); a histogram over -log2 of the weight, 64 bins to a
// factor of two, finds the bin in which the running count (top-k) or mass
// (top-p) reaches its goal, and the few elements of that bin are compared with
// one another.  More elements than CAP in a bin (many equal logits) are split
// again by the bits of an order-preserving integer key.  Min-p is a smallest
// key, found by search.  The draw adds up contiguous parts per CTA and per
// warp and follows the target down.
//
// Weights are computed in 64 bits (2^y = 2^(j/64) 2^e 2^r with a table of 64
// and a polynomial of degree 5 in r, |r| <= 1/128: the table-driven method of
// P. T. P. Tang, ACM TOMS 15 (1989), error below 2^-50) and held as whole
// numbers of 2^-s, s = min(50, 62 - ceil(log2 n)): sums are exact in any order,
// so neither atomics nor the shape of the cluster can change a draw, and a
// weight's rounding (2^-45 of the largest for a vocabulary of 152k) is far
// below what float32 sums lose.
#include <cooperative_groups.h>

#include <cmath>

#include "hd_internal.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int FNT = 512, FW = FNT / 32;
constexpr int FBINS = 2048, FGROUP = 32, FGROUPS = FBINS / FGROUP;
constexpr int CAP = 512;                     // elements compared with one another
constexpr int MAXC = 16;                     // CTAs per row
constexpr uint32_t KEY_NINF = 0x007fffffu;   // key of -infinity

// Larger float, larger key; NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return KEY_NINF;
    const uint32_t b = __float_as_uint(__fadd_rn(x, 0.f));
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

struct FShared {
    uint32_t lo[FBINS], hi[FBINS];           // the slice's histogram, 64 bits in two halves
    long long group[FGROUPS];                // its sums over groups of bins
    long long total[FGROUPS];                // the row's
    double table[64];                        // 2^(j / 64)
    uint32_t list[CAP], all[CAP + 1];        // the slice's elements of a bin; the row's
    long long weight[CAP + 1];
    long long wsum[FW], before;              // warps' sums of the draw
    int wtie[FW], tie_before, found;
    uint32_t n_list, lo_key, hi_key;         // of the bin's elements: number, smallest and largest key
    // what other CTAs of the cluster read
    uint32_t kmax;
    long long mass;
    int ties;
    // broadcasts within the CTA
    uint32_t pick;
    long long pick_above;
};

struct Row {
    const float *x;       // the slice
    int n;                // its length
    double m, a;          // largest logit, log2(e) / temperature
    uint32_t kmax;
    int bits;             // units per weight 1: 2^bits
    const double *table;
    __device__ __forceinline__ double log2w(float x) const { return ((double)x - m) * a; }
    // -64 log2(weight), rounded: the bin of the first histogram
    __device__ __forceinline__ int bin(uint32_t key, float x) const {
        if (key == kmax) return 0;
        const double y = log2w(x);
        return y >= -31.9 ? -__double2loint(y + 0x1.8p46) : FBINS - 1;
    }
    __device__ __forceinline__ double weight(uint32_t key, float x) const {
        if (key == kmax) return 1.0;
        const double y = log2w(x);
        if (!(y >= -64.0)) return 0.0;       // below half a unit; (-inf) * 0
        const double k = y + 0x1.8p46;       // y rounded to a multiple of 1 / 64
        const int ki = __double2loint(k);
        const double r = y - (k - 0x1.8p46);
        // 2^r - 1 = sum (r ln 2)^i / i!
        double p = 0x1.5d87fe78a6730p-10;
        p = fma(p, r, 0x1.3b2ab6fba4e77p-7);
        p = fma(p, r, 0x1.c6b08d704a0bfp-5);
        p = fma(p, r, 0x1.ebfbdff82c58ep-3);
        p = fma(p, r, 0x1.62e42fefa39efp-1);
        p *= r;
        const double t = table[ki & 63], w = fma(t, p, t);
        return __hiloint2double(__double2hiint(w) + ((ki >> 6) << 20), __double2loint(w));
    }
    __device__ __forceinline__ long long units(double w) const {
        // w 2^bits <= 2^50: adding 1.5 * 2^52 leaves the rounded integer in the low bits
        const double v = w == 0.0 ? 0.0 : __hiloint2double(__double2hiint(w) + (bits << 20), __double2loint(w));
        return __double_as_longlong(v + 0x1.8p52) - 0x4338000000000000ll;
    }
};

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ long long warp_scan(long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, v, o);
        if ((int)(threadIdx.x & 31) >= o) v += x;
    }
    return v;
}

// The key tau at which the running weight of the elements above `floor_key`
// (and of floor_ties of those equal to it), from the largest down, reaches its
// goal: `goal` of them, or (MASS) the share p of their units.  `above`: the
// weight of the elements > tau.  Every CTA of the cluster gets the same.
template <bool MASS>
__device__ uint32_t select(const Row &R, FShared &sm, uint32_t floor_key, long long floor_ties, double p, long long &goal,
                           long long &above) {
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned C = cluster.num_blocks();
    const long long floor_w = floor_ties > 0 ? floor_ties * (MASS ? R.units(R.weight(floor_key, key_value(floor_key))) : 1) : 0;
    uint32_t lo_key = 0, hi_key = 0xffffffffu;
    int shift = -1;                          // -1: bins of the weight; else of the key, from hi_key down
    above = 0;
    for (;;) {
        auto bin_of = [&](uint32_t key, float x) { return shift < 0 ? R.bin(key, x) : (int)((hi_key - key) >> shift); };
        for (int b = tid; b < FBINS; b += FNT) sm.lo[b] = sm.hi[b] = 0;
        if (tid == 0) {
            sm.n_list = 0;
            sm.lo_key = 0xffffffffu;
            sm.hi_key = 0;
        }
        __syncthreads();
#pragma unroll 2
        for (int i = tid; i < R.n; i += FNT) {
            const float x = R.x[i];
            const uint32_t key = order_key(x);
            if (key <= floor_key || key < lo_key || key > hi_key) continue;
            const int b = bin_of(key, x);
            if (MASS) {
                const unsigned long long w = (unsigned long long)R.units(R.weight(key, x));
                const uint32_t wl = (uint32_t)w, old = atomicAdd(&sm.lo[b], wl);
                const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old ? 1u : 0u);
                if (wh) atomicAdd(&sm.hi[b], wh);
            } else {
                atomicAdd(&sm.lo[b], 1u);
            }
        }
        __syncthreads();
        for (int q = warp; q < FGROUPS; q += FW) {
            const int b = q * FGROUP + lane;
            const long long s = warp_sum((long long)(((unsigned long long)sm.hi[b] << 32) | sm.lo[b]));
            if (lane == 0) sm.group[q] = s;
        }
        cluster.sync();
        const bool floor_in = floor_w > 0 && (shift < 0 || (floor_key >= lo_key && floor_key <= hi_key));
        const int floor_bin = floor_in ? bin_of(floor_key, key_value(floor_key)) : -1;
        if (tid < FGROUPS) {
            long long t = floor_in && floor_bin / FGROUP == tid ? floor_w : 0;
            for (unsigned r = 0; r < C; r++) t += cluster.map_shared_rank(&sm, r)->group[tid];
            sm.total[tid] = t;
        }
        __syncthreads();
        if (warp == 0) {
            const long long t0 = sm.total[2 * lane], t1 = sm.total[2 * lane + 1];
            const long long inc = warp_scan(t0 + t1);
            if (MASS && shift < 0) {
                const long long mass = __shfl_sync(0xffffffffu, inc, 31);
                goal = __double2ll_ru(p * (double)mass);
                goal = goal < 1 ? 1 : goal > mass ? mass : goal;
            }
            const long long b0 = above + inc - t0 - t1, b1 = b0 + t0, b2 = b1 + t1;
            const bool mine = b0 < goal && b2 >= goal;
            const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
            const int q = __shfl_sync(0xffffffffu, b1 >= goal ? 2 * lane : 2 * lane + 1, src);
            const long long base = __shfl_sync(0xffffffffu, b1 >= goal ? b0 : b1, src);
            long long v = floor_in && floor_bin == q * FGROUP + lane ? floor_w : 0;
            for (unsigned r = 0; r < C; r++) {
                const FShared *o = cluster.map_shared_rank(&sm, r);
                const int b = q * FGROUP + lane;
                v += (long long)(((unsigned long long)o->hi[b] << 32) | o->lo[b]);
            }
            const long long run = base + warp_scan(v);
            const int first = __ffs(__ballot_sync(0xffffffffu, run >= goal)) - 1;
            if (lane == first) {
                sm.pick = (uint32_t)(q * FGROUP + lane);
                sm.pick_above = run - v;
            }
            if (lane == 0) sm.before = goal;
        }
        __syncthreads();
        const int pick = (int)sm.pick;
        above = sm.pick_above;
        goal = sm.before;
        // the elements of that bin
        for (int i = tid; i < R.n; i += FNT) {
            const float x = R.x[i];
            const uint32_t key = order_key(x);
            if (key <= floor_key || key < lo_key || key > hi_key || bin_of(key, x) != pick) continue;
            const uint32_t at = atomicAdd(&sm.n_list, 1u);
            if (at < CAP) sm.list[at] = key;
            atomicMin(&sm.lo_key, key);
            atomicMax(&sm.hi_key, key);
        }
        cluster.sync();
        uint32_t count = 0, start[MAXC];
        uint32_t kl = 0xffffffffu, kh = 0;
#pragma unroll
        for (unsigned r = 0; r < MAXC; r++) {
            start[r] = count;
            if (r < C) {
                const FShared *o = cluster.map_shared_rank(&sm, r);
                count += o->n_list;
                kl = min(kl, o->lo_key);
                kh = max(kh, o->hi_key);
            }
        }
        if (floor_bin == pick) {             // below every other element of the bin
            kl = floor_key;
            if (count == 0) kh = floor_key;
        }
        if (kl == kh) {                      // one key: no other to compare with
            cluster.sync();
            return kl;
        }
        if (count <= CAP) {
#pragma unroll
            for (unsigned r = 0; r < MAXC; r++) {
                if (r >= C) continue;
                const FShared *o = cluster.map_shared_rank(&sm, r);
                for (uint32_t i = tid; i < o->n_list; i += FNT) {
                    const uint32_t key = o->list[i];
                    sm.all[start[r] + i] = key;
                    sm.weight[start[r] + i] = MASS ? R.units(R.weight(key, key_value(key))) : 1;
                }
            }
            const int L = (int)count + (floor_bin == pick ? 1 : 0);
            if (floor_bin == pick && tid == 0) {
                sm.all[count] = floor_key;
                sm.weight[count] = floor_w;
            }
            __syncthreads();
            for (int i = tid; i < L; i += FNT) {
                const uint32_t key = sm.all[i];
                long long over = above, with = 0;
                for (int j = 0; j < L; j++) {
                    const uint32_t kj = sm.all[j];
                    const long long w = sm.weight[j];
                    over += kj > key ? w : 0;
                    with += kj == key ? w : 0;
                }
                if (over < goal && over + with >= goal) {   // equal elements write the same
                    sm.pick = key;
                    sm.pick_above = over;
                }
            }
            cluster.sync();                  // others may still read this CTA's list
            above = sm.pick_above;
            return sm.pick;
        }
        lo_key = kl;
        hi_key = kh;
        shift = 0;
        while ((hi_key - lo_key) >> shift >= FBINS) shift++;
        cluster.sync();                      // before the histogram and the list are written again
    }
}

template <bool RESIDENT>
__global__ void __launch_bounds__(FNT, 2) k_sample_filtered(const float *__restrict__ logits, int64_t ld, int64_t n,
                                                         const float *__restrict__ temp, const int32_t *__restrict__ top_k,
                                                         const float *__restrict__ top_p, const float *__restrict__ min_p,
                                                         const float *__restrict__ uni, int64_t slice, int bits,
                                                         int32_t *__restrict__ out) {
    extern __shared__ __align__(16) uint8_t raw[];
    FShared &sm = *reinterpret_cast<FShared *>(raw);
    float *xs = reinterpret_cast<float *>(raw + sizeof(FShared));
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), C = cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / C, begin = min(n, rank * slice), end = min(n, begin + slice);
    const float *x = logits + r * ld + begin;
    Row R;
    R.n = (int)(end - begin);
    if (tid < 64) sm.table[tid] = exp2((double)tid / 64);
    if (tid == 0) sm.kmax = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    uint32_t km = 0;
#pragma unroll 8
    for (int i = tid; i < R.n; i += FNT) {
        const float v = x[i];
        km = max(km, order_key(v));
        if (RESIDENT) xs[i] = v;
    }
    R.x = RESIDENT ? xs : x;
    km = __reduce_max_sync(0xffffffffu, km);
    if (lane == 0) atomicMax(&sm.kmax, km);
    cluster.sync();
    R.kmax = 0;
    for (unsigned c = 0; c < C; c++) R.kmax = max(R.kmax, cluster.map_shared_rank(&sm, c)->kmax);
    const float T = temp ? temp[r] : 1.f, u = uni[r];
    int64_t k = top_k ? top_k[r] : 0;
    float p = top_p ? top_p[r] : 1.f;
    double mp = min_p ? (double)min_p[r] : 0.0;
    if (k <= 0 || k > n) k = n;
    if (p != p) p = 1.f;
    if (!(T > 0.f) || p <= 0.f) k = 1;
    mp = mp > 0.0 ? fmin(mp, 1.0) : 0.0;
    R.m = (double)key_value(R.kmax);
    R.a = 1.4426950408889634 / (double)T;
    R.bits = bits;
    R.table = sm.table;
    // tau, and how many of the elements equal to it stay
    uint32_t tau = 0;
    long long ties = 0, above, goal;
    const bool none = R.kmax == KEY_NINF;
    if (!none) {
        if (k == 1) {
            tau = R.kmax;
            ties = 1;
        } else {
            if (k < n) {
                goal = k;
                tau = select<false>(R, sm, 0, 0, 0.0, goal, above);
                ties = k - above;
            }
            if (p < 1.f) {
                tau = select<true>(R, sm, tau, ties, (double)p, goal, above);
                const long long w = R.units(R.weight(tau, key_value(tau)));
                ties = (goal - above + w - 1) / w;
            }
            if (mp > 0.0) {
                // the smallest key with weight >= min_p: 32 candidates at a time (the weight does not fall with the key)
                uint32_t lo = KEY_NINF, hi = R.kmax;      // weight(lo) < mp <= weight(hi)
                while (hi - lo > 1) {
                    const uint32_t step = (hi - lo + 32) / 33, c = (uint64_t)lo + (uint64_t)step * (lane + 1) < hi ? lo + step * (lane + 1) : hi;
                    const uint32_t ok = __ballot_sync(0xffffffffu, R.weight(c, key_value(c)) >= mp);
                    const int f = __ffs(ok) - 1;          // lane 31's candidate may fall short of hi
                    const uint32_t top = f < 0 ? hi : __shfl_sync(0xffffffffu, c, f);
                    const uint32_t bot = f == 0 ? lo : __shfl_sync(0xffffffffu, c, f < 0 ? 31 : f - 1);
                    hi = top;
                    lo = bot;
                }
                if (hi > tau) {
                    tau = hi;
                    ties = n;
                }
            }
        }
    }
    // ---- the draw
    const double wt = tau ? R.weight(tau, key_value(tau)) : 0.0;
    const long long wtau = R.units(wt);
    auto part = [&](int b, int e, long long &mass, int &tie) {   // a warp's elements b .. e - 1
        mass = 0;
        tie = 0;
#pragma unroll 2
        for (int i = b + lane; i < e; i += 32) {
            const float v = R.x[i];
            const uint32_t key = order_key(v);
            if (key > tau) mass += R.units(R.weight(key, v));
            tie += key == tau;
        }
        mass = warp_sum(mass);
        tie = __reduce_add_sync(0xffffffffu, tie);
    };
    const int chunk = (R.n + FW - 1) / FW;
    if (!none) {
        long long mass;
        int tie;
        part(min(R.n, warp * chunk), min(R.n, (warp + 1) * chunk), mass, tie);
        if (lane == 0) {
            sm.wsum[warp] = mass;
            sm.wtie[warp] = tie;
        }
    }
    __syncthreads();
    if (tid == 0) {
        long long mass = 0;
        int tie = 0;
        for (int w = 0; w < FW && !none; w++) {
            mass += sm.wsum[w];
            tie += sm.wtie[w];
        }
        sm.mass = mass;
        sm.ties = tie;
    }
    cluster.sync();
    // every CTA adds up the cluster; the one that holds the target goes on
    long long total = 0, mine = 0, my_mass = 0;
    long long tie_at = 0, my_tie = 0;
    for (unsigned c = 0; c < C; c++) {
        const FShared *o = cluster.map_shared_rank(&sm, c);
        if (c == rank) {
            mine = total;
            my_tie = tie_at;
        }
        const long long stay = max(0ll, min((long long)o->ties, ties - tie_at));
        const long long kept = o->mass + stay * wtau;
        if (c == rank) my_mass = kept;
        total += kept;
        tie_at += o->ties;
    }
    cluster.sync();                          // no CTA leaves while another reads it
    if (none) {
        if (rank == 0 && tid == 0) out[r] = -1;
        return;
    }
    long long target = (long long)((double)(u > 0.f ? u : 0.f) * (double)total);
    target = target > total - 1 ? total - 1 : target;
    if (!(mine <= target && target < mine + my_mass)) return;
    // from the CTA's slice to a warp's part of it, to a sixteenth of that, to the element
    int b = 0, len = R.n, step = chunk;
    for (int level = 0; level < 2; level++) {
        if (level) {
            long long mass;
            int tie;
            part(min(b + len, b + warp * step), min(b + len, b + (warp + 1) * step), mass, tie);
            if (lane == 0) {
                sm.wsum[warp] = mass;
                sm.wtie[warp] = tie;
            }
            __syncthreads();
        }
        if (tid == 0) {
            long long at = mine, t = my_tie;
            for (int w = 0; w < FW; w++) {
                const long long kept = sm.wsum[w] + max(0ll, min((long long)sm.wtie[w], ties - t)) * wtau;
                if (target < at + kept) {
                    sm.found = w;
                    sm.before = at;
                    sm.mass = t;
                    break;
                }
                at += kept;
                t += sm.wtie[w];
            }
        }
        __syncthreads();
        mine = sm.before;
        my_tie = sm.mass;
        const int e = min(b + len, b + (sm.found + 1) * step);
        b += sm.found * step;
        len = e - b;
        step = (len + FW - 1) / FW;
        __syncthreads();
    }
    if (warp != 0) return;
    for (int i0 = b; i0 < b + len; i0 += 32) {
        const int i = i0 + lane;
        const float v = i < b + len ? R.x[i] : 0.f;
        const uint32_t key = i < b + len ? order_key(v) : 0;
        const uint32_t eq = __ballot_sync(0xffffffffu, i < b + len && key == tau);
        long long w = 0;
        if (i < b + len) {
            if (key > tau) w = R.units(R.weight(key, v));
            else if (key == tau && my_tie + __popc(eq & ((1u << lane) - 1u)) < ties) w = wtau;
        }
        const long long run = mine + warp_scan(w);
        const uint32_t over = __ballot_sync(0xffffffffu, run > target);
        if (over) {
            if (lane == __ffs(over) - 1) out[r] = (int32_t)(begin + i);
            return;
        }
        mine = __shfl_sync(0xffffffffu, run, 31);
        my_tie += __popc(eq);
    }
}

template <bool RESIDENT>
cudaError_t launch(hd_ctx *ctx, int C, int64_t rows, int64_t slice, const float *logits, int64_t ld, int64_t n,
                   const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                   int bits, int32_t *idx) {
    const size_t smem = sizeof(FShared) + (RESIDENT ? (size_t)slice * sizeof(float) : 0);
    cudaError_t e = cudaFuncSetAttribute(k_sample_filtered<RESIDENT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && C > 8)
        e = cudaFuncSetAttribute(k_sample_filtered<RESIDENT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    return hd_launch_cluster(ctx, k_sample_filtered<RESIDENT>, dim3((unsigned)(rows * C)), dim3(FNT), smem, C, logits, ld, n,
                             temperature, top_k, top_p, min_p, u, slice, bits, idx);
}

}  // namespace

extern "C" int hd_sample_filtered(hd_ctx *ctx, const float *logits, int64_t ld, int64_t rows, int64_t n,
                                  const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                                  const float *u, int32_t *idx) {
    if ((rows > 0 && (!logits || !u || !idx))) return hd_fail(ctx, HD_E_ARG, "hd_sample_filtered: null argument");
    if (ld == 0) ld = n;
    HD_REQUIRE(ctx, rows >= 0 && rows < ((int64_t)1 << 27) && n > 0 && n < ((int64_t)1 << 31) && ld >= n, HD_E_SHAPE,
               "hd_sample_filtered: bad shape (rows %lld, n %lld, row stride %lld)", (long long)rows, (long long)n,
               (long long)ld);
    if (!ctx) return HD_E_ARG;
    if (rows == 0) return HD_OK;
    HdDevice on(ctx);
    int bits = 0;
    while (((int64_t)1 << bits) < n) bits++;
    bits = 62 - bits < 50 ? 62 - bits : 50;
    // CTAs per row: as few as keep a slice at 80 KB, so that two CTAs share an SM; more while the rows
    // alone leave SMs idle and a slice keeps 2048 elements
    constexpr int64_t HALF = 20480, FULL = 49152;
    auto slice_of = [&](int c) { return ((n + c - 1) / c + 3) / 4 * 4; };
    int C = 1;
    while (C < MAXC && (slice_of(C) > HALF || (rows * C < ctx->sm_count && slice_of(C) > 4096))) C *= 2;
    const int64_t slice = slice_of(C);
    cudaError_t e = slice <= FULL
                        ? launch<true>(ctx, C, rows, slice, logits, ld, n, temperature, top_k, top_p, min_p, u, bits, idx)
                        : launch<false>(ctx, C, rows, slice, logits, ld, n, temperature, top_k, top_p, min_p, u, bits, idx);
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "hd_sample_filtered: %s", cudaGetErrorString(e));
    return HD_OK;
}
