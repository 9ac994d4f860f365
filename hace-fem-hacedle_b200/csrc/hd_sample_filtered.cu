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

constexpr int FBINS = 2048, FGROUP = 32, FGROUPS = FBINS / FGROUP;
constexpr int CAP = 512;                     // elements compared with one another
constexpr int MAXC = 16;                     // CTAs per row
constexpr int MAXW = 32;                     // warps per CTA
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
    long long wsum[MAXW];                    // warps' sums
    int wtie[MAXW];
    uint32_t n_list, kmax;                   // what other CTAs of the cluster read ..
    long long mass;
    int ties;
    uint32_t pick;                           // .. and write
    long long pick_above;
    int bin;                                 // broadcasts within the CTA
    long long bin_above, goal, before, tie_before;
    uint32_t bound[2];
    int found;
};

struct Row {
    const float *x;       // the slice
    const uint4 *keys;    // its keys, where it is resident; padded with 0
    int n, n4;            // its length; in fours
    double m, a;          // largest logit, log2(e) / temperature
    uint32_t kmax;
    int bits;             // units per weight 1: 2^bits
    const double *table;
    template <bool RESIDENT>
    __device__ __forceinline__ uint4 four(int i) const {
        if (RESIDENT) return keys[i];
        auto key = [&](int j) { return j < n ? order_key(x[j]) : 0u; };
        return make_uint4(key(4 * i), key(4 * i + 1), key(4 * i + 2), key(4 * i + 3));
    }
    template <bool RESIDENT>
    __device__ __forceinline__ uint32_t one(int i) const {
        return RESIDENT ? ((const uint32_t *)keys)[i] : order_key(x[i]);
    }
    // log2 of the weight, rounded to a multiple of 1 / 64 (`k`: 1.5 * 2^46 above it)
    __device__ __forceinline__ double log2w(uint32_t key, double &k) const {
        const double y = ((double)key_value(key) - m) * a;
        k = y + 0x1.8p46;
        return y;
    }
    // The bin of the first histogram: -64 log2(weight).
    __device__ __forceinline__ static int bin(bool largest, double y, double k) {
        return largest ? 0 : y >= -31.9 ? -__double2loint(k) : FBINS - 1;
    }
    __device__ __forceinline__ int bin(uint32_t key) const {
        double k;
        const double y = log2w(key, k);
        return bin(key == kmax, y, k);
    }
    __device__ __forceinline__ double weight(bool largest, double y, double k) const {
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
        const double v = __hiloint2double(__double2hiint(w) + ((ki >> 6) << 20), __double2loint(w));
        // below half a unit, or (-inf) * 0: nothing
        return largest ? 1.0 : y >= -64.0 ? v : 0.0;
    }
    __device__ __forceinline__ double weight(uint32_t key) const {
        double k;
        const double y = log2w(key, k);
        return weight(key == kmax, y, k);
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

// f(rank) summed over the cluster, every load in flight at once.
template <typename F>
__device__ __forceinline__ long long cluster_sum(unsigned C, F f) {
    long long v = 0;
#pragma unroll
    for (unsigned r = 0; r < MAXC; r++) {
        const long long x = f(r < C ? r : 0);
        v += r < C ? x : 0;
    }
    return v;
}

// The largest key <= top for which `low` holds, by a warp; it holds for
// KEY_NINF, not for top, and for all keys below one for which it holds.
template <typename F>
__device__ uint32_t last_key(uint32_t top, F low) {
    const int lane = threadIdx.x & 31;
    uint32_t lo = KEY_NINF, hi = top;
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 32) / 33;
        const uint64_t c64 = (uint64_t)lo + (uint64_t)step * (lane + 1);
        const uint32_t c = c64 < hi ? (uint32_t)c64 : hi;
        const uint32_t high = ~__ballot_sync(0xffffffffu, c < hi && low(c));
        const int f = __ffs(high) - 1;       // the first candidate beyond; none: all 32 are low
        const uint32_t at = __shfl_sync(0xffffffffu, c, f < 0 ? 31 : f), under = __shfl_sync(0xffffffffu, c, f <= 0 ? 0 : f - 1);
        lo = f < 0 ? at : f == 0 ? lo : under;
        hi = f < 0 ? hi : at;
    }
    return lo;
}

// The key tau at which the running weight of the elements above `floor_key`
// (and of floor_ties of those equal to it), from the largest down, reaches its
// goal: `goal` of them, or (MASS) the share p of their units.  `above`: the
// weight of the elements > tau.  Every CTA of the cluster gets the same.
// `own` becomes the slice's own weight above tau and its elements equal to it
// where the histogram tells (MASS, one level), and -1 elsewhere.
template <int NT, bool RESIDENT, bool MASS>
__device__ uint32_t select(const Row &R, FShared &sm, uint32_t floor_key, long long floor_ties, double p, long long &goal,
                           long long &above, long long &own, int &own_ties) {
    constexpr int NW = NT / 32;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const long long floor_w = floor_ties > 0 ? floor_ties * (MASS ? R.units(R.weight(floor_key)) : 1) : 0;
    uint32_t lo_key = floor_key + 1, hi_key = R.kmax;   // the elements in question; the floor's own come on top
    bool with_floor = floor_w > 0;
    int shift = -1;                          // -1: bins of the weight; else of the key, from hi_key down
    above = 0;
    own = -1;
    own_ties = 0;
    for (;;) {
        for (int b = tid; b < FBINS; b += NT) sm.lo[b] = sm.hi[b] = 0;
        if (tid == 0) sm.n_list = 0;
        __syncthreads();
        auto count = [&](uint32_t key) {
            if (key < lo_key || key > hi_key) return;
            double k, y;
            int b;
            if (shift < 0) {
                y = R.log2w(key, k);
                b = Row::bin(key == R.kmax, y, k);
            } else {
                b = (int)((hi_key - key) >> shift);
                if (MASS) y = R.log2w(key, k);
            }
            if (MASS) {
                const unsigned long long w = (unsigned long long)R.units(R.weight(key == R.kmax, y, k));
                const uint32_t wl = (uint32_t)w, old = atomicAdd(&sm.lo[b], wl);
                const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old ? 1u : 0u);
                if (wh) atomicAdd(&sm.hi[b], wh);
            } else {
                atomicAdd(&sm.lo[b], 1u);
            }
        };
        for (int i = tid; i < R.n4; i += NT) {
            const uint4 k = R.four<RESIDENT>(i);
            count(k.x);
            count(k.y);
            count(k.z);
            count(k.w);
        }
        __syncthreads();
        // groups of 32 bins: eight threads a group
        for (int q = tid / 8; q < FGROUPS; q += NT / 8) {
            unsigned long long s = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int b = q * FGROUP + 4 * (tid & 7) + i;
                s += ((unsigned long long)sm.hi[b] << 32) | sm.lo[b];
            }
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if ((tid & 7) == 0) sm.group[q] = (long long)s;
        }
        cluster.sync();
        const int floor_bin = !with_floor ? -1 : shift < 0 ? R.bin(floor_key) : (int)((hi_key - floor_key) >> shift);
        if (tid < FGROUPS)
            sm.total[tid] = (floor_bin >= 0 && floor_bin / FGROUP == tid ? floor_w : 0) +
                            cluster_sum(C, [&](unsigned r) { return cluster.map_shared_rank(&sm, r)->group[tid]; });
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
            const int b = q * FGROUP + lane;
            const long long v = (floor_bin == b ? floor_w : 0) + cluster_sum(C, [&](unsigned r) {
                                    const FShared *o = cluster.map_shared_rank(&sm, r);
                                    return (long long)(((unsigned long long)o->hi[b] << 32) | o->lo[b]);
                                });
            const long long run = base + warp_scan(v);
            const int first = __ffs(__ballot_sync(0xffffffffu, run >= goal)) - 1;
            if (lane == first) {
                sm.bin = b;
                sm.bin_above = run - v;
            }
            if (lane == 0) sm.goal = goal;
        }
        __syncthreads();
        const int pick = sm.bin;
        above = sm.bin_above;
        goal = sm.goal;
        // the bin's keys
        uint32_t kl, kh;
        if (shift < 0) {
            if (warp < 2) {
                const int v = pick + warp;   // the largest key of a bin >= v
                const uint32_t k = v == 0 ? R.kmax : v >= FBINS ? KEY_NINF - 1 : last_key(R.kmax, [&](uint32_t c) { return R.bin(c) >= v; });
                if (lane == 0) sm.bound[warp] = k;
            }
            __syncthreads();
            kl = max(lo_key, sm.bound[1] + 1);
            kh = sm.bound[0];
        } else {
            kh = hi_key - ((uint32_t)pick << shift);
            const uint32_t width = (1u << shift) - 1;
            kl = kh - lo_key < width ? lo_key : kh - width;
        }
        if (floor_bin == pick) kl = floor_key;           // with the floor's own below the others
        with_floor = floor_bin == pick;
        if (kl == kh) {
            cluster.sync();                  // before the histogram is written again
            return kl;
        }
        const uint32_t kl_list = with_floor ? floor_key + 1 : kl;
        auto put = [&](uint32_t key) {
            if (key < kl_list || key > kh) return;
            const uint32_t at = atomicAdd(&sm.n_list, 1u);
            if (at < CAP) sm.list[at] = key;
        };
        for (int i = tid; i < R.n4; i += NT) {
            const uint4 k = R.four<RESIDENT>(i);
            put(k.x);
            put(k.y);
            put(k.z);
            put(k.w);
        }
        cluster.sync();
        uint32_t number[MAXC], all = 0;
#pragma unroll
        for (unsigned r = 0; r < MAXC; r++) number[r] = cluster.map_shared_rank(&sm, r < C ? r : 0)->n_list;
#pragma unroll
        for (unsigned r = 0; r < MAXC; r++) all += r < C ? number[r] : 0;
        if (all <= CAP) {
            // a warp per CTA's list
            uint32_t start = 0;
#pragma unroll
            for (unsigned r = 0; r < MAXC; r++) {
                if (r < C && (int)(r % NW) == warp) {
                    const FShared *o = cluster.map_shared_rank(&sm, r);
                    for (uint32_t i = lane; i < number[r]; i += 32) sm.all[start + i] = o->list[i];
                }
                start += r < C ? number[r] : 0;
            }
            if (with_floor && tid == 0) sm.all[all] = floor_key;
            const int L = (int)all + (with_floor ? 1 : 0);
            __syncthreads();
            for (int i = tid; i < L; i += NT)
                sm.weight[i] = i == (int)all ? floor_w : MASS ? R.units(R.weight(sm.all[i])) : 1;
            __syncthreads();
            // every CTA compares its share of the elements with all of them, half a warp an element
            for (int i0 = (int)rank; i0 < L; i0 += (int)C * (NT / 16)) {
                const int i = i0 + (int)C * (tid / 16);
                const uint32_t key = sm.all[min(i, L - 1)];
                long long over = 0, with = 0;
                for (int j = lane & 15; j < L; j += 16) {
                    const uint32_t kj = sm.all[j];
                    const long long w = sm.weight[j];
                    over += kj > key ? w : 0;
                    with += kj == key ? w : 0;
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) {
                    over += __shfl_xor_sync(0xffffffffu, over, o);
                    with += __shfl_xor_sync(0xffffffffu, with, o);
                }
                over += above;
                // equal elements write the same; one lane a CTA of the cluster
                if (i < L && over < goal && over + with >= goal && (unsigned)(lane & 15) < C) {
                    FShared *o = cluster.map_shared_rank(&sm, lane & 15);
                    o->pick = key;
                    o->pick_above = over;
                }
            }
            cluster.sync();                  // pick is there, and no list is read any more
            const uint32_t tau = sm.pick;
            above = sm.pick_above;
            if (MASS && shift < 0) {
                // this slice above tau: its bins before the threshold's, and what the list adds
                long long mass = 0;
                for (int b = tid; b < pick; b += NT) mass += (long long)(((unsigned long long)sm.hi[b] << 32) | sm.lo[b]);
                int tie = 0;
                for (int i = tid; i < (int)sm.n_list; i += NT) {
                    const uint32_t key = sm.list[i];
                    if (key > tau) mass += R.units(R.weight(key));
                    tie += key == tau;
                }
                mass = warp_sum(mass);
                tie = __reduce_add_sync(0xffffffffu, tie);
                if (lane == 0) {
                    sm.wsum[warp] = mass;
                    sm.wtie[warp] = tie;
                }
                __syncthreads();
                own = 0;
                for (int w = 0; w < NW; w++) {
                    own += sm.wsum[w];
                    own_ties += sm.wtie[w];
                }
                if (with_floor && tau == floor_key) own = -1;   // the floor's own are not in the list
                __syncthreads();
            }
            return tau;
        }
        lo_key = kl_list;
        hi_key = kh;
        shift = 0;
        while ((hi_key - kl) >> shift >= FBINS) shift++;
        cluster.sync();                      // before the histogram and the list are written again
    }
}

template <int NT, bool RESIDENT>
__global__ void __launch_bounds__(NT, 1024 / NT) k_sample_filtered(const float *__restrict__ logits, int64_t ld, int64_t n,
                                                                   const float *__restrict__ temp,
                                                                   const int32_t *__restrict__ top_k,
                                                                   const float *__restrict__ top_p,
                                                                   const float *__restrict__ min_p,
                                                                   const float *__restrict__ uni, int64_t slice, int bits,
                                                                   int wide, int32_t *__restrict__ out) {
    constexpr int NW = NT / 32;
    extern __shared__ __align__(16) uint8_t raw[];
    FShared &sm = *reinterpret_cast<FShared *>(raw);
    uint4 *keys = reinterpret_cast<uint4 *>(raw + (sizeof(FShared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), C = cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / C, begin = min(n, rank * slice), end = min(n, begin + slice);
    Row R;
    R.x = logits + r * ld + begin;
    R.keys = keys;
    R.n = (int)(end - begin);
    R.n4 = (R.n + 3) / 4;
    if (tid < 64) sm.table[tid] = exp2((double)tid / 64);
    if (tid == 0) sm.kmax = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    uint32_t km = 0;
    const int whole = wide ? R.n / 4 : 0;    // 16-byte loads of an aligned row
#pragma unroll 4
    for (int i = tid; i < whole; i += NT) {
        const float4 v = __ldcs((const float4 *)R.x + i);
        const uint4 k = make_uint4(order_key(v.x), order_key(v.y), order_key(v.z), order_key(v.w));
        km = max(max(km, max(k.x, k.y)), max(k.z, k.w));
        if (RESIDENT) keys[i] = k;
    }
#pragma unroll 4
    for (int i = 4 * whole + tid; i < 4 * R.n4; i += NT) {
        const uint32_t k = i < R.n ? order_key(R.x[i]) : 0;
        km = max(km, k);
        if (RESIDENT) ((uint32_t *)keys)[i] = k;
    }
    km = __reduce_max_sync(0xffffffffu, km);
    if (lane == 0) atomicMax(&sm.kmax, km);
    const float T = temp ? temp[r] : 1.f, u = uni[r];
    int64_t k = top_k ? top_k[r] : 0;
    float p = top_p ? top_p[r] : 1.f;
    double mp = min_p ? (double)min_p[r] : 0.0;
    cluster.sync();
    R.kmax = 0;
#pragma unroll
    for (unsigned c = 0; c < MAXC; c++) R.kmax = max(R.kmax, cluster.map_shared_rank(&sm, c < C ? c : 0)->kmax);
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
    long long ties = 0, above, goal, own = -1;
    int own_ties = 0;
    const bool none = R.kmax == KEY_NINF;
    if (!none) {
        if (k == 1) {
            tau = R.kmax;
            ties = 1;
        } else {
            if (k < n) {
                goal = k;
                tau = select<NT, RESIDENT, false>(R, sm, 0, 0, 0.0, goal, above, own, own_ties);
                ties = k - above;
            }
            if (p < 1.f) {
                tau = select<NT, RESIDENT, true>(R, sm, tau, ties, (double)p, goal, above, own, own_ties);
                const long long w = R.units(R.weight(tau));
                ties = (goal - above + w - 1) / w;
            }
            if (mp > 0.0) {
                // the smallest key with weight >= min_p
                const uint32_t least = last_key(R.kmax, [&](uint32_t c) { return R.weight(c) < mp; }) + 1;
                if (least > tau) {
                    tau = least;
                    ties = n;
                    own = -1;
                }
            }
        }
    }
    // ---- the draw
    const long long wtau = tau ? R.units(R.weight(tau)) : 0;
    auto part = [&](int b, int e) {          // a warp's fours b .. e - 1: their weight above tau, and ties
        long long mass = 0;
        int tie = 0;
        auto add = [&](uint32_t key) {
            if (key > tau) mass += R.units(R.weight(key));
            tie += key == tau;
        };
        for (int i = b + lane; i < e; i += 32) {
            const uint4 q = R.four<RESIDENT>(i);
            add(q.x);
            add(q.y);
            add(q.z);
            add(q.w);
        }
        mass = warp_sum(mass);
        tie = __reduce_add_sync(0xffffffffu, tau ? tie : 0);
        if (lane == 0) {
            sm.wsum[warp] = mass;
            sm.wtie[warp] = tie;
        }
    };
    int step = (R.n4 + NW - 1) / NW;
    const bool known = own >= 0;             // the same in every CTA of the cluster
    if (!none && !known) part(min(R.n4, warp * step), min(R.n4, (warp + 1) * step));
    __syncthreads();
    if (tid == 0) {
        long long mass = known ? own : 0;
        int tie = known ? own_ties : 0;
        for (int w = 0; w < NW && !known && !none; w++) {
            mass += sm.wsum[w];
            tie += sm.wtie[w];
        }
        sm.mass = mass;
        sm.ties = tie;
    }
    cluster.sync();
    // every CTA adds up the cluster; the one that holds the target goes on
    long long masses[MAXC];
    int tie_of[MAXC];
#pragma unroll
    for (unsigned c = 0; c < MAXC; c++) {
        const FShared *o = cluster.map_shared_rank(&sm, c < C ? c : 0);
        masses[c] = o->mass;
        tie_of[c] = o->ties;
    }
    long long total = 0, mine = 0, my_mass = 0, tie_at = 0, my_tie = 0;
#pragma unroll
    for (unsigned c = 0; c < MAXC; c++) {
        if (c >= C) continue;
        if (c == rank) {
            mine = total;
            my_tie = tie_at;
        }
        const long long kept = masses[c] + max(0ll, min((long long)tie_of[c], ties - tie_at)) * wtau;
        if (c == rank) my_mass = kept;
        total += kept;
        tie_at += tie_of[c];
    }
    cluster.sync();                          // no CTA leaves while another reads it
    if (none) {
        if (rank == 0 && tid == 0) out[r] = -1;
        return;
    }
    long long target = (long long)((double)(u > 0.f ? u : 0.f) * (double)total);
    target = target > total - 1 ? total - 1 : target;
    if (!(mine <= target && target < mine + my_mass)) return;
    // from the slice to a warp's part of it, to a warp's part of that, to the element
    int b = 0, len = R.n4;
    for (int level = 0; level < 2; level++) {
        if (level || known) part(min(b + len, b + warp * step), min(b + len, b + (warp + 1) * step));
        __syncthreads();
        if (warp == 0) {
            const long long mass = lane < NW ? sm.wsum[lane] : 0, tie = lane < NW ? sm.wtie[lane] : 0;
            const long long t = my_tie + warp_scan(tie) - tie;
            const long long kept = mass + max(0ll, min(tie, ties - t)) * wtau, to = mine + warp_scan(kept);
            if (to - kept <= target && target < to) {
                sm.found = lane;
                sm.before = to - kept;
                sm.tie_before = t;
            }
        }
        __syncthreads();
        mine = sm.before;
        my_tie = sm.tie_before;
        const int e = min(b + len, b + (sm.found + 1) * step);
        b += sm.found * step;
        len = e - b;
        step = (len + NW - 1) / NW;
        __syncthreads();
    }
    if (warp != 0) return;
    const int stop = min(R.n, 4 * (b + len));
    for (int i0 = 4 * b; i0 < stop; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < stop ? R.one<RESIDENT>(i) : 0;
        const uint32_t eq = __ballot_sync(0xffffffffu, tau && key == tau);
        long long w = 0;
        if (key > tau) w = R.units(R.weight(key));
        else if (tau && key == tau && my_tie + __popc(eq & ((1u << lane) - 1u)) < ties) w = wtau;
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

template <int NT, bool RESIDENT>
cudaError_t launch(hd_ctx *ctx, int C, int64_t rows, int64_t slice, const float *logits, int64_t ld, int64_t n,
                   const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                   int bits, int32_t *idx) {
    const size_t smem = (sizeof(FShared) + 15) / 16 * 16 + (RESIDENT ? (size_t)slice * sizeof(float) : 0);
    auto kernel = k_sample_filtered<NT, RESIDENT>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess && C > 8) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    const int wide = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    return hd_launch_cluster(ctx, kernel, dim3((unsigned)(rows * C)), dim3(NT), smem, C, logits, ld, n, temperature, top_k,
                             top_p, min_p, u, slice, bits, wide, idx);
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
    const bool few = rows * C <= ctx->sm_count;   // one CTA an SM: twice the threads
#define HD_SAMPLE(NT, RES) launch<NT, RES>(ctx, C, rows, slice, logits, ld, n, temperature, top_k, top_p, min_p, u, bits, idx)
    cudaError_t e = slice > FULL ? HD_SAMPLE(1024, false) : few ? HD_SAMPLE(1024, true) : HD_SAMPLE(512, true);
#undef HD_SAMPLE
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "hd_sample_filtered: %s", cudaGetErrorString(e));
    return HD_OK;
}
