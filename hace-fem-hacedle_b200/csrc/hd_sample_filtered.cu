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
// (read from memory once).  A histogram of 64 bins over -log2 of the weight,
// two to a factor of two, finds the bin in which the running count (top-k) or
// mass (top-p) reaches its goal; that bin's elements are listed and split into
// 1024 by the bits of an order-preserving integer key, and the few elements of
// the one that is left are compared with one another (more than CAP of them --
// many equal logits -- are split again).  Min-p is a smallest key, found by search.  The draw adds
// up contiguous parts per CTA and per warp and follows the target down.
//
// The first histogram has a copy per lane, a bank each: with a single one the
// atomics on shared memory were 13 of a row's 33 us, since logits crowd into
// few bins.  A place in the list is found for 16 elements of a thread at a
// time (4: 1.5 us more per row), and the search for a bin's bounds tries the
// keys next to the computed one first (1.2 us less).
//
// 256 rows of 151936 logits, most with top-p 0.95, take 0.285 ms (156 MB: 24 us
// at the measured copy rate), one row 31 us.  What bounds it: a row passes through
// some 20 steps, eight of them behind a barrier of its cluster, of which only
// the load, the first histogram (about 50 instructions an element) and the list
// touch every element; registers allow two rows at a time on an SM, 41 us a
// pair, so the steps in between leave it half idle (issue slots 45% busy).  One CTA per row that reads its row from L2 again at every pass came
// to the same time with top-k and to 0.5 ms with top-p.
//
// Weights are computed in 64 bits (2^y = 2^(j/256) 2^e 2^r with a table of 256
// and a polynomial of degree 4 in r, |r| <= 1/512: the table-driven method of
// P. T. P. Tang, ACM TOMS 15 (1989), error below 2^-50) and held as whole
// numbers of 2^-s: sums are exact in any order, so neither atomics nor the
// shape of the cluster can change a draw.  s follows from n alone: 50 up to
// 2048 logits, 42 for a vocabulary of 152k, 40 at least up to 737280, then 62 -
// log2(n) rounded up, 31 for the longest.  A weight is off by at most 2^-(s+1)
// of the largest and a running sum by n times that: 1.7e-8 for 152k, below
// what a float32 sum loses at one addition, and up to 0.5 for the longest.
#include <cooperative_groups.h>

#include <cmath>

#include "hd_internal.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int FBINS = 1024, FGROUP = 16, FGROUPS = FBINS / FGROUP;   // FGROUPS: also the first histogram's bins
constexpr int CANDS = 2048;                  // elements of the first histogram's bin that a slice lists
constexpr int CAP = 512;                     // elements compared with one another
constexpr int64_t FULL = 46080;              // elements of a slice that shared memory holds at most
constexpr int MAXC = 16;                     // CTAs per row
constexpr int MAXW = 32;                     // warps per CTA
constexpr uint32_t KEY_NINF = 0x007fffffu;   // key of -infinity

// Larger float, larger key (no NaN, no -0).
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// NaN as -infinity, -0 as 0.
__device__ __forceinline__ float plain(float v) { return v == v ? __fadd_rn(v, 0.f) : -INFINITY; }

struct Row {
    const float *x;       // the slice
    const float4 *held;   // the same, where it is resident: NaN as -infinity, -0 as 0, and a NaN past the end
    int n, n4;            // its length; in fours
    double m, a;          // largest logit, log2(e) / temperature
    float top;            // m
    bool inf;             // the largest is +infinity: read as 0, and all others as -infinity
    int half;             // half the bits of a unit's weight 1
    const double *table;
    __device__ __forceinline__ float seen(float v) const { return !inf || v != v ? v : v == INFINITY ? 0.f : -INFINITY; }
    template <bool RESIDENT>
    __device__ __forceinline__ float4 four(int i) const {
        if (RESIDENT) return held[i];
        auto one = [&](int j) { return j < n ? seen(plain(x[j])) : NAN; };
        return make_float4(one(4 * i), one(4 * i + 1), one(4 * i + 2), one(4 * i + 3));
    }
    template <bool RESIDENT>
    __device__ __forceinline__ float one(int i) const {
        return RESIDENT ? ((const float *)held)[i] : seen(plain(x[i]));
    }
    // y = log2 of the weight, <= 0, and k, whose low bits are 256 y rounded
    __device__ __forceinline__ double log2w(float v, double &k) const {
        const double y = ((double)v - m) * a;
        k = y + 0x1.8p44;
        return y;
    }
    // y < -64, where a weight is below half a unit (the high words of doubles <= 0 order as integers)
    __device__ __forceinline__ static bool tiny(double y) { return (uint32_t)__double2hiint(y) >= 0xC0500000u; }
    // The bin of the first histogram: -2 log2(weight).
    __device__ __forceinline__ static int bin(bool tiny, double k) {
        return tiny ? FGROUPS - 1 : min(-__double2loint(k) >> 7, FGROUPS - 1);
    }
    __device__ __forceinline__ int bin(float v) const {
        double k;
        const double y = log2w(v, k);
        return bin(tiny(y), k);
    }
    // The weight in units, as a double (not for tiny ones).
    __device__ __forceinline__ double weight(double y, double k) const {
        const int ki = __double2loint(k);
        const double r = y - (k - 0x1.8p44);
        // 2^r - 1 = sum (r ln 2)^i / i!
        double p = 0x1.3b2ab6fba4e77p-7;
        p = fma(p, r, 0x1.c6b08d704a0bfp-5);
        p = fma(p, r, 0x1.ebfbdff82c58ep-3);
        p = fma(p, r, 0x1.62e42fefa39efp-1);
        p *= r;
        const double t = table[ki & 255], w = fma(t, p, t);
        return __hiloint2double(__double2hiint(w) + ((ki >> 8) << 20), __double2loint(w));
    }
    __device__ __forceinline__ double weight(float v) const {
        double k;
        const double y = log2w(v, k);
        return tiny(y) ? 0.0 : weight(y, k);
    }
    // Rounded to whole units: at most 2^50 of them, so adding 1.5 * 2^52 leaves them in the low bits.
    __device__ __forceinline__ static long long whole(double w) {
        return __double_as_longlong(w + 0x1.8p52) - 0x4338000000000000ll;
    }
    // Branch-free, so that a thread's four elements interleave.
    __device__ __forceinline__ long long units(float v) const {
        double k;
        const double y = log2w(v, k);
        const long long w = whole(weight(y, k));
        return tiny(y) ? 0 : w;
    }
};

struct FShared {
    union {
        struct {                             // the first histogram, a copy per lane; weights cut at Row::half bits
            uint32_t lane_lo[FGROUPS * 32], lane_hi[FGROUPS * 32];
        };
        struct {                             // the others, 64 bits in two halves; the listed elements
            uint32_t lo[FBINS], hi[FBINS];
            float cand[CANDS];
        };
    };
    long long part[MAXC][FGROUP];            // a group's bins of every CTA
    long long group[FGROUPS];                // its sums over groups of bins
    long long total[FGROUPS];                // the row's
    Row row;
    double table[256];                       // 2^(j / 256), in units
    uint32_t list[CAP], all[CAP + 1];        // the slice's elements of a bin; the row's
    long long weight[CAP + 1];
    long long wsum[MAXW];                    // warps' sums
    int wtie[MAXW];
    uint32_t n_list, n_cand, kmax;           // what other CTAs of the cluster read ..
    long long mass;
    int ties;
    uint32_t pick;                           // .. and write
    long long pick_above;
    int bin;                                 // broadcasts within the CTA
    long long bin_above, goal, before, tie_before;
    uint32_t bound[2];
    int found;
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

// 64 bits in two halves of 32, with the carry.
__device__ __forceinline__ void add64(uint32_t *lo, uint32_t *hi, int b, unsigned long long w) {
    const uint32_t wl = (uint32_t)w, old = atomicAdd(&lo[b], wl);
    const uint32_t wh = (uint32_t)(w >> 32) + (old + wl < old ? 1u : 0u);
    if (wh) atomicAdd(&hi[b], wh);
}

// The loops over a slice are functions of their own: inlined, what the rest of
// the kernel holds was spilled inside them (14 of 45 instructions an element).

// Every element >= least into the first histogram: 1, or (MASS) its units.
template <int NT, bool RESIDENT, bool MASS>
__device__ __noinline__ void first_histogram(FShared &sm, float least) {
    const Row R = sm.row;
    const int tid = threadIdx.x, lane = tid & 31;
    const uint32_t low = (1u << R.half) - 1;
    auto count = [&](float v, double y, double k, unsigned long long w) {
        const bool tiny = Row::tiny(y);
        const int at = Row::bin(tiny, k) * 32 + lane;
        if (!(v >= least)) return;
        if (!MASS) {
            atomicAdd(&sm.lane_lo[at], 1u);
        } else if (tiny) {
            return;
        } else if (RESIDENT) {       // neither half can overflow, and no atomic returns anything
            atomicAdd(&sm.lane_lo[at], (uint32_t)w & low);
            atomicAdd(&sm.lane_hi[at], __funnelshift_r((uint32_t)w, (uint32_t)(w >> 32), R.half));
        } else {
            add64(sm.lane_lo, sm.lane_hi, at, w);
        }
    };
    for (int i = tid; i < R.n4; i += NT) {
        const float4 v = R.four<RESIDENT>(i);
        if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= least)) continue;
        double y[4], k[4];
        unsigned long long w[4] = {0, 0, 0, 0};
        y[0] = R.log2w(v.x, k[0]);
        y[1] = R.log2w(v.y, k[1]);
        y[2] = R.log2w(v.z, k[2]);
        y[3] = R.log2w(v.w, k[3]);
        if (MASS) {
#pragma unroll
            for (int c = 0; c < 4; c++) w[c] = (unsigned long long)Row::whole(R.weight(y[c], k[c]));
        }
        count(v.x, y[0], k[0], w[0]);
        count(v.y, y[1], k[1], w[1]);
        count(v.z, y[2], k[2], w[2]);
        count(v.w, y[3], k[3], w[3]);
    }
}

// The elements lo .. hi into cand, in any order (once there are too many: only their number counts).
template <int NT, bool RESIDENT>
__device__ __noinline__ void list_bin(FShared &sm, float lo, float hi) {
    constexpr int FOURS = 4;                 // a place for a thread's elements costs as much for 16 as for 4
    const Row R = sm.row;
    const int tid = threadIdx.x, lane = tid & 31;
    for (int i0 = 0; i0 < R.n4; i0 += FOURS * NT) {
        float v[4 * FOURS];
        bool in[4 * FOURS];
        int mine = 0;
#pragma unroll
        for (int f = 0; f < FOURS; f++) {
            const int i = i0 + f * NT + tid;
            const float4 x = i < R.n4 ? R.four<RESIDENT>(i) : make_float4(NAN, NAN, NAN, NAN);
            v[4 * f] = x.x;
            v[4 * f + 1] = x.y;
            v[4 * f + 2] = x.z;
            v[4 * f + 3] = x.w;
        }
#pragma unroll
        for (int c = 0; c < 4 * FOURS; c++) {
            in[c] = v[c] >= lo && v[c] <= hi;
            mine += in[c];
        }
        if (!__any_sync(0xffffffffu, mine)) continue;
        int at = mine;                       // a place for each lane's in the warp's run
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, at, o);
            if (lane >= o) at += x;
        }
        uint32_t base = 0;
        if (lane == 31 && at) base = atomicAdd(&sm.n_cand, (uint32_t)at);
        base = __shfl_sync(0xffffffffu, base, 31);
        float *to = sm.cand + base + at - mine;
        if (!mine || base + at > CANDS) continue;
#pragma unroll
        for (int c = 0; c < 4 * FOURS; c++)
            if (in[c]) *to++ = v[c];
    }
}

// A warp's fours b .. e - 1: their weight above ft, and how many equal it.
template <bool RESIDENT>
__device__ __noinline__ void part(FShared &sm, int b, int e, float ft) {
    const Row R = sm.row;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long mass = 0;
    int tie = 0;
    for (int i = b + lane; i < e; i += 32) {
        const float4 v = R.four<RESIDENT>(i);
        tie += (int)(v.x == ft) + (int)(v.y == ft) + (int)(v.z == ft) + (int)(v.w == ft);
        if (!(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) > ft)) continue;
        const long long w0 = R.units(v.x), w1 = R.units(v.y), w2 = R.units(v.z), w3 = R.units(v.w);
        mass += (v.x > ft ? w0 : 0) + (v.y > ft ? w1 : 0) + (v.z > ft ? w2 : 0) + (v.w > ft ? w3 : 0);
    }
    mass = warp_sum(mass);
    tie = __reduce_add_sync(0xffffffffu, tie);
    if (lane == 0) {
        sm.wsum[warp] = mass;
        sm.wtie[warp] = tie;
    }
}

// f(rank) summed over the cluster, four loads in flight at a time.
template <typename F>
__device__ __forceinline__ long long cluster_sum(unsigned C, F f) {
    long long v = 0;
    for (unsigned r = 0; r < C; r += 4) {
        long long x[4];
#pragma unroll
        for (unsigned i = 0; i < 4; i++) x[i] = f(r + i < C ? r + i : r);
#pragma unroll
        for (unsigned i = 0; i < 4; i++) v += r + i < C ? x[i] : 0;
    }
    return v;
}

// The largest key <= top for which `low` holds, by a warp; it holds for
// KEY_NINF, not for top, and for all keys below one for which it holds.  The
// keys next to a guess are tried first.
template <typename F>
__device__ uint32_t last_key(uint32_t top, double guess, F low) {
    const int lane = threadIdx.x & 31;
    uint32_t lo = KEY_NINF, hi = top;
    {
        const int64_t c64 = (int64_t)order_key(plain((float)guess)) + lane - 16;
        const uint32_t c = c64 < lo ? lo : c64 > hi ? hi : (uint32_t)c64;
        const uint32_t high = ~__ballot_sync(0xffffffffu, c == lo || (c != hi && low(c)));
        if (high & ~1u && !(high & 1u)) return __shfl_sync(0xffffffffu, c, __ffs(high) - 2);
    }
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
// `few`: the elements above the floor are at most CAP together (top-k has
// left them): they are listed at once and compared, without a histogram.
// `clear`: the first histogram is all zeros already.
// `own` becomes the slice's own weight above tau and its elements equal to it
// where the histogram tells (MASS, one level), and -1 elsewhere.
template <int NT, bool RESIDENT, bool MASS>
__device__ uint32_t select(const Row &R, FShared &sm, uint32_t floor_key, long long floor_ties, bool few, bool clear, double p,
                           long long &goal, long long &above, long long &own, int &own_ties) {
    constexpr int NW = NT / 32;
    static_assert(NW >= MAXC && NW <= MAXW, "a warp per CTA of the cluster");
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const unsigned C = cluster.num_blocks(), rank = cluster.block_rank();
    const long long floor_w = floor_ties > 0 ? floor_ties * (MASS ? R.units(key_value(floor_key)) : 1) : 0;
    uint32_t lo_key = max(floor_key + 1, KEY_NINF), hi_key = order_key(R.top);   // the elements in question; the floor's own come on top
    bool with_floor = floor_w > 0;
    int shift = -1;                          // -1: the first histogram; else bins of the key, from hi_key down
    long long own_above = 0;
    above = 0;
    own = -1;
    own_ties = 0;
    bool listed = false;                     // the elements in question are in every CTA's cand
    // f(key) of each of them (and of the lanes' own pace; for few elements)
    auto each = [&](auto f) {
        if (listed) {
            for (int i = tid; i < (int)sm.n_cand; i += NT) f(order_key(sm.cand[i]));
        } else {
            const float lo = key_value(lo_key), hi = key_value(hi_key);
            auto in = [&](float v) { if (v >= lo && v <= hi) f(order_key(v)); };
            for (int i = tid; i < R.n4; i += NT) {
                const float4 v = R.four<RESIDENT>(i);
                in(v.x);
                in(v.y);
                in(v.z);
                in(v.w);
            }
        }
    };
    for (int level = 0;; level++) {
        int pick = 0;
        uint32_t kl_list = lo_key, kh = hi_key;
        if (few) {
            if (tid == 0) sm.n_list = 0;
            __syncthreads();
        } else {
            if (level == 0) {
                if (!clear)
                    for (int b = tid; b < FGROUPS * 32; b += NT) sm.lane_lo[b] = sm.lane_hi[b] = 0;
            } else
                for (int b = tid; b < FBINS; b += NT) sm.lo[b] = sm.hi[b] = 0;
            if (tid == 0) sm.n_list = 0;
            __syncthreads();
            if (level == 0) {
                first_histogram<NT, RESIDENT, MASS>(sm, key_value(lo_key));
            } else {
                auto count = [&](uint32_t key) {
                    if (key < lo_key || key > hi_key) return;
                    const int b = (int)((hi_key - key) >> shift);
                    if (!MASS) {
                        atomicAdd(&sm.lo[b], 1u);
                    } else {
                        add64(sm.lo, sm.hi, b, (unsigned long long)R.units(key_value(key)));
                    }
                };
                each(count);
            }
            __syncthreads();
            // groups of 16 bins, or the first histogram's bins of 32 lanes: eight threads each
            for (int q = tid / 8; q < FGROUPS; q += NT / 8) {
                unsigned long long s = 0;
                if (level == 0) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int b = q * 32 + 4 * (tid & 7) + i;
                        s += ((unsigned long long)sm.lane_hi[b] << (RESIDENT ? R.half : 32)) + sm.lane_lo[b];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < FGROUP / 8; i++) {
                        const int b = q * FGROUP + FGROUP / 8 * (tid & 7) + i;
                        s += ((unsigned long long)sm.hi[b] << 32) + sm.lo[b];
                    }
                }
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if ((tid & 7) == 0) sm.group[q] = (long long)s;
            }
            cluster.sync();
            const int floor_bin = !with_floor ? -1 : level == 0 ? R.bin(key_value(floor_key)) * FGROUP : (int)((hi_key - floor_key) >> shift);
            if (tid < FGROUPS)
                sm.total[tid] = (floor_bin >= 0 && floor_bin / FGROUP == tid ? floor_w : 0) +
                                cluster_sum(C, [&](unsigned r) { return cluster.map_shared_rank(&sm, r)->group[tid]; });
            __syncthreads();
            if (warp == 0) {
                const long long t0 = sm.total[2 * lane], t1 = sm.total[2 * lane + 1];
                const long long inc = warp_scan(t0 + t1);
                if (MASS && level == 0) {
                    const long long mass = __shfl_sync(0xffffffffu, inc, 31);
                    goal = __double2ll_ru(p * (double)mass);
                    goal = goal < 1 ? 1 : goal > mass ? mass : goal;
                }
                const long long b0 = above + inc - t0 - t1, b1 = b0 + t0, b2 = b1 + t1;
                const bool mine = b0 < goal && b2 >= goal;
                const int src = __ffs(__ballot_sync(0xffffffffu, mine)) - 1;
                const int q = __shfl_sync(0xffffffffu, b1 >= goal ? 2 * lane : 2 * lane + 1, src);
                const long long base = __shfl_sync(0xffffffffu, b1 >= goal ? b0 : b1, src);
                if (lane == 0) {
                    sm.bin = q;
                    sm.bin_above = base;
                    sm.goal = goal;
                }
            }
            __syncthreads();
            goal = sm.goal;
            if (level > 0) {
                // the group's bins: a warp per CTA fetches them, one adds them up
                const int q = sm.bin;
                if (warp < (int)C && lane < FGROUP) {
                    const FShared *o = cluster.map_shared_rank(&sm, warp);
                    sm.part[warp][lane] = (long long)(((unsigned long long)o->hi[q * FGROUP + lane] << 32) | o->lo[q * FGROUP + lane]);
                }
                __syncthreads();
                if (warp == 0) {
                    const int b = q * FGROUP + lane;
                    long long v = lane < FGROUP && floor_bin == b ? floor_w : 0;
                    if (lane < FGROUP)
                        for (unsigned r = 0; r < C; r++) v += sm.part[r][lane];
                    const long long run = sm.bin_above + warp_scan(v);
                    const int first = __ffs(__ballot_sync(0xffffffffu, run >= goal)) - 1;
                    __syncwarp();
                    if (lane == first) {
                        sm.bin = b;
                        sm.bin_above = run - v;
                    }
                }
                __syncthreads();
            }
            pick = sm.bin;
            above = sm.bin_above;
            // the bin's keys
            uint32_t kl;
            if (level == 0) {
                if (warp < 2) {
                    const int v = pick + warp;   // the largest key of a bin >= v
                    const uint32_t k = v == 0 ? order_key(R.top) : v >= FGROUPS ? KEY_NINF - 1 : last_key(order_key(R.top), R.m - (128.0 * v - 0.5) / 256 / R.a, [&](uint32_t c) { return R.bin(key_value(c)) >= v; });
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
            with_floor = with_floor && (level == 0 ? floor_bin / FGROUP : floor_bin) == pick;
            if (with_floor) kl = floor_key;      // the floor's own below the others
            if (kl == kh) {
                cluster.sync();                  // before the histogram is written again
                return kl;
            }
            if (level == 0) {
                if (MASS) own_above = warp_sum((lane < pick ? sm.group[lane] : 0) + (lane + 32 < pick ? sm.group[lane + 32] : 0));
                lo_key = with_floor ? floor_key + 1 : kl;
                hi_key = kh;
                shift = 0;
                while ((hi_key - kl) >> shift >= FBINS) shift++;
                // list the bin's elements, over the histogram: its sums are in group, which nobody reads any more
                // from here on but this CTA
                if (tid == 0) sm.n_cand = 0;
                __syncthreads();
                list_bin<NT, RESIDENT>(sm, key_value(lo_key), key_value(hi_key));
                cluster.sync();
                // by a warp, for all
                if (warp == 0) {
                    const uint32_t c = cluster.map_shared_rank(&sm, lane < (int)C ? lane : 0)->n_cand;
                    const int ok = __all_sync(0xffffffffu, c <= CANDS);
                    if (lane == 0) sm.found = ok;
                }
                __syncthreads();
                listed = sm.found;
                continue;
            }
            kl_list = with_floor ? floor_key + 1 : kl;
        }
        auto put = [&](uint32_t key) {
            if (key < kl_list || key > kh) return;
            const uint32_t at = atomicAdd(&sm.n_list, 1u);
            if (at < CAP) sm.list[at] = key;
        };
        each(put);
        cluster.sync();
        // every warp learns the lists' lengths, a lane a CTA
        const uint32_t number = lane < (int)C ? cluster.map_shared_rank(&sm, lane)->n_list : 0;
        uint32_t upto = number;
#pragma unroll
        for (int o = 1; o < MAXC; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, upto, MAXC - 1);
        if (all <= CAP) {
            // a warp per CTA's list
            const uint32_t len = __shfl_sync(0xffffffffu, number, warp & (MAXC - 1));
            const uint32_t start = __shfl_sync(0xffffffffu, upto, warp & (MAXC - 1)) - len;
            if (warp < (int)C) {
                const FShared *o = cluster.map_shared_rank(&sm, warp);
                for (uint32_t i = lane; i < len; i += 32) sm.all[start + i] = o->list[i];
            }
            if (with_floor && tid == 0) sm.all[all] = floor_key;
            const int L = (int)all + (with_floor ? 1 : 0);
            __syncthreads();
            for (int i = tid; i < L; i += NT)
                sm.weight[i] = i == (int)all ? floor_w : MASS ? R.units(key_value(sm.all[i])) : 1;
            __syncthreads();
            if (few) {                       // their mass is known only now
                if (warp == 0) {
                    long long mass = 0;
                    for (int i = lane; i < L; i += 32) mass += sm.weight[i];
                    mass = warp_sum(mass);
                    if (lane == 0) {
                        const long long to = __double2ll_ru(p * (double)mass);
                        sm.goal = to < 1 ? 1 : to > mass ? mass : to;
                    }
                }
                __syncthreads();
                goal = sm.goal;
            }
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
            if (MASS && level == 1 && !few) {
                // this slice above tau: its bins before the threshold's, and what the list adds
                long long mass = 0;
                for (int b = tid; b < pick; b += NT) mass += (long long)(((unsigned long long)sm.hi[b] << 32) | sm.lo[b]);
                int tie = 0;
                for (int i = tid; i < (int)sm.n_list; i += NT) {
                    const uint32_t key = sm.list[i];
                    if (key > tau) mass += R.units(key_value(key));
                    tie += key == tau;
                }
                mass = warp_sum(mass);
                tie = __reduce_add_sync(0xffffffffu, tie);
                if (lane == 0) {
                    sm.wsum[warp] = mass;
                    sm.wtie[warp] = tie;
                }
                __syncthreads();
                own = own_above + warp_sum(lane < NW ? sm.wsum[lane] : 0);
                own_ties = __reduce_add_sync(0xffffffffu, lane < NW ? sm.wtie[lane] : 0);
                if (with_floor && tau == floor_key) own = -1;   // the floor's own are not in the list
                __syncthreads();
            }
            return tau;
        }
        lo_key = kl_list;
        hi_key = kh;
        shift = 0;
        while ((hi_key - (with_floor ? floor_key : lo_key)) >> shift >= FBINS) shift++;
        cluster.sync();                      // before the histogram and the list are written again
    }
}

template <int NT, bool RESIDENT>
__global__ void __launch_bounds__(NT, 1024 / NT) k_sample_filtered(const float *__restrict__ logits, int64_t ld, int64_t n,
                                                                   const float *__restrict__ temp,
                                                                   const int32_t *__restrict__ top_k,
                                                                   const float *__restrict__ top_p,
                                                                   const float *__restrict__ min_p,
                                                                   const float *__restrict__ uni, int64_t slice, double unit, int half,
                                                                   int wide, int32_t *__restrict__ out) {
    constexpr int NW = NT / 32;
    extern __shared__ __align__(16) uint8_t raw[];
    FShared &sm = *reinterpret_cast<FShared *>(raw);
    float4 *held = reinterpret_cast<float4 *>(raw + (sizeof(FShared) + 15) / 16 * 16);
    cg::cluster_group cluster = cg::this_cluster();
    const unsigned rank = cluster.block_rank(), C = cluster.num_blocks();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t r = blockIdx.x / C, begin = min(n, rank * slice), end = min(n, begin + slice);
    Row R;
    R.x = logits + r * ld + begin;
    R.held = held;
    R.inf = false;
    R.n = (int)(end - begin);
    R.n4 = (R.n + 3) / 4;
    for (int i = tid; i < 256; i += NT) sm.table[i] = exp2((double)i / 256) * unit;
    for (int b = tid; b < FGROUPS * 32; b += NT) sm.lane_lo[b] = sm.lane_hi[b] = 0;
    if (tid == 0) sm.kmax = 0;
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    float mx = -INFINITY;
    const int whole = wide ? R.n / 4 : 0;    // 16-byte loads of an aligned row
#pragma unroll 4
    for (int i = tid; i < whole; i += NT) {
        const float4 v = __ldcs((const float4 *)R.x + i);
        const float4 q = make_float4(plain(v.x), plain(v.y), plain(v.z), plain(v.w));
        mx = fmaxf(fmaxf(mx, fmaxf(q.x, q.y)), fmaxf(q.z, q.w));
        if (RESIDENT) held[i] = q;
    }
#pragma unroll 4
    for (int i = 4 * whole + tid; i < 4 * R.n4; i += NT) {
        const float q = i < R.n ? plain(R.x[i]) : NAN;
        mx = fmaxf(mx, q);
        if (RESIDENT) ((float *)held)[i] = q;
    }
    const uint32_t km = __reduce_max_sync(0xffffffffu, order_key(mx));
    if (lane == 0) atomicMax(&sm.kmax, km);
    const float T = temp ? temp[r] : 1.f, u = uni[r];
    int64_t k = top_k ? top_k[r] : 0;
    float p = top_p ? top_p[r] : 1.f;
    double mp = min_p ? (double)min_p[r] : 0.0;
    cluster.sync();
    const uint32_t kmax = __reduce_max_sync(0xffffffffu, cluster.map_shared_rank(&sm, lane < (int)C ? lane : 0)->kmax);
    R.top = key_value(kmax);
    if (k <= 0 || k > n) k = n;
    if (p != p) p = 1.f;
    if (!(T > 0.f) || p <= 0.f) k = 1;
    mp = mp > 0.0 ? fmin(mp, 1.0) : 0.0;
    if (R.top == INFINITY) {
        R.inf = true;
        R.top = 0.f;
        if (RESIDENT) {
            for (int i = tid; i < R.n4; i += NT) held[i] = make_float4(R.seen(held[i].x), R.seen(held[i].y), R.seen(held[i].z), R.seen(held[i].w));
            __syncthreads();
        }
    }
    R.m = (double)R.top;
    R.a = T > 0.f ? fmax(1.4426950408889634 / (double)T, 1e-300) : 1.0;   // an infinite temperature leaves -infinity behind
    R.half = half;
    R.table = sm.table;
    if (tid == 0) sm.row = R;
    __syncthreads();
    // tau, and how many of the elements equal to it stay
    uint32_t tau = 0;
    long long ties = 0, above, goal, own = -1;
    int own_ties = 0;
    const bool none = kmax == KEY_NINF;
    if (!none) {
        if (k == 1) {
            tau = order_key(R.top);
            ties = 1;
        } else {
            if (k < n) {
                goal = k;
                tau = select<NT, RESIDENT, false>(R, sm, 0, 0, false, true, 0.0, goal, above, own, own_ties);
                ties = k - above;
            }
            if (p < 1.f) {
                tau = select<NT, RESIDENT, true>(R, sm, tau, ties, k <= CAP, k == n, (double)p, goal, above, own, own_ties);
                const long long w = R.units(key_value(tau));
                ties = (goal - above + w - 1) / w;
            }
            if (mp > 0.0) {
                // the smallest key with weight >= min_p
                const uint32_t least = last_key(order_key(R.top), R.m + log2(mp) / R.a, [&](uint32_t c) { return R.weight(key_value(c)) < mp * unit; }) + 1;
                if (least > tau) {
                    tau = least;
                    ties = n;
                    own = -1;
                }
            }
        }
    }
    // ---- the draw
    const float ft = tau ? key_value(tau) : -INFINITY;   // (no filter: -infinity's weight is 0, kept or not)
    const long long wtau = tau ? R.units(ft) : 0;
    int step = (R.n4 + NW - 1) / NW;
    const bool known = own >= 0;             // the same in every CTA of the cluster
    if (!none && !known) part<RESIDENT>(sm, min(R.n4, warp * step), min(R.n4, (warp + 1) * step), ft);
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
    // every CTA adds up the cluster, a lane a CTA; the one that holds the target goes on
    if (warp == 0) {
        const FShared *o = cluster.map_shared_rank(&sm, lane < (int)C ? lane : 0);
        const long long mass = lane < (int)C ? o->mass : 0, tie = lane < (int)C ? o->ties : 0;
        const long long t = warp_scan(tie) - tie;
        const long long kept = mass + max(0ll, min(tie, ties - t)) * wtau, to = warp_scan(kept);
        const long long total = __shfl_sync(0xffffffffu, to, 31);
        long long target = (long long)((double)(u > 0.f ? u : 0.f) * (double)total);
        target = target > total - 1 ? total - 1 : target;
        if (lane == (int)rank) {
            sm.found = to - kept <= target && target < to;
            sm.goal = target;
            sm.before = to - kept;
            sm.tie_before = t;
        }
    }
    cluster.sync();                          // no CTA leaves while another reads it
    if (none) {
        if (rank == 0 && tid == 0) out[r] = -1;
        return;
    }
    if (!sm.found) return;
    const long long target = sm.goal;
    long long mine = sm.before, my_tie = sm.tie_before;
    __syncthreads();
    // from the slice to a warp's part of it, to a warp's part of that, to the element
    int b = 0, len = R.n4;
    for (int level = 0; level < 2; level++) {
        if (level || known) part<RESIDENT>(sm, min(b + len, b + warp * step), min(b + len, b + (warp + 1) * step), ft);
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
        const float v = i < stop ? R.one<RESIDENT>(i) : NAN;
        const uint32_t eq = __ballot_sync(0xffffffffu, tau && v == ft);
        long long w = 0;
        if (v > ft) w = R.units(v);
        else if (tau && v == ft && my_tie + __popc(eq & ((1u << lane) - 1u)) < ties) w = wtau;
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

constexpr int64_t HALF = 19456;              // elements of a slice of which two fit an SM
template <int NT, bool RESIDENT>
cudaError_t allow(const hd_ctx *ctx) {
    static std::atomic<uint64_t> allowed{0};
    return hd_allow_smem(allowed, ctx, (const void *)k_sample_filtered<NT, RESIDENT>,
                         sizeof(FShared) + 16 + (RESIDENT ? FULL * sizeof(float) : 0), true);
}

// Clusters of 2^c CTAs with slices of up to HALF that the device runs at a
// time; a cluster lies within one GPC, so these are fewer than the SMs allow.
template <int NT>
int at_a_time(const hd_ctx *ctx, int c) {
    static std::atomic<int> known[64][8];    // 0: not asked yet
    const bool keep = ctx->device < 64 && c < 8;
    const int before = keep ? known[ctx->device][c].load(std::memory_order_relaxed) : 0;
    if (before) return before - 1;
    cudaLaunchConfig_t cfg{};
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1u << c;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3(1u << c);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = sizeof(FShared) + 16 + HALF * sizeof(float);
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (allow<NT, true>(ctx) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, k_sample_filtered<NT, true>, &cfg) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    if (keep) known[ctx->device][c].store(n + 1, std::memory_order_relaxed);
    return n;
}

template <int NT, bool RESIDENT>
cudaError_t launch(hd_ctx *ctx, int C, int64_t rows, int64_t slice, const float *logits, int64_t ld, int64_t n,
                   const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p, const float *u,
                   double unit, int half, int32_t *idx) {
    const size_t smem = (sizeof(FShared) + 15) / 16 * 16 + (RESIDENT ? (size_t)slice * sizeof(float) : 0);
    auto kernel = k_sample_filtered<NT, RESIDENT>;
    cudaError_t e = allow<NT, RESIDENT>(ctx);
    if (e != cudaSuccess) return e;
    const int wide = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    return hd_launch_cluster(ctx, kernel, dim3((unsigned)(rows * C)), dim3(NT), smem, C, logits, ld, n, temperature, top_k,
                             top_p, min_p, u, slice, unit, half, wide, idx);
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
    // CTAs per row, and their threads.  A row's steps are the quicker the more of them (151936 logits, all rows at
    // a time: 16 CTAs of 1024 threads 31 us, 8 of 1024 33, 16 of 512 35, 8 of 512 46), while slices keep 2048
    // elements, but rows in a second wave cost as much again (8 rows: 56 us with 16 CTAs, 33 with 8).  So: the first
    // of these that runs all rows at a time; with more rows than any of them, as few CTAs as keep two slices on an
    // SM.
    auto slice_of = [&](int c) { return ((n + c - 1) / c + 3) / 4 * 4; };
    int least = 0, most;                     // log2 of the CTAs
    while ((1 << least) < MAXC && slice_of(1 << least) > HALF) least++;
    for (most = least; (1 << most) < MAXC && slice_of(1 << most) > 4096;) most++;
    int C = 0;
    bool few = true;
    for (int c = most; c >= least && !C; c--)
        if (rows <= at_a_time<1024>(ctx, c)) C = 1 << c;
    if (!C) {
        few = false;
        for (int c = most; c >= least && !C; c--)
            if (rows <= at_a_time<512>(ctx, c)) C = 1 << c;
        if (!C) C = 1 << least;
    }
    const int64_t slice = slice_of(C);
    // Units: n of them sum below 2^62, and a lane's share of a resident slice times half of their bits below 2^32.  The
    // slice is the longest that any number of rows leads to, so that a row's weights are the same in every batch.
    auto log2_up = [](int64_t v) {
        int b = 0;
        while (((int64_t)1 << b) < v) b++;
        return b;
    };
    int bits = 62 - log2_up(n) < 50 ? 62 - log2_up(n) : 50;
    const int64_t longest = slice_of(1 << least);
    const int room = 2 * (36 - log2_up(longest));
    if (longest <= FULL && bits > room) bits = room;
    const int half = (bits + 1) / 2;
    const double unit = std::ldexp(1.0, bits);
#define HD_SAMPLE(NT, RES) launch<NT, RES>(ctx, C, rows, slice, logits, ld, n, temperature, top_k, top_p, min_p, u, unit, half, idx)
    cudaError_t e = slice > FULL ? HD_SAMPLE(1024, false) : few ? HD_SAMPLE(1024, true) : HD_SAMPLE(512, true);
#undef HD_SAMPLE
    if (e != cudaSuccess) return hd_fail(ctx, HD_E_CUDA, "hd_sample_filtered: %s", cudaGetErrorString(e));
    return HD_OK;
}
