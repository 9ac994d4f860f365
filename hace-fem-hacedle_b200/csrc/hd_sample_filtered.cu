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
// set is "key above tau, or one of the first c elements equal to tau" with a
// weight bound: tau is found by selecting on the bits of an order-preserving
// integer key, counts for top-k and masses for top-p, without a sort.
// Weights are computed in 64 bits and held as whole numbers of 2^-s, s = 62 -
// ceil(log2 n): sums are exact, in any order, so the draw does not depend on
// the schedule, and the rounding of a weight (2^-45 of the largest at a
// vocabulary of 152k) is far below a float32 sum's.
#include <cmath>

#include "hd_internal.cuh"

namespace {

constexpr int FNT = 1024;
constexpr int FBINS = 2048;
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

template <typename T>
__device__ T block_sum(T v, T *buf) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) buf[warp] = v;
    __syncthreads();
    T t = 0;
    for (int w = 0; w < FNT / 32; w++) t += buf[w];
    return t;
}

// Sum of v over the threads below this one; the total in t.
__device__ long long block_scan(long long v, long long *buf, long long &t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += x;
    }
    __syncthreads();
    if (lane == 31) buf[warp] = inc;
    __syncthreads();
    long long before = 0;
    t = 0;
    for (int w = 0; w < FNT / 32; w++) {
        if (w == warp) before = t;
        t += buf[w];
    }
    return before + inc - v;
}

struct Row {
    const float *x;
    int64_t n;
    uint32_t kmax;
    double m, t;          // largest logit, temperature
    double unit;          // 2^s
    // weight of a key in 64 bits, and as a whole number of units
    __device__ double weight(uint32_t key) const {
        const double w = key == kmax ? 1.0 : exp(((double)key_value(key) - m) / t);
        return w == w ? w : 0.0;   // (-inf) / inf
    }
    __device__ long long units(double w) const { return __double2ll_rn(w * unit); }
};

// The largest key tau such that elements >= tau (of those above `floor_key`,
// or equal to it and among `floor_ties`) weigh at least `goal`; `above` is the
// weight of those > tau.  MASS: weigh by units, else by count.
template <bool MASS>
__device__ uint32_t select(const Row &R, uint32_t floor_key, long long floor_ties, long long goal, long long *hist,
                           long long *buf, long long &above) {
    __shared__ uint32_t pick;
    __shared__ long long pick_above;
    uint32_t prefix = 0;
    int shift = 32;
    above = 0;
    for (int level = 0; level < 3; level++) {
        const int bits = level < 2 ? 11 : 10, lo = shift - bits;
        for (int b = threadIdx.x; b < FBINS; b += FNT) hist[b] = 0;
        __syncthreads();
        for (int64_t i = threadIdx.x; i < R.n; i += FNT) {
            const uint32_t key = order_key(R.x[i]);
            if (key <= floor_key) continue;
            if (shift < 32 && (key >> shift) != prefix) continue;
            const long long w = MASS ? R.units(R.weight(key)) : 1;
            atomicAdd((unsigned long long *)&hist[(key >> lo) & ((1u << bits) - 1)], (unsigned long long)w);
        }
        // the elements equal to the floor that count
        if (threadIdx.x == 0 && floor_ties > 0 && (shift == 32 || (floor_key >> shift) == prefix))
            atomicAdd((unsigned long long *)&hist[(floor_key >> lo) & ((1u << bits) - 1)],
                      (unsigned long long)(floor_ties * (MASS ? R.units(R.weight(floor_key)) : 1)));
        __syncthreads();
        // two bins a thread from the top down: the bin in which the running weight reaches the goal
        const int b1 = FBINS - 1 - 2 * threadIdx.x, b0 = b1 - 1;
        long long total;
        const long long before = above + block_scan(hist[b1] + hist[b0], buf, total);
        if (before < goal && before + hist[b1] + hist[b0] >= goal) {
            const bool first = before + hist[b1] >= goal;
            pick = first ? b1 : b0;
            pick_above = first ? before : before + hist[b1];
        }
        __syncthreads();
        prefix = (prefix << bits) | pick;
        above = pick_above;
        shift = lo;
        __syncthreads();
    }
    return prefix;
}

__global__ void __launch_bounds__(FNT) k_sample_filtered(const float *__restrict__ logits, int64_t ld, int64_t n,
                                                         const float *__restrict__ temp, const int32_t *__restrict__ top_k,
                                                         const float *__restrict__ top_p, const float *__restrict__ min_p,
                                                         const float *__restrict__ uni, int scale_bits,
                                                         int32_t *__restrict__ out) {
    __shared__ long long hist[FBINS], buf[FNT / 32];
    __shared__ uint32_t mx;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x;
    const int64_t r = blockIdx.x;
    Row R;
    R.x = logits + r * ld;
    R.n = n;
    if (tid == 0) mx = 0;
    __syncthreads();
    uint32_t km = 0;
    for (int64_t i = tid; i < n; i += FNT) km = max(km, order_key(R.x[i]));
    km = __reduce_max_sync(0xffffffffu, km);
    if ((tid & 31) == 0) atomicMax(&mx, km);
    __syncthreads();
    R.kmax = mx;
    R.m = (double)key_value(R.kmax);
    if (R.kmax == KEY_NINF) {
        if (tid == 0) out[r] = -1;
        return;
    }
    const float T = temp ? temp[r] : 1.f;
    R.t = (double)T;
    R.unit = (double)(1ll << scale_bits);
    int64_t k = top_k ? top_k[r] : 0;
    if (k <= 0 || k > n) k = n;
    float p = top_p ? top_p[r] : 1.f;
    if (p != p) p = 1.f;
    if (!(T > 0.f) || p <= 0.f) k = 1;
    double mp = min_p ? (double)min_p[r] : 0.0;
    mp = mp > 0.0 ? fmin(mp, 1.0) : 0.0;
    // tau, and how many of the elements equal to it stay
    uint32_t tau = 0;
    long long ties = 0, above;
    if (k == 1) {
        tau = R.kmax;
        ties = 1;
    } else {
        if (k < n) {
            tau = select<false>(R, 0, 0, k, hist, buf, above);
            ties = k - above;
        }
        if (p < 1.f) {
            long long part = 0;
            for (int64_t i = tid; i < n; i += FNT) {
                const uint32_t key = order_key(R.x[i]);
                if (key > tau) part += R.units(R.weight(key));
            }
            long long mass = block_sum(part, buf);
            if (k < n) mass += ties * R.units(R.weight(tau));
            long long goal = __double2ll_ru((double)p * (double)mass);
            goal = goal < 1 ? 1 : goal > mass ? mass : goal;
            tau = select<true>(R, tau, k < n ? ties : 0, goal, hist, buf, above);
            const long long w = R.units(R.weight(tau));
            ties = w > 0 ? (goal - above + w - 1) / w : 1;
        }
    }
    // the draw: contiguous runs of indices, one a thread
    const int64_t run = (n + FNT - 1) / FNT, b = min(n, (int64_t)tid * run), e = min(n, b + run);
    const double wt = tau ? R.weight(tau) : 0.0;
    const long long wtau = wt >= mp ? R.units(wt) : 0;
    long long equal = 0, sum = 0, total;
    for (int64_t i = b; i < e; i++) {
        const uint32_t key = order_key(R.x[i]);
        equal += key == tau;
        if (key > tau) {
            const double w = R.weight(key);
            if (w >= mp) sum += R.units(w);
        }
    }
    long long used = block_scan(equal, buf, total);
    const long long stay = max(0ll, min(equal, ties - used));
    sum += stay * wtau;
    const long long before = block_scan(sum, buf, total);
    const float u = uni[r];
    long long target = (long long)((double)(u > 0.f ? u : 0.f) * (double)total);
    target = target > total - 1 ? total - 1 : target;
    if (!(before <= target && target < before + sum)) return;
    long long acc = before;
    for (int64_t i = b; i < e; i++) {
        const uint32_t key = order_key(R.x[i]);
        if (key < tau) continue;
        if (key == tau) {
            if (used++ >= ties) continue;
            acc += wtau;
        } else {
            const double w = R.weight(key);
            if (w >= mp) acc += R.units(w);
        }
        if (acc > target) {
            out[r] = (int32_t)i;
            return;
        }
    }
}

}  // namespace

extern "C" int hd_sample_filtered(hd_ctx *ctx, const float *logits, int64_t ld, int64_t rows, int64_t n,
                                  const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                                  const float *u, int32_t *idx) {
    if ((rows > 0 && (!logits || !u || !idx))) return hd_fail(ctx, HD_E_ARG, "hd_sample_filtered: null argument");
    if (ld == 0) ld = n;
    HD_REQUIRE(ctx, rows >= 0 && rows < ((int64_t)1 << 31) && n > 0 && n < ((int64_t)1 << 31) && ld >= n, HD_E_SHAPE,
               "hd_sample_filtered: bad shape (rows %lld, n %lld, row stride %lld)", (long long)rows, (long long)n,
               (long long)ld);
    if (!ctx) return HD_E_ARG;
    if (rows == 0) return HD_OK;
    HdDevice on(ctx);
    int bits = 0;
    while (((int64_t)1 << bits) < n) bits++;
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_sample_filtered, dim3((unsigned)rows), dim3(FNT), 0, logits, ld, n, temperature, top_k,
                               top_p, min_p, u, 62 - bits, idx));
    return HD_OK;
}
