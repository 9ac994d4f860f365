// hd_kv_pages.cu -- page tables and slot maps of a paged KV cache, built on
// the device from request lengths, and the return of finished requests'
// pages.
//
// Request r holds len[r] cached tokens in the first ceil(len[r] / P) entries
// of its table.  A step adds new[r] tokens to it, so it needs
// ceil((len + new) / P) - ceil(len / P) more pages, which come off the top of
// the free stack in request order.  With row0 the exclusive prefix sum of
// new and page0 that of the needed pages, the token of row row0[r] + t sits
// at position p = len[r] + t in page p / P of the request:
//   k = p / P < ceil(len / P)   table[r][k]                (a page it holds)
//   otherwise                   free[n_free - 1 - (page0[r] + k - ceil(len / P))]
// so a row's slot follows from the two prefix sums alone and no thread waits
// for a table entry that another one writes.
//
// One launch: every CTA of one cluster scans all requests (a few KB that the
// L2 holds), and the cluster's threads share the rows.  The barrier of the
// cluster stands between the last read of lens / n_free and the first write
// of lens_out / n_free_out, which may be the same arrays.  A step that only
// decodes (up to 512 requests, a token each at most) is placed request by
// request: no search, and the table entry is on its way during the scan (4.4 us
// for the kernel alone, caches cold, 8.7 without; a step of 1024 requests, 96 of
// which bring chunks, takes the other way: 11.1).  The call moves 8 bytes a row;
// what bounds it is the latency of loads and scan, and from Python the binding
// (7.8 us a call for a decode step of 256 requests, of which the checks of eleven
// tensors' devices are 0.5, and 8.1 for the step with chunks; a launch that does
// nothing takes 2.5).
#include <climits>

#include "hd_internal.cuh"
#include "hd_mma.cuh"

namespace {

constexpr int PNT = 512;       // threads per CTA
constexpr int PMAXREQ = 8192;  // three int arrays of this length fit shared memory
enum { PAGES_OK = 0, PAGES_SHORT = 1, PAGES_BAD_REQUEST = 2, PAGES_ROWS = 3 };

// Exclusive prefix sums of (a, b) over the CTA; the totals in ta, tb.
__device__ void scan2(int64_t &a, int64_t &b, int64_t &ta, int64_t &tb) {
    __shared__ int64_t wa[PNT / 32], wb[PNT / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t ia = a, ib = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t xa = __shfl_up_sync(0xffffffffu, ia, o), xb = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane >= o) {
            ia += xa;
            ib += xb;
        }
    }
    if (lane == 31) {
        wa[warp] = ia;
        wb[warp] = ib;
    }
    __syncthreads();
    int64_t ba = 0, bb = 0;
    ta = tb = 0;
    for (int w = 0; w < PNT / 32; w++) {
        if (w == warp) {
            ba = ta;
            bb = tb;
        }
        ta += wa[w];
        tb += wb[w];
    }
    a = ba + ia - a;
    b = bb + ib - b;
}

// Pages that hold l >= 0 tokens.
__device__ __forceinline__ int pages_of(int l, int shift) { return (int)(((unsigned)l + (1u << shift) - 1u) >> shift); }

// The last index r of s[0..n] (ascending, s[0] = 0) with s[r] <= v, for v < s[n].
__device__ __forceinline__ int find_run(const int *s, int n, int v) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(PNT) k_pages_assign(const int32_t *lens, const int32_t *__restrict__ nnew, int reqs,
                                                      int32_t *tables, int max_pages, int shift,
                                                      const int32_t *__restrict__ free_list, const int32_t *n_free,
                                                      int free_cap, int pages, int32_t *n_free_out, int32_t *lens_out,
                                                      int32_t *__restrict__ row0, int32_t *__restrict__ slots,
                                                      int32_t *__restrict__ pos, int64_t max_rows,
                                                      int32_t *__restrict__ status) {
    extern __shared__ int sm[];
    int *r0 = sm, *p0 = r0 + reqs + 1, *ln = p0 + reqs + 1;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x, page = 1 << shift;
    const int per = (reqs + PNT - 1) / PNT, b = min(reqs, tid * per), e = min(reqs, b + per);
    const int have_free = *n_free;
    int64_t rows = 0, got = 0;
    bool bad = false, many = false;
    int id = -1;                       // the page that a single request's first new token lies on, if it is held
    for (int r = b; r < e; r++) {
        const int l = lens[r], n = nnew[r];
        const bool wrong = l < 0 || n < 0 || (int64_t)l + n > (int64_t)max_pages << shift;
        ln[r] = l;
        r0[r] = n;
        bad |= wrong;
        many |= n > 1;
        rows += wrong ? 0 : n;
        got += wrong ? 0 : pages_of((int)((unsigned)l + (unsigned)n), shift) - pages_of(l, shift);
    }
    if (per == 1 && b < e && !bad && r0[b] > 0 && (ln[b] & (page - 1))) id = tables[(int64_t)b * max_pages + (ln[b] >> shift)];
    __shared__ uint32_t flags[PNT / 32];
    const uint32_t mine = __reduce_or_sync(0xffffffffu, (bad ? 1u : 0u) | (many ? 2u : 0u));
    if ((tid & 31) == 0) flags[tid >> 5] = mine;
    int64_t trows, tpages, arow = rows, apage = got;
    scan2(arow, apage, trows, tpages);             // (its barrier is the flags', too)
    const uint32_t seen = __reduce_or_sync(0xffffffffu, (tid & 31) < PNT / 32 ? flags[tid & 31] : 0u);
    const bool any_bad = seen & 1, runs = seen & 2 || per > 1;
    const int st = any_bad || have_free < 0 || have_free > free_cap ? PAGES_BAD_REQUEST
                   : tpages > have_free                             ? PAGES_SHORT
                   : trows > max_rows                               ? PAGES_ROWS
                                                                    : PAGES_OK;
    const int64_t me = (int64_t)blockIdx.x * PNT + tid, all = (int64_t)gridDim.x * PNT;
    if (__builtin_expect(st == PAGES_OK && !runs, 0)) {
        // a decode step (no request brings more than one token, no thread has two): each thread places its own
        if (gridDim.x > 1) {           // every CTA of the cluster has read lens and n_free
            mm_cluster_arrive_release();
            mm_cluster_wait();
        }
        if (blockIdx.x == 0) {
            if (tid == 0) {
                row0[reqs] = (int)trows;
                *n_free_out = have_free - (int)tpages;
                *status = st;
            }
            if (b < e) {
                const int l = ln[b], n = r0[b];
                row0[b] = (int)arow;
                lens_out[b] = l + n;
                if (n) {
                    if (!(l & (page - 1))) {
                        id = free_list[have_free - 1 - (int)apage];
                        tables[(int64_t)b * max_pages + (l >> shift)] = id;
                    }
                    slots[arow] = id >= 0 && id < pages ? (id << shift) + (l & (page - 1)) : -1;
                    pos[arow] = l;
                }
            }
        }
        for (int64_t t = trows + me; t < max_rows; t += all) slots[t] = pos[t] = -1;
        return;
    }
    for (int r = b; r < e; r++) {
        const int l = ln[r], n = st == PAGES_OK ? r0[r] : 0;
        r0[r] = st == PAGES_OK ? (int)arow : 0;
        p0[r] = st == PAGES_OK ? (int)apage : 0;
        ln[r] = l;
        arow += n;
        if (st == PAGES_OK) apage += pages_of(l + n, shift) - pages_of(l, shift);
    }
    if (st != PAGES_OK) trows = tpages = 0;
    if (tid == 0) {
        r0[reqs] = (int)trows;
        p0[reqs] = (int)tpages;
    }
    if (gridDim.x > 1) {               // every CTA of the cluster has read lens and n_free
        mm_cluster_arrive_release();
        mm_cluster_wait();
    }
    __syncthreads();
    for (int64_t r = me; r <= reqs; r += all) {
        row0[r] = r0[r];
        if (r < reqs) lens_out[r] = ln[r] + (r0[r + 1] - r0[r]);
    }
    if (me == 0) {
        *n_free_out = have_free - (int)tpages;
        *status = st;
    }
    for (int64_t i = me; i < tpages; i += all) {
        const int r = find_run(p0, reqs, (int)i);
        const int k = pages_of(ln[r], shift) + (int)i - p0[r];
        tables[(int64_t)r * max_pages + k] = free_list[have_free - 1 - (int)i];
    }
    // four consecutive rows a thread: one search, then a walk
    for (int64_t t0 = 4 * me; t0 < max_rows; t0 += 4 * all) {
        int r = t0 < trows ? find_run(r0, reqs, (int)t0) : 0;
        for (int c = 0; c < 4 && t0 + c < max_rows; c++) {
            const int64_t t = t0 + c;
            int slot = -1, p = -1;
            if (t < trows) {
                while (t >= r0[r + 1]) r++;
                p = ln[r] + (int)t - r0[r];
                const int k = p >> shift, held = pages_of(ln[r], shift);
                const int id = k < held ? tables[(int64_t)r * max_pages + k]
                                        : free_list[have_free - 1 - (p0[r] + k - held)];
                if (id >= 0 && id < pages) slot = (id << shift) + (p & (page - 1));
            }
            slots[t] = slot;
            pos[t] = p;
        }
    }
}

// One CTA: the held entries of the finished requests lie in one line (p0),
// which its threads share; those that name a page go to the free stack in that
// order.  Entries below 0 (pages given back early behind a window) or beyond
// what any cache of fewer than 2^31 slots has name none: on the stack they
// would be dealt to another request, whose tokens would then have no slot.
// A call among others takes 6.0 us for 1695 pages of 14 requests out of 256, 14
// for 6977 (16 with one entry a thread at a time), 219 for 193834: a search and
// a load in turn, on one SM, bound it.
__global__ void __launch_bounds__(PNT) k_pages_release(const int32_t *__restrict__ done, int32_t *lens, int reqs,
                                                       int32_t *tables, int max_pages, int shift, int32_t *free_list,
                                                       int32_t *n_free, int free_cap, int32_t *__restrict__ status) {
    extern __shared__ int sm[];
    int *p0 = sm;
    pdl_wait();
    pdl_trigger();
    const int tid = threadIdx.x;
    const int per = (reqs + PNT - 1) / PNT, b = min(reqs, tid * per), e = min(reqs, b + per);
    int64_t got = 0, none = 0, tp, tn;
    bool bad = false;
    for (int r = b; r < e; r++) {
        if (!done[r]) continue;
        const int64_t l = lens[r];
        if (l < 0 || l > (int64_t)max_pages << shift) {
            bad = true;
            break;
        }
        got += pages_of((int)l, shift);
    }
    const int have = *n_free;
    int64_t at = got;
    scan2(at, none, tp, tn);
    bad = __syncthreads_or(bad);
    int st = bad || have < 0 || have > free_cap ? PAGES_BAD_REQUEST : tp > INT_MAX ? PAGES_SHORT : PAGES_OK;
    // held entries i0 + tid, + PNT, ... of the line, four of a thread's on their way at a time; -1 behind the last
    int32_t *t[4];
    int id[4];
    auto load = [&](int64_t i0) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int64_t i = i0 + c * PNT + tid;
            t[c] = nullptr;
            if (i < tp) {
                const int r = find_run(p0, reqs, (int)i);
                t[c] = tables + (int64_t)r * max_pages + ((int)i - p0[r]);
            }
            id[c] = t[c] ? *t[c] : -1;
        }
    };
    auto names_page = [&](int page) { return (unsigned)page < (1u << 31) >> shift; };
    if (st == PAGES_OK) {
        for (int r = b; r < e; r++) {
            p0[r] = (int)at;
            if (done[r]) at += pages_of(lens[r], shift);
        }
        if (tid == 0) p0[reqs] = (int)tp;
        __syncthreads();
        if (have + tp > free_cap) {    // they fit only if some of them name no page
            int64_t mine = 0, all;
            for (int64_t i0 = 0; i0 < tp; i0 += 4 * PNT) {
                load(i0);
#pragma unroll
                for (int c = 0; c < 4; c++) mine += names_page(id[c]);
            }
            scan2(mine, none, all, tn);
            if (have + all > free_cap) st = PAGES_SHORT;
        }
    }
    if (tid == 0) *status = st;
    if (st != PAGES_OK) return;
    int64_t run = have;                // the stack's end
    for (int64_t i0 = 0; i0 < tp; i0 += 4 * PNT) {
        load(i0);
        bool dropped = false;
#pragma unroll
        for (int c = 0; c < 4; c++) dropped |= t[c] && !names_page(id[c]);
        if (!__syncthreads_or(dropped)) {
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (t[c]) free_list[run + c * PNT + tid] = id[c];
            run += min((int64_t)4 * PNT, tp - i0);
        } else {
#pragma unroll
            for (int c = 0; c < 4; c++) {
                int64_t place = names_page(id[c]), all;
                __syncthreads();       // the sums of the scan before are read
                scan2(place, none, all, tn);
                if (names_page(id[c])) free_list[run + place] = id[c];
                run += all;
            }
        }
#pragma unroll
        for (int c = 0; c < 4; c++)
            if (t[c]) *t[c] = -1;
    }
    if (tid == 0) *n_free = (int)run;
    for (int r = b; r < e; r++)
        if (done[r]) lens[r] = 0;
}

int page_shift(int page) {
    if (page < 16 || page > 1024 || (page & (page - 1))) return -1;
    int s = 4;
    while ((1 << s) < page) s++;
    return s;
}

int check_pages(hd_ctx *ctx, const char *name, int reqs, int max_pages, int page) {
    HD_REQUIRE(ctx, reqs >= 0 && max_pages > 0 && page_shift(page) > 0, HD_E_SHAPE,
               "%s: bad shape (requests %d, table width %d, page size %d: a power of two, 16 to 1024)", name, reqs, max_pages,
               page);
    HD_REQUIRE(ctx, (int64_t)max_pages * page < ((int64_t)1 << 31), HD_E_SHAPE, "%s: positions beyond 2^31", name);
    HD_REQUIRE(ctx, reqs <= PMAXREQ, HD_E_UNSUPPORTED, "%s: %d requests (at most %d)", name, reqs, PMAXREQ);
    return HD_OK;
}

}  // namespace

extern "C" int hd_kv_pages_assign(hd_ctx *ctx, const int32_t *lens, const int32_t *new_tokens, int reqs, int32_t *tables,
                                  int max_pages, int page_size, int pages, const int32_t *free_list,
                                  const int32_t *n_free, int free_cap, int32_t *n_free_out, int32_t *lens_out, int32_t *row0,
                                  int32_t *slots, int32_t *pos, int64_t max_rows, int32_t *status) {
    if (!n_free || !n_free_out || !row0 || !status || (reqs > 0 && (!lens || !new_tokens || !tables || !lens_out)) ||
        (max_rows > 0 && (!slots || !pos)) || (free_cap > 0 && !free_list))
        return hd_fail(ctx, HD_E_ARG, "hd_kv_pages_assign: null argument");
    int rc = check_pages(ctx, "hd_kv_pages_assign", reqs, max_pages, page_size);
    if (rc) return rc;
    HD_REQUIRE(ctx, max_rows >= 0 && max_rows < ((int64_t)1 << 31) && free_cap >= 0 && pages >= 0 &&
                        (int64_t)pages * page_size < ((int64_t)1 << 31),
               HD_E_SHAPE, "hd_kv_pages_assign: bad shape (rows %lld, free list of %d, pages %d: fewer than 2^31 slots)",
               (long long)max_rows, free_cap, pages);
    if (!ctx) return HD_E_ARG;
    HdDevice on(ctx);
    const size_t smem = (size_t)(3 * reqs + 2) * sizeof(int);
    static std::atomic<uint64_t> allowed{0};
    HD_CUDA_TRY(ctx, hd_allow_smem(allowed, ctx, (const void *)k_pages_assign, (3 * PMAXREQ + 2) * sizeof(int)));
    // one CTA up to 2048 rows (four a thread), then one more for each 2048, eight at most
    const int64_t want = (max_rows + 4 * PNT - 1) / (4 * PNT);
    const int ctas = want < 1 ? 1 : want > 8 ? 8 : (int)want;
    HD_CUDA_TRY(ctx, hd_launch_cluster(ctx, k_pages_assign, dim3(ctas), dim3(PNT), smem, ctas, lens, new_tokens, reqs, tables,
                                       max_pages, page_shift(page_size), free_list, n_free, free_cap, pages, n_free_out, lens_out,
                                       row0, slots, pos, max_rows, status));
    return HD_OK;
}

extern "C" int hd_kv_pages_release(hd_ctx *ctx, const int32_t *done, int32_t *lens, int reqs, int32_t *tables,
                                   int max_pages, int page_size, int32_t *free_list, int32_t *n_free, int free_cap,
                                   int32_t *status) {
    if (!n_free || !free_list || !status || (reqs > 0 && (!done || !lens || !tables)))
        return hd_fail(ctx, HD_E_ARG, "hd_kv_pages_release: null argument");
    int rc = check_pages(ctx, "hd_kv_pages_release", reqs, max_pages, page_size);
    if (rc) return rc;
    HD_REQUIRE(ctx, free_cap >= 0, HD_E_SHAPE, "hd_kv_pages_release: free list of %d", free_cap);
    if (!ctx) return HD_E_ARG;
    HdDevice on(ctx);
    const size_t smem = (size_t)(reqs + 1) * sizeof(int);
    HD_CUDA_TRY(ctx, hd_launch(ctx, k_pages_release, dim3(1), dim3(PNT), smem, done, lens, reqs, tables, max_pages,
                               page_shift(page_size), free_list, n_free, free_cap, status));
    return HD_OK;
}
