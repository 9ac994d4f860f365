// hd_kv4_attention.cu -- what attention over the paged 4-bit cache takes.
//
// The query at position i of its request sees position j when j <= i and
// (window == 0 or j > i - window or j < sinks); its output is
// sum_j softmax_j(scale q . k_j) v_j over those, and zeros when it sees none
// (no length, or only table entries that name no page).  The kernels:
// hd_kv4_decode.cu, hd_kv4_prefill.cu.
#include <cmath>

#include "hd_internal.cuh"
#include "hd_kv4_args.cuh"

int hd_kv4_attention_check(hd_ctx *ctx, const char *name, Kv4Args &A, int page_size, int hd) {
    if ((A.rows > 0 && (!A.q || !A.out)) || (A.seqs > 0 && (!A.tables || !A.lens)) || (A.pages > 0 && !A.cache))
        return hd_fail(ctx, HD_E_ARG, "%s: null argument", name);
    int rc = hd_kv4_check(ctx, name, A.cache, A.pages, page_size, A.n_kv, hd);
    if (rc) return rc;
    HD_REQUIRE(ctx, A.n_heads > 0 && A.n_heads % A.n_kv == 0 && A.n_heads / A.n_kv <= MAXREP4, HD_E_SHAPE,
               "%s: n_heads %d must be a multiple of n_kv %d, at most %d per kv head", name, A.n_heads, A.n_kv, MAXREP4);
    HD_REQUIRE(ctx, A.seqs >= 0 && A.seqs < 1 << 30 && A.rows >= 0 && A.rows < ((int64_t)1 << 31) && A.max_pages > 0 &&
                        (int64_t)A.max_pages * page_size < ((int64_t)1 << 31),
               HD_E_SHAPE, "%s: bad shape (requests %d, rows %lld, table width %d)", name, A.seqs, (long long)A.rows,
               A.max_pages);
    HD_REQUIRE(ctx, A.window >= 0 && A.sinks >= 0 && A.scale >= 0.f && std::isfinite(A.scale), HD_E_ARG,
               "%s: window %d, sinks %d and scale %g must not be negative", name, A.window, A.sinks, (double)A.scale);
    if (A.q_ld == 0) A.q_ld = (int64_t)A.n_heads * hd;
    HD_REQUIRE(ctx, A.q_ld >= (int64_t)A.n_heads * hd, HD_E_SHAPE, "%s: row stride %lld of q", name, (long long)A.q_ld);
    HD_REQUIRE(ctx, A.q_ld % 4 == 0 && (((uintptr_t)A.q | (uintptr_t)A.out) & 15) == 0, HD_E_ARG,
               "%s: rows must be 16-byte aligned", name);
    if (!ctx) return HD_E_ARG;
    if (A.scale == 0.f) A.scale = 1.0f / sqrtf((float)hd);
    A.scale_m = frexpf(A.scale, &A.scale_e) * 1.4426950408889634f;
    A.shift = 4;
    while ((1 << A.shift) < page_size) A.shift++;
    return HD_OK;
}
