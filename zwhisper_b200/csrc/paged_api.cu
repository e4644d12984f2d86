// C-ABI entry points of the cache in pages and of trees of drafted tokens (include/zwgpu.h): zwg_paged_append /
// _attn / _keep and zwg_tree_accept. Every call checks its arguments, before it asks for a context, then launches
// on the caller's stream: no allocation, no synchronization.
#include <cuda_runtime.h>

#include "../../include/zwgpu.h"
#include "api_internal.h"
#include "kernels.h"
#include "seqs_api.h"

using namespace zwg::capi;

namespace {

int check_cache(const zwg_paged* c, const char* what) {
    if (!c || !c->k || !c->v || !c->table) return fail("%s: null cache buffer", what);
    if (c->type != ZWG_TYPE_F16 && c->type != ZWG_TYPE_BF16)
        return fail("%s: a cache in pages is of ZWG_TYPE_F16 or ZWG_TYPE_BF16, not %d", what, c->type);
    if (!al(c->k, 16) || !al(c->v, 16)) return fail("%s: k and v of the cache must be 16-byte aligned", what);
    if (!al(c->table, 4)) return fail("%s: the table must be 4-byte aligned", what);
    if (c->d != 64 && c->d != 128) return fail("%s: d = %zu, the cache in pages has 64 or 128", what, c->d);
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1)))
        return fail("%s: page = %zu must be a power of two from 16 to 256", what, c->page);
    if (c->n_pages == 0 || c->n_pages >= kMost) return fail("%s: n_pages = %zu must be positive and below 2^30", what, c->n_pages);
    if (c->max_pages == 0 || c->max_pages >= kMost / c->page)
        return fail("%s: max_pages = %zu must be positive, and max_pages * page below 2^30", what, c->max_pages);
    if (c->n_head_kv == 0 || c->n_batch >= kMost || c->n_head_kv >= kMost || c->n_batch * c->n_head_kv > 65535)
        return fail("%s: n_batch * n_head_kv = %zu * %zu must be at most 65535", what, c->n_batch, c->n_head_kv);
    if (c->page_stride % 8 || c->page_stride < c->n_head_kv * c->page * c->d || c->page_stride >= (size_t)1 << 38)
        return fail("%s: page_stride = %zu must be a multiple of 8, at least a page's %zu elements and below 2^38", what, c->page_stride,
                    c->n_head_kv * c->page * c->d);
    if ((c->n_batch > 1 && c->table_stride < c->max_pages) || c->table_stride > ((size_t)1 << 60) / (c->n_batch + 1))
        return fail("%s: table_stride = %zu below the row's %zu entries, or too large", what, c->table_stride, c->max_pages);
    return ZWG_OK;
}

size_t room_of(const zwg_paged* c) { return c->max_pages * c->page; }

int check_call(const zwg_paged* c, const zwg_seqs* s, const char* what) {
    int rc = check_cache(c, what);
    if (!rc) rc = check_seqs(s, room_of(c), what);
    if (!rc && s->n_batch != c->n_batch) rc = fail("%s: %zu sequences, the cache has %zu", what, s->n_batch, c->n_batch);
    return rc;
}

int check_tree(const zwg_tree* t, const zwg_seqs* s, const char* what) {
    if (!t) return ZWG_OK;
    if (!t->parent && s->n) return fail("%s: null parents", what);
    if (!al(t->parent, 4)) return fail("%s: parents must be 4-byte aligned", what);
    if (s->n > ZWG_MAX_TREE) return fail("%s: a tree of %zu tokens, at most %d are taken", what, s->n, ZWG_MAX_TREE);
    if (t->batch_stride > ((size_t)1 << 60) / (s->n_batch + 1)) return fail("%s: parents' stride too large", what);
    return ZWG_OK;
}

int check_pair(const zwg_paged* c, int type, const char* what) {
    int rc = check_type(type, what);
    if (!rc && (type == ZWG_TYPE_BF16) != (c->type == ZWG_TYPE_BF16))
        rc = fail("%s: f32 rows go with an f16 cache, bf16 rows with a bf16 one", what);
    return rc;
}

zwg::Paged cache_of(const zwg_paged* c) {
    int log_page = 4;
    while (((size_t)1 << log_page) < c->page) log_page++;
    return zwg::Paged{c->k, c->v, c->table, c->table_stride, c->page_stride, (int)c->n_head_kv, (int)c->d, log_page,
                      (int)c->n_pages, (int)room_of(c), c->type == ZWG_TYPE_BF16 ? zwg::TYPE_BF16 : zwg::TYPE_F16};
}

zwg::Tree tree_of(const zwg_tree* t) { return t ? zwg::Tree{t->parent, t->batch_stride} : zwg::Tree{nullptr, 0}; }

int check_heads(const zwg_paged* c, const zwg_seqs* s, size_t n_head, const char* what) {
    if (n_head == 0 || n_head >= kMost || n_head % c->n_head_kv)
        return fail("%s: n_head %zu must be a positive multiple of n_head_kv %zu", what, n_head, c->n_head_kv);
    if (s->n && n_head >= kMost / s->n) return fail("%s: too many query rows", what);
    return ZWG_OK;
}

}  // namespace

extern "C" {

int zwg_paged_append(const zwg_paged* cache, const zwg_seqs* s, const zwg_tree* tree, int type, const zwg_rows* k,
                     const zwg_rows* v, const zwg_rope_tables* rope, size_t n_head, const zwg_rows* q, const zwg_rows* q_out,
                     void* stream) {
    const char* what = "paged_append";
    int rc = check_call(cache, s, what);
    if (!rc) rc = check_tree(tree, s, what);
    if (!rc) rc = check_pair(cache, type, what);
    if (!rc && rope) rc = check_tables(rope, cache->d, what);
    if (!rc && rope) rc = check_seqs(s, rope->n_ctx, "paged_append: rotary tables");
    if (!rc && !q && q_out) rc = fail("%s: q_out without q", what);
    if (!rc && q && !rope) rc = fail("%s: q is given to be rotated, without rotary tables", what);
    if (!rc && q && (n_head == 0 || n_head > 65536)) rc = fail("%s: bad head sizes", what);
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    const size_t w = cache->n_head_kv * cache->d;
    rc = check_rows(k, s, w, type, false, what, "k");
    if (!rc) rc = check_rows(v, s, w, type, false, what, "v");
    if (!q_out) q_out = q;
    if (!rc && q) rc = check_rows(q, s, n_head * cache->d, type, false, what, "q");
    if (!rc && q) rc = check_rows(q_out, s, n_head * cache->d, type, true, what, "q_out");
    if (!rc && cache->k == cache->v) rc = fail("%s: k and v of the cache are one buffer", what);
    if (rc) return rc;
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    zwg::PagedAppend p{};
    p.c = cache_of(cache);
    p.s = seqs_of(s);
    p.tree = tree_of(tree);
    p.n_head = q ? (int)n_head : 0;
    if (q) {
        p.q = rows_of(q);
        p.q_out = rows_of(q_out);
    }
    p.k = rows_of(k);
    p.v = rows_of(v);
    if (rope) p.rope = tables_of(rope);
    p.err = c->err;
    if (zwg::paged_append_launch(p, type, (cudaStream_t)stream)) return cuda_fail("paged_append launch", cudaGetLastError());
    return ZWG_OK;
}

size_t zwg_paged_attn_workspace(const zwg_paged* cache, const zwg_seqs* s, size_t n_head) {
    Ctx* c = cur();
    if (!c || check_call(cache, s, "paged_attn") || check_heads(cache, s, n_head, "paged_attn")) return 0;
    const OnDevice on(c->device);
    return zwg::paged_attn_workspace_bytes(cache_of(cache), seqs_of(s), (int)n_head, c->sm_count);
}

int zwg_paged_attn(const zwg_paged* cache, const zwg_seqs* s, const zwg_tree* tree, int type, size_t n_head, const zwg_rows* q,
                   const zwg_rows* out, void* workspace, size_t workspace_bytes, void* stream) {
    const char* what = "paged_attn";
    int rc = check_call(cache, s, what);
    if (!rc) rc = check_tree(tree, s, what);
    if (!rc) rc = check_pair(cache, type, what);
    if (!rc) rc = check_heads(cache, s, n_head, what);
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    rc = check_rows(q, s, n_head * cache->d, type, false, what, "q");
    if (!rc) rc = check_rows(out, s, n_head * cache->d, type, true, what, "out");
    if (rc) return rc;
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    zwg::PagedAttn p{};
    p.c = cache_of(cache);
    p.s = seqs_of(s);
    const size_t need = zwg::paged_attn_workspace_bytes(p.c, p.s, (int)n_head, c->sm_count);
    if (need && (!workspace || workspace_bytes < need))
        return fail("%s: workspace of %zu bytes, %zu needed", what, workspace ? workspace_bytes : 0, need);
    if (!al(workspace, 16)) return fail("%s: workspace must be 16-byte aligned", what);
    p.tree = tree_of(tree);
    p.n_head = (int)n_head;
    p.q = rows_of(q);
    p.out = rows_of(out);
    p.ws = (float*)workspace;
    p.err = c->err;
    if (zwg::paged_attn_launch(p, type, c->math & ZWG_MATH_TF32 ? 1 : 2, c->sm_count, (cudaStream_t)stream))
        return cuda_fail("paged_attn launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg_tree_accept(const zwg_seqs* s, const zwg_tree* tree, const int32_t* tokens, const int32_t* ids, int32_t* path,
                    int32_t* n_path, int32_t* next, void* stream) {
    const char* what = "tree_accept";
    if (!s || !tree) return fail("%s: null seqs or tree", what);
    zwg_seqs sq{s->n_batch, s->n, 0, nullptr, s->count, nullptr};
    int rc = check_seqs(&sq, kMost, what);
    if (!rc) rc = check_tree(tree, &sq, what);
    if (rc || s->n_batch == 0) return rc;
    if ((s->n && (!tokens || !ids || !path)) || !n_path || !next) return fail("%s: null buffer", what);
    if (!al(tokens, 4) || !al(ids, 4) || !al(path, 4) || !al(n_path, 4) || !al(next, 4)) return fail("%s: 4-byte alignment required", what);
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    zwg::TreeAccept p{seqs_of(&sq), tree_of(tree), tokens, ids, path, n_path, next, c->err};
    if (zwg::tree_accept_launch(p, (cudaStream_t)stream)) return cuda_fail("tree_accept launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg_paged_keep(const zwg_paged* caches, size_t n_caches, const zwg_seqs* s, const int32_t* path, const int32_t* n_path,
                   void* stream) {
    const char* what = "paged_keep";
    if (n_caches && !caches) return fail("%s: null caches", what);
    int rc = ZWG_OK;
    for (size_t i = 0; i < n_caches && !rc; i++) {
        const zwg_paged &a = caches[i], &o = caches[0];
        rc = check_cache(&a, what);
        if (!rc && (a.type != o.type || a.table != o.table || a.table_stride != o.table_stride || a.n_batch != o.n_batch ||
                    a.n_head_kv != o.n_head_kv || a.d != o.d || a.page != o.page || a.n_pages != o.n_pages ||
                    a.max_pages != o.max_pages || a.page_stride != o.page_stride))
            rc = fail("%s: cache %zu differs from the first one in more than k and v", what, i);
    }
    if (rc || n_caches == 0) return rc;
    zwg_seqs sq{0, 0, 0, nullptr, n_path, nullptr};
    if (!s) return fail("%s: null seqs", what);
    sq.n_batch = s->n_batch;
    sq.n = s->n;
    sq.n_past = s->n_past;
    sq.past = s->past;
    rc = check_call(&caches[0], &sq, what);
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    if (s->n > ZWG_MAX_TREE) return fail("%s: %zu tokens, at most %d are taken", what, s->n, ZWG_MAX_TREE);
    if (!path || !n_path) return fail("%s: null path", what);
    if (!al(path, 4)) return fail("%s: path must be 4-byte aligned", what);
    for (size_t i = 0; i < n_caches; i++) {  // rows that were moved may not be moved again
        const void *k = caches[i].k, *v = caches[i].v;
        bool twice = k == v;
        for (size_t j = 0; j < i; j++) twice |= caches[j].k == k || caches[j].v == k || caches[j].k == v || caches[j].v == v;
        if (twice) return fail("%s: a buffer of cache %zu is given twice", what, i);
    }
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    for (size_t i = 0; i < n_caches; i += zwg::MOST_KEPT) {
        zwg::PagedKeep p{};
        p.c = cache_of(&caches[0]);
        p.s = seqs_of(&sq);
        p.path = path;
        p.n_path = n_path;
        p.n = (int)std::min<size_t>(zwg::MOST_KEPT, n_caches - i);
        for (int j = 0; j < p.n; j++) {
            p.k[j] = caches[i + j].k;
            p.v[j] = caches[i + j].v;
        }
        p.err = c->err;
        if (zwg::paged_keep_launch(p, (cudaStream_t)stream)) return cuda_fail("paged_keep launch", cudaGetLastError());
    }
    return ZWG_OK;
}

}  // extern "C"
