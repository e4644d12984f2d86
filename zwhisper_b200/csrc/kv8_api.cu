// C-ABI entry points of the decode step over a cache in 8 bits (include/zwgpu.h): zwg_rope,
// zwg_kv8_append / _read / _attn, zwg_llm_logits, and the states that keep such caches. Every
// call checks its arguments, before it asks for a context, then launches on the caller's stream:
// no allocation (but for a state's creation), no synchronization.
#include <cuda_runtime.h>

#include <cmath>
#include <utility>

#include "../../include/zwgpu.h"
#include "api_internal.h"
#include "kernels.h"

using namespace zwg::capi;

namespace {

constexpr size_t kMost = (size_t)1 << 30;

size_t type_size(int type) { return type == ZWG_TYPE_F32 ? 4 : type == ZWG_TYPE_BF16 ? 2 : 0; }

bool al(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

int check_seqs(const zwg_seqs* s, size_t room, const char* what) {
    if (!s) return fail("%s: null seqs", what);
    if (s->n_batch >= kMost || s->n >= kMost || s->n_batch * s->n >= kMost) return fail("%s: too many tokens", what);
    if (s->n_past > room || (!s->past && !s->count && s->n_past + s->n > room))
        return fail("%s: context full (%zu + %zu > %zu)", what, s->n_past, s->n, room);
    if (!al(s->past, 4) || !al(s->count, 4) || !al(s->first, 4)) return fail("%s: past, count and first must be 4-byte aligned", what);
    return ZWG_OK;
}

zwg::Seqs seqs_of(const zwg_seqs* s) {
    return zwg::Seqs{(int)s->n_batch, (int)s->n, (int)s->n_past, s->past, s->count, s->first};
}

int check_rows(const zwg_rows* r, const zwg_seqs* s, size_t width, int type, bool written, const char* what, const char* name) {
    if (!r || !r->data) return fail("%s: null %s", what, name);
    if (!al(r->data, type_size(type))) return fail("%s: %s must be aligned to its elements", what, name);
    if (r->batch_stride >= ((size_t)1 << 60) / (s->n_batch + 1) || r->token_stride >= ((size_t)1 << 60) / (s->n + 1))
        return fail("%s: %s strides too large", what, name);
    if (written) {  // rows that are written may not overlap
        size_t inner = r->token_stride, n_inner = s->n, outer = r->batch_stride, n_outer = s->n_batch;
        if (n_inner > 1 && n_outer > 1 && inner > outer) {
            std::swap(inner, outer);
            std::swap(n_inner, n_outer);
        }
        if ((n_inner > 1 && inner < width) || (n_outer > 1 && outer < (n_inner > 1 ? inner * (n_inner - 1) : 0) + width))
            return fail("%s: %s rows overlap (strides %zu, %zu for rows of %zu)", what, name, r->batch_stride, r->token_stride, width);
    }
    return ZWG_OK;
}

zwg::Rows rows_of(const zwg_rows* r) { return zwg::Rows{r->data, r->batch_stride, r->token_stride}; }

int check_type(int type, const char* what) {
    return type_size(type) ? ZWG_OK : fail("%s: type %d is neither ZWG_TYPE_F32 nor ZWG_TYPE_BF16", what, type);
}

int check_tables(const zwg_rope_tables* t, size_t d, const char* what) {
    if (!t || !t->cos || !t->sin) return fail("%s: null rotary tables", what);
    if (!al(t->cos, 4) || !al(t->sin, 4)) return fail("%s: rotary tables must be 4-byte aligned", what);
    if (t->rot == 0 || t->rot % 2 || t->rot > d) return fail("%s: rot = %zu must be even and at most d = %zu", what, t->rot, d);
    if (t->n_ctx >= kMost) return fail("%s: rotary tables too long", what);
    return ZWG_OK;
}

zwg::RopeTables tables_of(const zwg_rope_tables* t) {
    return zwg::RopeTables{t->cos, t->sin, (int)t->n_ctx, (int)t->rot, t->interleaved ? 1 : 0};
}

int check_cache(const zwg_kv8* c, const char* what) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_open || !c->v_open || !c->open_block)
        return fail("%s: null cache buffer", what);
    if (!al(c->k, 16) || !al(c->v, 16) || !al(c->k_open, 16) || !al(c->v_open, 16))
        return fail("%s: int8 and open rows of the cache must be 16-byte aligned", what);
    if (!al(c->k_scale, 4) || !al(c->v_scale, 4) || !al(c->open_block, 4)) return fail("%s: cache scales must be 4-byte aligned", what);
    if (c->d != 64 && c->d != 128) return fail("%s: d = %zu, the cache in 8 bits has 64 or 128", what, c->d);
    if (c->n_ctx == 0 || c->n_ctx % 32 || c->n_ctx >= kMost) return fail("%s: n_ctx = %zu must be a positive multiple of 32", what, c->n_ctx);
    if (c->n_head_kv == 0 || c->n_batch >= kMost || c->n_head_kv >= kMost || c->n_batch * c->n_head_kv > 65535)
        return fail("%s: n_batch * n_head_kv = %zu * %zu must be at most 65535", what, c->n_batch, c->n_head_kv);
    return ZWG_OK;
}

int check_batch(const zwg_kv8* c, const zwg_seqs* s, const char* what) {
    return s->n_batch == c->n_batch ? ZWG_OK : fail("%s: %zu sequences, the cache has %zu", what, s->n_batch, c->n_batch);
}

zwg::Kv8 cache_of(const zwg_kv8* c) {
    return zwg::Kv8{c->k, c->k_scale, c->v, c->v_scale, c->k_open, c->v_open, c->open_block,
                    (int)c->n_head_kv, (int)c->d, (int)(c->n_ctx / 32)};
}

int check_heads(const zwg_kv8* c, const zwg_seqs* s, size_t n_head, const char* what) {
    if (n_head == 0 || n_head >= kMost || n_head % c->n_head_kv)
        return fail("%s: n_head %zu must be a positive multiple of n_head_kv %zu", what, n_head, c->n_head_kv);
    if (s->n * n_head >= kMost) return fail("%s: too many query rows", what);
    return ZWG_OK;
}

size_t attn_workspace(const zwg_kv8* c, const zwg_seqs* s, size_t n_head, int sm_count) {
    return zwg::kv8_attn_workspace_bytes(cache_of(c), seqs_of(s), (int)n_head, sm_count);
}

}  // namespace

// The state's calls (state.cu, llm_api.cu) on a cache in 8 bits.
int zwg::capi::kv8_llm_append(zwg_llm_state* st, size_t layer, float* q, const float* k, const float* v, size_t n_past,
                              size_t n, cudaStream_t s) {
    if (n > st->n_chunk) return fail("llm_append_rope: %zu tokens, the state was made for chunks of %zu", n, st->n_chunk);
    const size_t w = st->n_head * st->d, kvw = st->n_head_kv * st->d;
    const zwg_seqs sq{st->n_batch, n, n_past, nullptr, nullptr, nullptr};
    const zwg_rope_tables t{st->cos_tab, st->sin_tab, st->n_ctx, st->d, 0};
    const zwg_rows qr{q, n * w, w}, kr{const_cast<float*>(k), n * kvw, kvw}, vr{const_cast<float*>(v), n * kvw, kvw};
    int rc = zwg_rope(&sq, &t, ZWG_TYPE_F32, st->d, st->n_head, &qr, nullptr, 0, nullptr, nullptr, s);
    if (!rc) rc = zwg_kv8_append(&st->kv8[layer], &sq, ZWG_TYPE_F32, &kr, &vr, &t, s);
    return rc;
}

int zwg::capi::kv8_llm_append_staged(zwg_llm_state* st, size_t layer, size_t n_past, size_t n, cudaStream_t s) {
    Ctx* c = ctx_for(st->device);
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    const size_t kvw = st->n_head_kv * st->d, pitch = st->stage_pitch(n);
    zwg::Kv8Append p{};
    p.c = cache_of(&st->kv8[layer]);
    p.s = zwg::Seqs{(int)st->n_batch, (int)n, (int)n_past, nullptr, nullptr, nullptr};
    p.k = zwg::Rows{st->stage_kt, kvw * pitch, 1};
    p.k_hs = st->d * pitch;
    p.k_es = pitch;
    p.v = zwg::Rows{st->stage_v, kvw * pitch, kvw};
    p.v_hs = st->d;
    p.err = c->err;
    if (zwg::kv8_append_launch(p, ZWG_TYPE_F32, s)) return cuda_fail("kv8 append launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg::capi::kv8_llm_attn(zwg_llm_state* st, size_t layer, const float* q, size_t n_past, size_t n, float* out,
                            cudaStream_t s) {
    if (n > st->n_chunk) return fail("llm attention: %zu tokens, the state was made for chunks of %zu", n, st->n_chunk);
    const size_t w = st->n_head * st->d;
    const zwg_seqs sq{st->n_batch, n, n_past, nullptr, nullptr, nullptr};
    const zwg_rows qr{const_cast<float*>(q), n * w, w}, o{out, n * w, w};
    return zwg_kv8_attn(&st->kv8[layer], &sq, ZWG_TYPE_F32, st->n_head, &qr, &o, st->ws.ptr, st->ws.cap, s);
}

extern "C" {

int zwg_rope(const zwg_seqs* s, const zwg_rope_tables* t, int type, size_t d, size_t n_head, const zwg_rows* q,
             const zwg_rows* q_out, size_t n_head_kv, const zwg_rows* k, const zwg_rows* k_out, void* stream) {
    if (d == 0 || d > 1024 || n_head == 0 || n_head >= kMost / d || n_head_kv >= kMost / d || n_head + n_head_kv > 65536) return fail("rope: bad head sizes");
    int rc = check_type(type, "rope");
    if (!rc) rc = check_tables(t, d, "rope");
    if (!rc) rc = check_seqs(s, t->n_ctx, "rope");
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    if (!q_out) q_out = q;
    if (!k_out) k_out = k;
    rc = check_rows(q, s, n_head * d, type, false, "rope", "q");
    if (!rc) rc = check_rows(q_out, s, n_head * d, type, true, "rope", "q_out");
    if (!rc && k) rc = check_rows(k, s, n_head_kv * d, type, false, "rope", "k");
    if (!rc && k) rc = check_rows(k_out, s, n_head_kv * d, type, true, "rope", "k_out");
    if (rc) return rc;
    if (!k && k_out) return fail("rope: k_out without k");
    if (s->n * (n_head + (k ? n_head_kv : 0)) >= kMost / d) return fail("rope: too many elements in a sequence");
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    zwg::RopeCall p{};
    p.s = seqs_of(s);
    p.t = tables_of(t);
    p.d = (int)d;
    p.n_head = (int)n_head;
    p.n_head_kv = k ? (int)n_head_kv : 0;
    p.q = rows_of(q);
    p.q_out = rows_of(q_out);
    if (k) {
        p.k = rows_of(k);
        p.k_out = rows_of(k_out);
    }
    p.err = c->err;
    if (zwg::rope_launch(p, type, (cudaStream_t)stream)) return cuda_fail("rope launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg_kv8_append(const zwg_kv8* cache, const zwg_seqs* s, int type, const zwg_rows* k, const zwg_rows* v,
                   const zwg_rope_tables* rope, void* stream) {
    int rc = check_cache(cache, "kv8_append");
    if (!rc) rc = check_type(type, "kv8_append");
    if (!rc) rc = check_seqs(s, cache->n_ctx, "kv8_append");
    if (!rc) rc = check_batch(cache, s, "kv8_append");
    if (!rc && rope) rc = check_tables(rope, cache->d, "kv8_append");
    if (!rc && rope) rc = check_seqs(s, rope->n_ctx, "kv8_append: rotary tables");
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    const size_t w = cache->n_head_kv * cache->d;
    rc = check_rows(k, s, w, type, false, "kv8_append", "k");
    if (!rc) rc = check_rows(v, s, w, type, false, "kv8_append", "v");
    if (rc) return rc;
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    zwg::Kv8Append p{};
    p.c = cache_of(cache);
    p.s = seqs_of(s);
    p.k = rows_of(k);
    p.v = rows_of(v);
    p.k_hs = p.v_hs = cache->d;
    p.k_es = 1;
    if (rope) p.rope = tables_of(rope);
    p.err = c->err;
    if (zwg::kv8_append_launch(p, type, (cudaStream_t)stream)) return cuda_fail("kv8_append launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg_kv8_read(const zwg_kv8* cache, const zwg_seqs* s, float* k, float* v, void* stream) {
    int rc = check_cache(cache, "kv8_read");
    if (!rc) rc = check_seqs(s, cache->n_ctx, "kv8_read");
    if (!rc) rc = check_batch(cache, s, "kv8_read");
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    if (!al(k, 16) || !al(v, 16)) return fail("kv8_read: k and v must be 16-byte aligned");
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    if (zwg::kv8_read_launch(cache_of(cache), seqs_of(s), k, v, c->err, (cudaStream_t)stream))
        return cuda_fail("kv8_read launch", cudaGetLastError());
    return ZWG_OK;
}

size_t zwg_kv8_attn_workspace(const zwg_kv8* cache, const zwg_seqs* s, size_t n_head) {
    Ctx* c = cur();
    if (!c || check_cache(cache, "kv8_attn") || check_seqs(s, cache->n_ctx, "kv8_attn") || check_batch(cache, s, "kv8_attn") ||
        check_heads(cache, s, n_head, "kv8_attn"))
        return 0;
    const OnDevice on(c->device);
    return attn_workspace(cache, s, n_head, c->sm_count);
}

int zwg_kv8_attn(const zwg_kv8* cache, const zwg_seqs* s, int type, size_t n_head, const zwg_rows* q, const zwg_rows* out,
                 void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_cache(cache, "kv8_attn");
    if (!rc) rc = check_type(type, "kv8_attn");
    if (!rc) rc = check_seqs(s, cache->n_ctx, "kv8_attn");
    if (!rc) rc = check_batch(cache, s, "kv8_attn");
    if (!rc) rc = check_heads(cache, s, n_head, "kv8_attn");
    if (rc || s->n_batch == 0 || s->n == 0) return rc;
    const size_t w = n_head * cache->d;
    rc = check_rows(q, s, w, type, false, "kv8_attn", "q");
    if (!rc) rc = check_rows(out, s, w, type, true, "kv8_attn", "out");
    if (rc) return rc;
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    const size_t need = attn_workspace(cache, s, n_head, c->sm_count);
    if (need && (!workspace || workspace_bytes < need))
        return fail("kv8_attn: workspace of %zu bytes, %zu needed", workspace ? workspace_bytes : 0, need);
    if (!al(workspace, 16)) return fail("kv8_attn: workspace must be 16-byte aligned");
    zwg::Kv8Attn p{};
    p.c = cache_of(cache);
    p.s = seqs_of(s);
    p.n_head = (int)n_head;
    p.q = rows_of(q);
    p.out = rows_of(out);
    p.ws = (float*)workspace;
    p.err = c->err;
    const int pieces = c->math & ZWG_MATH_TF32 ? 1 : 2;
    if (zwg::kv8_attn_launch(p, type, pieces, c->sm_count, (cudaStream_t)stream))
        return cuda_fail("kv8_attn launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg_llm_logits(float* logits, size_t m, size_t n_vocab, size_t stride, const zwg_logit_rules* r, int32_t* out,
                   size_t out_stride, void* stream) {
    if (!r) return fail("llm_logits: null rules");
    if (n_vocab == 0 || n_vocab >= kMost || m >= kMost) return fail("llm_logits: bad sizes (%zu rows of %zu)", m, n_vocab);
    if (m == 0) return ZWG_OK;
    if (!logits) return fail("llm_logits: null logits");
    if (stride < n_vocab && m > 1) return fail("llm_logits: row stride %zu below the vocabulary's %zu", stride, n_vocab);
    if (r->n_recent && !r->recent) return fail("llm_logits: null recent tokens");
    if (r->n_recent >= kMost) return fail("llm_logits: too many recent tokens");
    if ((r->window < r->n_recent ? r->window : r->n_recent) >= (1u << 19))
        return fail("llm_logits: a window of %zu tokens, at most 524287 are taken", r->window);
    if (r->n_bias > ZWG_MAX_BIAS) return fail("llm_logits: %zu biases, at most %d are taken", r->n_bias, ZWG_MAX_BIAS);
    if (r->n_bias && (!r->bias_ids || !r->bias)) return fail("llm_logits: null biases");
    if (!(r->repeat > 0.f) || !std::isfinite(r->repeat) || !std::isfinite(1.f / r->repeat) || !std::isfinite(r->presence) || !std::isfinite(r->frequency))
        return fail("llm_logits: repeat must be positive, all penalties finite");
    if (out && out_stride == 0 && m > 1) return fail("llm_logits: out needs a stride");
    if (!al(logits, 4) || !al(out, 4) || !al(r->recent, 4) || !al(r->n_recents, 4) || !al(r->bias_ids, 4) ||
        !al(r->bias, 4) || !al(r->allow, 4))
        return fail("llm_logits: 4-byte alignment required");
    Ctx* c = cur();
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    const size_t window = r->window < r->n_recent ? r->window : r->n_recent;
    zwg::LogitRules p{r->recent, r->recent_stride, window ? (int)r->n_recent : 0, window ? r->n_recents : nullptr,
                      (int)window, r->repeat, 1.f / r->repeat, r->presence, r->frequency, r->bias_ids, r->bias,
                      (int)r->n_bias, r->bias_stride, r->allow, r->allow_stride};
    if (zwg::logit_rules_launch(logits, m, (int)n_vocab, stride, p, out, out_stride, c->sm_count, c->err, (cudaStream_t)stream))
        return cuda_fail("llm_logits launch", cudaGetLastError());
    return ZWG_OK;
}

int zwg_llm_state_kv8(const zwg_llm_state* st, size_t layer, zwg_kv8* out) {
    if (!st || layer >= st->n_layer || !out) return fail("llm_state_kv8: bad arguments");
    if (st->kv8.empty()) return fail("llm_state_kv8: the state's caches are f32");
    *out = st->kv8[layer];
    return ZWG_OK;
}

int zwg_llm_state_set_rope(zwg_llm_state* st, const float* cos, const float* sin, void* stream) {
    if (!st || !cos || !sin) return fail("llm_state_set_rope: null state or tables");
    Ctx* c = ctx_for(st->device);
    if (!c) return ZWG_ERROR;
    const OnDevice on(c->device);
    const size_t bytes = st->n_ctx * (st->d / 2) * sizeof(float);
    cudaError_t e = cudaMemcpyAsync(st->cos_tab, cos, bytes, cudaMemcpyDefault, (cudaStream_t)stream);
    if (e == cudaSuccess) e = cudaMemcpyAsync(st->sin_tab, sin, bytes, cudaMemcpyDefault, (cudaStream_t)stream);
    return e == cudaSuccess ? ZWG_OK : cuda_fail("llm_state_set_rope copy", e);
}

}  // extern "C"
