// Checks and conversions of the arguments that the calls on sequences of tokens share (zwg_seqs, zwg_rows,
// zwg_rope_tables): kv8_api.cu, paged_api.cu.
#pragma once
#include <utility>

#include "../../include/zwgpu.h"
#include "api_internal.h"
#include "kernels.h"

namespace zwg {
namespace capi {

constexpr size_t kMost = (size_t)1 << 30;

inline size_t type_size(int type) { return type == ZWG_TYPE_F32 ? 4 : type == ZWG_TYPE_BF16 ? 2 : 0; }

inline bool al(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

inline int check_seqs(const zwg_seqs* s, size_t room, const char* what) {
    if (!s) return fail("%s: null seqs", what);
    if (s->n_batch >= kMost || s->n >= kMost || s->n_batch * s->n >= kMost) return fail("%s: too many tokens", what);
    if (s->n_past > room || (!s->past && !s->count && s->n_past + s->n > room))
        return fail("%s: context full (%zu + %zu > %zu)", what, s->n_past, s->n, room);
    if (!al(s->past, 4) || !al(s->count, 4) || !al(s->first, 4)) return fail("%s: past, count and first must be 4-byte aligned", what);
    return ZWG_OK;
}

inline zwg::Seqs seqs_of(const zwg_seqs* s) {
    return zwg::Seqs{(int)s->n_batch, (int)s->n, (int)s->n_past, s->past, s->count, s->first};
}

inline int check_rows(const zwg_rows* r, const zwg_seqs* s, size_t width, int type, bool written, const char* what, const char* name) {
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

inline zwg::Rows rows_of(const zwg_rows* r) { return zwg::Rows{r->data, r->batch_stride, r->token_stride}; }

inline int check_type(int type, const char* what) {
    return type_size(type) ? ZWG_OK : fail("%s: type %d is neither ZWG_TYPE_F32 nor ZWG_TYPE_BF16", what, type);
}

inline int check_tables(const zwg_rope_tables* t, size_t d, const char* what) {
    if (!t || !t->cos || !t->sin) return fail("%s: null rotary tables", what);
    if (!al(t->cos, 4) || !al(t->sin, 4)) return fail("%s: rotary tables must be 4-byte aligned", what);
    if (t->rot == 0 || t->rot % 2 || t->rot > d) return fail("%s: rot = %zu must be even and at most d = %zu", what, t->rot, d);
    if (t->n_ctx >= kMost) return fail("%s: rotary tables too long", what);
    return ZWG_OK;
}

inline zwg::RopeTables tables_of(const zwg_rope_tables* t) {
    return zwg::RopeTables{t->cos, t->sin, (int)t->n_ctx, (int)t->rot, t->interleaved ? 1 : 0};
}

}  // namespace capi
}  // namespace zwg
