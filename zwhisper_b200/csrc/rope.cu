// Rotary positions of any layout (zwg_rope): pairs of halves or interleaved pairs, the first
// `rot` elements of a head, at positions of each sequence's own, on q and k in one launch.
//
//   a' = a cos - b sin,  b' = a sin + b cos,  (a, b) = (x[i], x[i + rot/2]) or (x[2i], x[2i + 1])
//
// in f32 with separately rounded products and sums, as rope_kt_append_kernel, so a rotation
// by this kernel and one by the fused projections give the same bits.
//
// Bound by memory: each row is read and written once, the tables come from L2 (all heads of
// a token share one row of them). A CTA takes one token; a thread takes 16-byte pieces, both
// sides of its pairs, so the loads and stores are whole 128-bit ones. Rows that are not
// aligned for that, and rotated parts that do not divide into it, take one element a time.
#include <cuda_bf16.h>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "seqs.cuh"

namespace zwg {
namespace {

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T e[N];
};

ZWG_DEV float up(float x) { return x; }
ZWG_DEV float up(__nv_bfloat16 x) { return __bfloat162float(x); }
ZWG_DEV void down(float x, float& y) { y = x; }
ZWG_DEV void down(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

ZWG_DEV float turn_a(float a, float b, float c, float s) { return __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s)); }
ZWG_DEV float turn_b(float a, float b, float c, float s) { return __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c)); }

// N: elements a thread moves at a time (16 bytes of them, or 1).
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(128) rope_kernel(RopeCall p) {
    chain_release();
    const int z = chain_wait();
    const int b = blockIdx.x / p.s.n, i = blockIdx.x % p.s.n;
    const Place at = place_of(p.s, b, p.t.n_ctx, threadIdx.x == 0 && i == 0 ? p.err : nullptr);
    if (i >= at.count) return;
    const int half = p.t.rot / 2;
    const float* cs = p.t.cos + (size_t)(at.past + i) * half + z;
    const float* sn = p.t.sin + (size_t)(at.past + i) * half + z;
    // pieces of a head: pairs of pieces (or one piece of pairs), then the part that stays
    const int turned = INTER ? (N > 1 ? p.t.rot / N : half) : half / N;
    const int rest = (p.d - p.t.rot) / N, per_head = turned + rest;
    const int all = (p.n_head + p.n_head_kv) * per_head;
    using V = Vec<T, N>;
    for (int idx = threadIdx.x; idx < all; idx += blockDim.x) {
        const int h = idx / per_head, u = idx % per_head;
        const bool is_q = h < p.n_head;
        const Rows& from = is_q ? p.q : p.k;
        const Rows& to = is_q ? p.q_out : p.k_out;
        const size_t hd = (size_t)(is_q ? h : h - p.n_head) * p.d;
        const T* x = static_cast<const T*>(from.data) + b * from.bs + i * from.ts + hd + z;
        T* y = static_cast<T*>(const_cast<void*>(to.data)) + b * to.bs + i * to.ts + hd + z;
        if (u >= turned) {
            const int e = p.t.rot + (u - turned) * N;
            *reinterpret_cast<V*>(y + e) = *reinterpret_cast<const V*>(x + e);
        } else if (!INTER) {
            const int e = u * N;
            const V a = *reinterpret_cast<const V*>(x + e), c = *reinterpret_cast<const V*>(x + half + e);
            V ra, rc;
#pragma unroll
            for (int j = 0; j < N; j++) {
                const float co = cs[e + j], si = sn[e + j];
                down(turn_a(up(a.e[j]), up(c.e[j]), co, si), ra.e[j]);
                down(turn_b(up(a.e[j]), up(c.e[j]), co, si), rc.e[j]);
            }
            *reinterpret_cast<V*>(y + e) = ra;
            *reinterpret_cast<V*>(y + half + e) = rc;
        } else if (N > 1) {
            const int e = u * N;
            const V a = *reinterpret_cast<const V*>(x + e);
            V r;
#pragma unroll
            for (int j = 0; j + 1 < N; j += 2) {
                const float co = cs[(e + j) / 2], si = sn[(e + j) / 2];
                down(turn_a(up(a.e[j]), up(a.e[j + 1]), co, si), r.e[j]);
                down(turn_b(up(a.e[j]), up(a.e[j + 1]), co, si), r.e[j + 1]);
            }
            *reinterpret_cast<V*>(y + e) = r;
        } else {
            const float a = up(x[2 * u]), c = up(x[2 * u + 1]);
            down(turn_a(a, c, cs[u], sn[u]), y[2 * u]);
            down(turn_b(a, c, cs[u], sn[u]), y[2 * u + 1]);
        }
    }
}

bool aligned(const Rows& r, size_t elem) {
    return ((uintptr_t)r.data | (r.bs * elem) | (r.ts * elem)) % 16 == 0;
}

template <typename T>
int launch(const RopeCall& p, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const bool vec = aligned(p.q, sizeof(T)) && aligned(p.q_out, sizeof(T)) && aligned(p.k, sizeof(T)) &&
                     aligned(p.k_out, sizeof(T)) && p.d % N == 0 && (p.t.interleaved ? p.t.rot : p.t.rot / 2) % N == 0;
    void (*kern)(RopeCall) = p.t.interleaved ? (vec ? rope_kernel<T, N, true> : rope_kernel<T, 1, true>)
                                             : (vec ? rope_kernel<T, N, false> : rope_kernel<T, 1, false>);
    return launch_chained(kern, dim3((unsigned)p.s.n_batch * p.s.n), dim3(128), st, p) == cudaSuccess ? 0 : -1;
}

}  // namespace

int rope_launch(const RopeCall& p, int type, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    return type == TYPE_BF16 ? launch<__nv_bfloat16>(p, st) : launch<float>(p, st);
}

}  // namespace zwg
