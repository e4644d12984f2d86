// Rotary positions of any layout (zwg_rope): pairs of halves or interleaved pairs, the first
// `rot` elements of a head, at positions of each sequence's own, on q and k in one launch.
//
//   a' = a cos - b sin,  b' = a sin + b cos,  (a, b) = (x[i], x[i + rot/2]) or (x[2i], x[2i + 1])
//
// in f32 with separately rounded products and sums, as rope_kt_append_kernel, so a rotation
// by this kernel and one by the fused projections give the same bits.
//
// Bound by memory: each row is read and written once. A thread takes one piece of 16 bytes (or,
// where pairs are halves, both sides' pieces) of up to eight (four) heads of a token: they share its
// table entries, its loads are whole 128-bit ones and all on their way before the first is used.
// Rows that are not aligned for that, and rotated parts that do not divide into it, go one element
// at a time. 64 sequences x 256 tokens of 12 + 2 heads of d 128 in bf16 (117 MB in and out): 17.9 us,
// 6.5 TB/s, what a copy gets (31 us an element at a time; 12.5 us out of L2, pairs of either kind); one
// token of 16 sequences: 1.6 us, a launch.
#include <cuda_bf16.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "seqs.cuh"

namespace zwg {
namespace {

template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec {
    T e[N];
};

ZWG_DEV float up(float x) { return x; }
ZWG_DEV float up(__nv_bfloat16 x) { return __bfloat162float(x); }
ZWG_DEV void down(float x, float& y) { y = x; }
ZWG_DEV void down(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

// Heads of a thread: eight pieces of 16 bytes on their way.
constexpr int heads_of(bool one) { return one ? 8 : 4; }

// x / d for x < 2^31, as a multiplication.
struct Divisor {
    uint32_t d, mul, shift;
    explicit Divisor(uint32_t n) : d(n), mul(0), shift(0) {
        while ((1ull << shift) < n) shift++;
        mul = (uint32_t)(((1ull << 32) * ((1ull << shift) - n)) / n + 1);
    }
    ZWG_DEV uint32_t div(uint32_t x) const { return (__umulhi(x, mul) + x) >> shift; }
};

// C pairs, products and sums rounded one by one (the packed f32x2 forms would be contracted).
template <int C>
ZWG_DEV void turn_pairs(float (&a)[C], float (&b)[C], const float (&co)[C], const float (&si)[C]) {
#pragma unroll
    for (int j = 0; j < C; j++) {
        const float x = a[j], y = b[j];
        a[j] = __fsub_rn(__fmul_rn(x, co[j]), __fmul_rn(y, si[j]));
        b[j] = __fadd_rn(__fmul_rn(x, si[j]), __fmul_rn(y, co[j]));
    }
}

// N: elements a thread moves at a time (16 bytes of them, or 1). Threads: (piece, token).
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(N > 1 ? 256 : 1024) rope_kernel(RopeCall p, Divisor per_seq) {
    chain_release();
    const int z = chain_wait();
    using V = Vec<T, N>;
    constexpr bool ONE = INTER && N > 1;       // a piece holds both sides of its pairs
    constexpr int C = ONE ? N / 2 : N;         // pairs of a piece
    constexpr int HEADS = heads_of(ONE);
    using F = Vec<float, C>;
    const uint32_t row = blockIdx.x * blockDim.y + threadIdx.y;
    const int b = per_seq.div(row), i = row - b * p.s.n, piece = threadIdx.x;
    if (b >= p.s.n_batch) return;
    const Place at = place_of(p.s, b, p.t.n_ctx, piece == 0 && i == 0 && blockIdx.y == 0 ? p.err : nullptr);
    if (i >= at.count) return;
    const int half = p.t.rot / 2;
    const int turned = ONE ? p.t.rot / N : half / N;  // pieces of a head that are rotated; the others stay
    const bool turn = piece < turned;
    int ea, eb;  // where the two sides of a pair are (a piece that holds both: one place)
    if (!turn) ea = eb = p.t.rot + (piece - turned) * N;
    else if (ONE) ea = eb = piece * N;
    else if (INTER) ea = 2 * piece, eb = ea + 1;
    else ea = piece * N, eb = ea + half;
    const int h0 = blockIdx.y * HEADS, heads = min(HEADS, p.n_head + p.n_head_kv - h0);
    const T* q = static_cast<const T*>(p.q.data) + (b * p.q.bs + i * p.q.ts + z);
    const T* k = static_cast<const T*>(p.k.data) + (b * p.k.bs + i * p.k.ts + z);
    V va[HEADS], vb[HEADS];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        if (u >= heads) break;
        const int h = h0 + u;
        const T* x = h < p.n_head ? q + h * p.d : k + (h - p.n_head) * p.d;
        va[u] = *reinterpret_cast<const V*>(x + ea);
        if (!ONE && turn) vb[u] = *reinterpret_cast<const V*>(x + eb);
    }
    F co, si;
    if (turn) {
        const size_t t = (size_t)(at.past + i) * half + piece * C;
        co = *reinterpret_cast<const F*>(p.t.cos + t + z);
        si = *reinterpret_cast<const F*>(p.t.sin + t + z);
    }
    T* qo = static_cast<T*>(const_cast<void*>(p.q_out.data)) + (b * p.q_out.bs + i * p.q_out.ts + z);
    T* ko = static_cast<T*>(const_cast<void*>(p.k_out.data)) + (b * p.k_out.bs + i * p.k_out.ts + z);
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        if (u >= heads) break;
        const int h = h0 + u;
        T* y = h < p.n_head ? qo + h * p.d : ko + (h - p.n_head) * p.d;
        if (turn) {
            float a[C], c[C];
#pragma unroll
            for (int j = 0; j < C; j++) {
                a[j] = up(ONE ? va[u].e[(2 * j) % N] : va[u].e[j]);
                c[j] = up(ONE ? va[u].e[(2 * j + 1) % N] : vb[u].e[j]);
            }
            turn_pairs<C>(a, c, co.e, si.e);
#pragma unroll
            for (int j = 0; j < C; j++) {
                if constexpr (sizeof(T) == 2 && ONE) {
                    *reinterpret_cast<__nv_bfloat162*>(&va[u].e[2 * j]) = __floats2bfloat162_rn(a[j], c[j]);
                } else if constexpr (sizeof(T) == 2 && N > 1) {
                    if (j % 2) continue;
                    *reinterpret_cast<__nv_bfloat162*>(&va[u].e[j]) = __floats2bfloat162_rn(a[j], a[(j + 1) % C]);
                    *reinterpret_cast<__nv_bfloat162*>(&vb[u].e[j]) = __floats2bfloat162_rn(c[j], c[(j + 1) % C]);
                } else {
                    down(a[j], ONE ? va[u].e[(2 * j) % N] : va[u].e[j]);
                    down(c[j], ONE ? va[u].e[(2 * j + 1) % N] : vb[u].e[j]);
                }
            }
            if (!ONE) *reinterpret_cast<V*>(y + eb) = vb[u];
        }
        *reinterpret_cast<V*>(y + ea) = va[u];
    }
}

bool aligned(const Rows& r, size_t elem) {
    return ((uintptr_t)r.data | (r.bs * elem) | (r.ts * elem)) % 16 == 0;
}

template <typename T, int N>
int launch(const RopeCall& p, cudaStream_t st) {
    // a head's pieces: a pair of pieces, or a piece that holds its pairs, counts once
    const bool inter = p.t.interleaved != 0;
    const int pieces = (inter && N > 1 ? p.t.rot / N : p.t.rot / 2 / N) + (p.d - p.t.rot) / N;
    const int rows = p.s.n_batch * p.s.n, tokens = std::min(std::max(1, 256 / pieces), rows);
    const int heads = heads_of(inter && N > 1);
    const dim3 grid((rows + tokens - 1) / tokens, (p.n_head + p.n_head_kv + heads - 1) / heads);
    return launch_chained(inter ? rope_kernel<T, N, true> : rope_kernel<T, N, false>, grid, dim3(pieces, tokens), st, p,
                          Divisor(p.s.n)) == cudaSuccess
               ? 0
               : -1;
}

template <typename T>
int launch_type(const RopeCall& p, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const int half = p.t.rot / 2, pairs = p.t.interleaved ? N / 2 : N;  // of a piece, and of its table entries
    const bool vec = aligned(p.q, sizeof(T)) && aligned(p.q_out, sizeof(T)) && aligned(p.k, sizeof(T)) &&
                     aligned(p.k_out, sizeof(T)) && p.d % N == 0 && (p.t.interleaved ? p.t.rot : half) % N == 0 &&
                     half % pairs == 0 && (((uintptr_t)p.t.cos | (uintptr_t)p.t.sin) % std::min(16, pairs * 4)) == 0;
    return vec ? launch<T, N>(p, st) : launch<T, 1>(p, st);
}

}  // namespace

int rope_launch(const RopeCall& p, int type, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    return type == TYPE_BF16 ? launch_type<__nv_bfloat16>(p, st) : launch_type<float>(p, st);
}

}  // namespace zwg
