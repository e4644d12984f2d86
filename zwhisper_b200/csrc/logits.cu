// The rules on a step's logits (zwg_llm_logits): penalties for recent tokens, biases, an allow
// mask, and the index of the largest logit, in one pass over the logits.
//
// Bound by memory: 4 bytes in and, where something changes, 4 out for each logit. A cluster of
// 8 CTAs takes a row, a CTA an eighth of its vocabulary in pieces of up to 8192 tokens. For each
// piece the CTA scans the row's recent tokens and biases (from L2; they are short next to the
// logits) into dense counters in shared memory, so the pass over the logits looks each token up
// by its index and no order of the lists matters: counts are integers, and biases of one token are
// added in the order of the list, one round for each time that a token is there again. Only
// 16-byte pieces that change are written back. The CTAs' largest logits meet in CTA 0's shared
// memory, so there is no workspace and no second launch.
#include <cooperative_groups.h>
#include <limits.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"

namespace zwg {
namespace {

namespace cg = cooperative_groups;

constexpr int CTAS = 8, THREADS = 512, PIECE = 8192, MAX_BIAS = 4096;

ZWG_DEV void better(float& v, int& i, float ov, int oi) {
    if (ov > v || (ov == v && oi < i)) {
        v = ov;
        i = oi;
    }
}

struct Best {
    float v;
    int i;
};

// The rules on one logit: c times recent, bias add, allowed or not.
ZWG_DEV float ruled(float x, int c, float add, bool allowed, const LogitRules& r) {
    if (c > 0) {
        x = x > 0.f ? __fdiv_rn(x, r.repeat) : __fmul_rn(x, r.repeat);
        x = __fsub_rn(x, __fadd_rn(__fmul_rn((float)c, r.frequency), r.presence));
    }
    if (add != 0.f) x = __fadd_rn(x, add);
    return allowed ? x : -INFINITY;
}

__global__ void __launch_bounds__(THREADS) __cluster_dims__(CTAS, 1, 1)
    logit_rules_kernel(float* logits, int n_vocab, size_t stride, LogitRules r, int32_t* out, size_t out_stride, int vec,
                       int* err) {
    chain_release();
    const int z = chain_wait();
    extern __shared__ int counts[];                              // [PIECE]
    float* adds = reinterpret_cast<float*>(counts + PIECE);      // [PIECE], where there are biases
    __shared__ Best warp_best[THREADS / 32], cta_best[CTAS];
    const int row = blockIdx.y, rank = blockIdx.x, tid = threadIdx.x;
    float* x = logits + (size_t)row * stride + z;
    const int share = ((n_vocab + CTAS - 1) / CTAS + 31) & ~31;  // whole mask words
    const int begin = min(n_vocab, rank * share), end = min(n_vocab, begin + share);
    const uint32_t* allow = r.allow ? r.allow + (size_t)row * r.allow_stride + z : nullptr;
    const int32_t* ids = r.n_bias ? r.bias_ids + (size_t)row * r.bias_stride + z : nullptr;
    const float* bias = r.n_bias ? r.bias + (size_t)row * r.bias_stride + z : nullptr;
    int n_recent = r.n_recent;
    if (r.n_recents) {
        const int n = __ldcg(r.n_recents + row + z);
        if (n < 0 || n > n_recent) {
            if (tid == 0) set_error(err, kErrBounds);
            n_recent = n < 0 ? 0 : n_recent;
        } else {
            n_recent = n;
        }
    }
    const int32_t* recent = n_recent ? r.recent + (size_t)row * r.recent_stride + z : nullptr;
    const int oldest = n_recent > r.window ? n_recent - r.window : 0;
    const bool counted = n_recent > oldest;

    float bv = -INFINITY;
    int bi = INT_MAX;
    for (int seg = begin; seg < end; seg += PIECE) {
        const int n = min(PIECE, end - seg);
        if (ids) {
            for (int j = tid; j < n; j += THREADS) {
                counts[j] = INT_MAX;
                adds[j] = 0.f;
            }
            __syncthreads();
            uint32_t todo = 0;  // entries tid + e * THREADS of the list that are still to be added
            for (int e = 0; e * THREADS + tid < r.n_bias; e++) {
                const int t = __ldcg(ids + e * THREADS + tid);
                if (t < 0 || t >= n_vocab) set_error(err, kErrBounds);
                else if (t >= seg && t < seg + n) todo |= 1u << e;
            }
            while (__syncthreads_or(todo != 0)) {
                for (uint32_t w = todo; w; w &= w - 1) {
                    const int j = (__ffs(w) - 1) * THREADS + tid;
                    atomicMin(counts + __ldcg(ids + j) - seg, j);
                }
                __syncthreads();
                for (uint32_t w = todo; w; w &= w - 1) {
                    const int e = __ffs(w) - 1, j = e * THREADS + tid, t = __ldcg(ids + j) - seg;
                    if (*(volatile int*)(counts + t) == j) {  // the first of the token's entries that are left
                        adds[t] = __fadd_rn(adds[t], __ldcg(bias + j));
                        *(volatile int*)(counts + t) = INT_MAX;
                        todo &= ~(1u << e);
                    }
                }
            }
        }
        if (counted) {
            for (int j = tid; j < n; j += THREADS) counts[j] = 0;
            __syncthreads();
            for (int j = oldest + tid; j < n_recent; j += THREADS) {
                const int t = __ldcg(recent + j);
                if (t >= n_vocab) set_error(err, kErrBounds);
                else if (t >= seg && t < seg + n) atomicAdd(counts + t - seg, 1);
            }
            __syncthreads();
        }
        if (vec) {
            constexpr int U = 4;
            const int n4 = n / 4;
            float4* x4 = reinterpret_cast<float4*>(x + seg);
            for (int base = tid; base < n4; base += U * THREADS) {
                float4 v[U];
                uint32_t bits[U];
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int j = base + u * THREADS;
                    v[u] = j < n4 ? __ldcg(x4 + j) : make_float4(0.f, 0.f, 0.f, 0.f);
                    bits[u] = allow && j < n4 ? __ldcg(allow + (seg + 4 * j) / 32) >> (4 * j & 31) : ~0u;
                }
#pragma unroll
                for (int u = 0; u < U; u++) {
                    const int j = base + u * THREADS;
                    if (j >= n4) break;
                    const int4 c = counted ? reinterpret_cast<const int4*>(counts)[j] : make_int4(0, 0, 0, 0);
                    const float4 a = ids ? reinterpret_cast<const float4*>(adds)[j] : make_float4(0.f, 0.f, 0.f, 0.f);
                    const bool same = !(c.x | c.y | c.z | c.w) && a.x == 0.f && a.y == 0.f && a.z == 0.f &&
                                      a.w == 0.f && (bits[u] & 15) == 15;
                    if (!same) {
                        v[u].x = ruled(v[u].x, c.x, a.x, bits[u] & 1, r);
                        v[u].y = ruled(v[u].y, c.y, a.y, bits[u] & 2, r);
                        v[u].z = ruled(v[u].z, c.z, a.z, bits[u] & 4, r);
                        v[u].w = ruled(v[u].w, c.w, a.w, bits[u] & 8, r);
                        __stcg(x4 + j, v[u]);
                    }
                    const int t = seg + 4 * j;
                    better(bv, bi, v[u].x, t);
                    better(bv, bi, v[u].y, t + 1);
                    better(bv, bi, v[u].z, t + 2);
                    better(bv, bi, v[u].w, t + 3);
                }
            }
        }
        for (int j = (vec ? n / 4 * 4 : 0) + tid; j < n; j += THREADS) {
            const int t = seg + j, c = counted ? counts[j] : 0;
            const float a = ids ? adds[j] : 0.f, v = __ldcg(x + t);
            const bool allowed = !allow || (__ldcg(allow + t / 32) >> (t & 31) & 1);
            const float y = ruled(v, c, a, allowed, r);
            if (c || a != 0.f || !allowed) __stcg(x + t, y);
            better(bv, bi, y, t);
        }
        __syncthreads();
    }
    if (!out) return;  // the same for every CTA of the cluster
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
    if ((tid & 31) == 0) warp_best[tid >> 5] = Best{bv, bi};
    __syncthreads();
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();  // CTA 0 runs before its shared memory is written
    if (tid == 0) {
        for (int w = 1; w < THREADS / 32; w++) better(bv, bi, warp_best[w].v, warp_best[w].i);
        cluster.map_shared_rank(cta_best, 0)[rank] = Best{bv, bi};
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        for (int c = 0; c < CTAS; c++) better(bv, bi, cta_best[c].v, cta_best[c].i);
        out[row * out_stride + z] = bv > -INFINITY ? bi : -1;
    }
}

}  // namespace

int logit_rules_launch(float* logits, size_t m, int n_vocab, size_t stride, const LogitRules& r, int32_t* out,
                       size_t out_stride, int* err, cudaStream_t st) {
    static_assert(MAX_BIAS <= 32 * THREADS, "a thread's entries fit its mask");
    const int vec = ((uintptr_t)logits | (m > 1 ? stride * sizeof(float) : 0)) % 16 == 0;
    const size_t smem = r.n_bias ? 2 * PIECE * sizeof(int) : r.n_recent ? PIECE * sizeof(int) : 0;
    if (r.n_bias &&
        cudaFuncSetAttribute(logit_rules_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * PIECE * sizeof(int)))
        return -1;
    for (size_t row = 0; row < m; row += 65535) {  // rows are the grid's y
        const unsigned rows = (unsigned)std::min<size_t>(65535, m - row);
        LogitRules c = r;
        if (c.recent) c.recent += row * c.recent_stride;
        if (c.n_recents) c.n_recents += row;
        if (c.bias_ids) c.bias_ids += row * c.bias_stride;
        if (c.bias) c.bias += row * c.bias_stride;
        if (c.allow) c.allow += row * c.allow_stride;
        if (launch_chained_smem(logit_rules_kernel, dim3(CTAS, rows), dim3(THREADS), smem, st, logits + row * stride,
                                n_vocab, stride, c, out ? out + row * out_stride : out, out_stride, vec, err) !=
            cudaSuccess)
            return -1;
    }
    return 0;
}

}  // namespace zwg
