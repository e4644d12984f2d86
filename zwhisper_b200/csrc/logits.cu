// The rules on a step's logits (zwg_llm_logits): penalties for recent tokens, biases, an allow
// mask, and the index of the largest logit, in one pass over the logits.
//
// Bound by memory: 4 bytes in and, where something changes, 4 out for each logit. A cluster of
// 8 CTAs takes a row (16 where the rows are too few to fill the SMs), a CTA its share of the
// vocabulary in pieces of up to 9728 tokens. The row's recent tokens and biases are read into shared
// memory once; for each piece the CTA marks them in a dense array of one word a token (its count, and
// the place of its first bias in the list) while the piece's logits are on their way into registers,
// so the pass over the logits looks each token up by its index and no order of the lists matters:
// counts are integers, and further biases of a token are added to its first one's in the order of
// the list, one round for each. Only 16-byte pieces that change are written back. The CTAs' largest
// logits meet in CTA 0's shared memory, so there is no workspace and no second launch.
#include <cooperative_groups.h>
#include <limits.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"

namespace zwg {
namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 512, PIECE = 19 * THREADS, MAX_BIAS = 4096;  // U float4 a thread and piece, below
constexpr int COUNT_BITS = 19;  // of a token's word; the rest is 1 + MAX_BIAS - its first bias's place, or 0
constexpr int STAGED = 4096;  // recent tokens that are kept in shared memory; longer windows are read again
constexpr int MAX_CTAS = 16;

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

// Rules 1 and 2 on one logit, by its word: c times recent, a sum of biases.
__device__ __noinline__ float ruled(float x, uint32_t word, const float* sums, float repeat, float presence, float frequency) {
    const int c = word & ((1u << COUNT_BITS) - 1), place = word >> COUNT_BITS;
    if (c > 0) {
        x = x > 0.f ? __fdiv_rn(x, repeat) : __fmul_rn(x, repeat);
        x = __fsub_rn(x, __fadd_rn(__fmul_rn((float)c, frequency), presence));
    }
    if (place) {
        const float add = sums[1 + MAX_BIAS - place];
        if (add != 0.f) x = __fadd_rn(x, add);
    }
    return x;
}

__global__ void __launch_bounds__(THREADS)
    logit_rules_kernel(float* logits, int n_vocab, size_t stride, LogitRules r, int32_t* out, size_t out_stride, int vec,
                       int* err) {
    chain_release();
    const int z = chain_wait();
    extern __shared__ __align__(16) uint32_t words[];     // [PIECE]; then the lists:
    int* ids = reinterpret_cast<int*>(words + PIECE);      // [n_bias]
    float* sums = reinterpret_cast<float*>(ids + r.n_bias);  // [n_bias], at first the biases
    int* turn = reinterpret_cast<int*>(sums + r.n_bias);   // [n_bias]
    int* recent = turn + r.n_bias;                         // [the window, where it is staged]
    __shared__ Best warp_best[THREADS / 32], cta_best[MAX_CTAS];
    const int row = blockIdx.y, rank = blockIdx.x, n_ctas = gridDim.x, tid = threadIdx.x;
    float* x = logits + (size_t)row * stride + z;
    const int share = ((n_vocab + n_ctas - 1) / n_ctas + 31) & ~31;  // whole mask words
    const int begin = min(n_vocab, rank * share), end = min(n_vocab, begin + share);
    const uint32_t* allow = r.allow ? r.allow + (size_t)row * r.allow_stride + z : nullptr;
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
    const int oldest = n_recent > r.window ? n_recent - r.window : 0, in_window = n_recent - oldest;
    const int32_t* all_recent = r.recent + (size_t)row * r.recent_stride + oldest + z;
    const bool counted = in_window > 0, staged = r.window <= STAGED;
    const auto check = [&](int t, bool padding) {
        if (t >= n_vocab || (t < 0 && !padding)) set_error(err, kErrBounds);
        return t;
    };
    for (int j = tid; j < r.n_bias; j += THREADS) {
        ids[j] = check(__ldcg(r.bias_ids + (size_t)row * r.bias_stride + j + z), false);
        sums[j] = __ldcg(r.bias + (size_t)row * r.bias_stride + j + z);
        turn[j] = INT_MAX;
    }
    for (int j = tid; j < in_window; j += THREADS) {
        const int t = check(__ldcg(all_recent + j), true);
        if (staged) recent[j] = t;
    }

    float bv = -INFINITY;
    int bi = INT_MAX;
    const bool marked = counted || r.n_bias > 0;
    constexpr int U = (PIECE / 4 + THREADS - 1) / THREADS;
    for (int seg = begin; seg < end; seg += PIECE) {
        const int n = min(PIECE, end - seg), n4 = vec ? n / 4 : 0;
        float4* x4 = reinterpret_cast<float4*>(x + seg);
        float4 v[U];
        uint32_t bits[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = tid + u * THREADS;
            v[u] = j < n4 ? __ldcg(x4 + j) : make_float4(0.f, 0.f, 0.f, 0.f);
            bits[u] = allow && j < n4 ? __ldcg(allow + (seg + 4 * j) / 32) >> (4 * j & 31) : ~0u;
        }
        if (marked) {
            __syncthreads();  // the last piece's words have been read
            for (int j = tid; j < PIECE / 4; j += THREADS) reinterpret_cast<uint4*>(words)[j] = make_uint4(0, 0, 0, 0);
            __syncthreads();  // and the lists are there
        }
        if (r.n_bias) {
            uint32_t mine = 0, todo = 0;  // entries tid + e * THREADS of the list in this piece
            for (int e = 0; e * THREADS + tid < r.n_bias; e++) {
                const int j = e * THREADS + tid, t = ids[j] - seg;
                if (t < 0 || t >= n) continue;
                mine |= 1u << e;
                atomicMax(words + t, (uint32_t)(1 + MAX_BIAS - j) << COUNT_BITS);
            }
            __syncthreads();
            for (uint32_t w = mine; w; w &= w - 1) {
                const int e = __ffs(w) - 1, j = e * THREADS + tid;
                if ((words[ids[j] - seg] >> COUNT_BITS) != (uint32_t)(1 + MAX_BIAS - j)) todo |= 1u << e;  // not the token's first
            }
            while (__syncthreads_or(todo != 0)) {
                for (uint32_t w = todo; w; w &= w - 1) {
                    const int j = (__ffs(w) - 1) * THREADS + tid;
                    atomicMin(turn + (1 + MAX_BIAS - (words[ids[j] - seg] >> COUNT_BITS)), j);
                }
                __syncthreads();
                for (uint32_t w = todo; w; w &= w - 1) {
                    const int e = __ffs(w) - 1, j = e * THREADS + tid;
                    const int home = 1 + MAX_BIAS - (words[ids[j] - seg] >> COUNT_BITS);
                    if (*(volatile int*)(turn + home) == j) {  // the first of the token's entries that are left
                        sums[home] = __fadd_rn(sums[home], sums[j]);
                        *(volatile int*)(turn + home) = INT_MAX;
                        todo &= ~(1u << e);
                    }
                }
            }
        }
        if (counted) {
            for (int j = tid; j < in_window; j += THREADS) {
                const int t = (staged ? recent[j] : __ldcg(all_recent + j)) - seg;
                if (t >= 0 && t < n) atomicAdd(words + t, 1u);
            }
        }
        if (marked) __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = tid + u * THREADS;
            if (j >= n4) break;
            const uint4 w = marked ? reinterpret_cast<const uint4*>(words)[j] : make_uint4(0, 0, 0, 0);
            bool changed = false;
            if (w.x | w.y | w.z | w.w) {
                if (w.x) v[u].x = ruled(v[u].x, w.x, sums, r.repeat, r.presence, r.frequency);
                if (w.y) v[u].y = ruled(v[u].y, w.y, sums, r.repeat, r.presence, r.frequency);
                if (w.z) v[u].z = ruled(v[u].z, w.z, sums, r.repeat, r.presence, r.frequency);
                if (w.w) v[u].w = ruled(v[u].w, w.w, sums, r.repeat, r.presence, r.frequency);
                changed = true;
            }
            if ((bits[u] & 15) != 15) {
                v[u].x = bits[u] & 1 ? v[u].x : -INFINITY;
                v[u].y = bits[u] & 2 ? v[u].y : -INFINITY;
                v[u].z = bits[u] & 4 ? v[u].z : -INFINITY;
                v[u].w = bits[u] & 8 ? v[u].w : -INFINITY;
                changed = true;
            }
            if (changed) __stcg(x4 + j, v[u]);
            if (fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w)) > bv) {  // no search for the place otherwise
                const int t = seg + 4 * j;
                better(bv, bi, v[u].x, t);
                better(bv, bi, v[u].y, t + 1);
                better(bv, bi, v[u].z, t + 2);
                better(bv, bi, v[u].w, t + 3);
            }
        }
        for (int j = n4 * 4 + tid; j < n; j += THREADS) {
            const int t = seg + j;
            const uint32_t w = marked ? words[j] : 0;
            const bool allowed = !allow || (__ldcg(allow + t / 32) >> (t & 31) & 1);
            float y = __ldcg(x + t);
            if (w) y = ruled(y, w, sums, r.repeat, r.presence, r.frequency);
            if (!allowed) y = -INFINITY;
            if (w || !allowed) __stcg(x + t, y);
            better(bv, bi, y, t);
        }
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
        for (int c = 0; c < n_ctas; c++) better(bv, bi, cta_best[c].v, cta_best[c].i);
        out[row * out_stride + z] = bv > -INFINITY ? bi : -1;
    }
}

}  // namespace

int logit_rules_launch(float* logits, size_t m, int n_vocab, size_t stride, const LogitRules& r, int32_t* out,
                       size_t out_stride, int sm_count, int* err, cudaStream_t st) {
    static_assert(MAX_BIAS <= 32 * THREADS, "a thread's entries fit its mask");
    const int vec = ((uintptr_t)logits | (m > 1 ? stride * sizeof(float) : 0)) % 16 == 0;
    const size_t smem = (PIECE + 3 * (size_t)r.n_bias + (r.window <= STAGED ? r.window : 0)) * sizeof(int);
    const unsigned ctas = m * MAX_CTAS <= (size_t)sm_count ? MAX_CTAS : MAX_CTAS / 2;
    if (cudaFuncSetAttribute(logit_rules_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (PIECE + 3 * MAX_BIAS + STAGED) * sizeof(int)) != cudaSuccess ||
        cudaFuncSetAttribute(logit_rules_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
        return -1;
    for (size_t row = 0; row < m; row += 65535) {  // rows are the grid's y
        const unsigned rows = (unsigned)std::min<size_t>(65535, m - row);
        LogitRules c = r;
        if (c.recent) c.recent += row * c.recent_stride;
        if (c.n_recents) c.n_recents += row;
        if (c.bias_ids) c.bias_ids += row * c.bias_stride;
        if (c.bias) c.bias += row * c.bias_stride;
        if (c.allow) c.allow += row * c.allow_stride;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas, rows);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = ctas;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        if (cudaLaunchKernelEx(&cfg, logit_rules_kernel, logits + row * stride, n_vocab, stride, c,
                               out ? out + row * out_stride : out, out_stride, vec, err) != cudaSuccess)
            return -1;
    }
    return 0;
}

}  // namespace zwg
