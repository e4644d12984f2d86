// The rules on a step's logits (zwg_llm_logits): penalties for recent tokens, biases, an allow
// mask, and the index of the largest logit, in one pass over the logits.
//
// Bound by memory: 4 bytes in and, where something changes, 4 out for each logit. Few tokens are in the
// lists, so rules 1 and 2 go first and touch only theirs: a CTA puts the recent tokens and biases of
// its share of the vocabulary into a hash table in shared memory (a token's word holds its count and
// the place of its first bias in the list) and changes those logits in place. What is left is one
// stream: 8 loads of 16 bytes a thread on their way, the mask, the maximum, and only 16-byte pieces
// that the mask changes written back. No order of the lists matters: counts are integers, and further
// biases of a token are added to its first one's in the order of the list, one round for each. Lists of
// more than 4096 entries go through the table as a dense array, 8192 tokens at a time, and are read once for each: a
// window of 4096 tokens 11.3 us for one row of 151936 and 23.1 us for 64, of 4097 14.2 and 36.1; 3796 and 300 biases
// 11.9 and 25.0, 3797 14.5 and 37.8.
// A row has a CTA, or a cluster of up to 16 where the rows are too few to fill the SMs; the CTAs'
// largest logits meet in CTA 0's shared memory, so there is no workspace and no second launch. The
// share's logits are hinted into L2 while the lists are read.
#include <cooperative_groups.h>
#include <limits.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace zwg {
namespace {

namespace cg = cooperative_groups;

constexpr int THREADS = 512, MAX_CTAS = 16, MAX_BIAS = 4096;
constexpr int MOST_SLOTS = 8192, MOST_HASHED = MOST_SLOTS / 2;  // of the table; entries that are hashed
constexpr int COUNT_BITS = 19;  // of a token's word; the rest is 1 + MAX_BIAS - its first bias's place, or 0
constexpr uint32_t EMPTY = 0xffffffffu;
constexpr size_t MOST_SMEM = 10 * MOST_SLOTS + 12 * MAX_BIAS, SMEM_FOR_TWO = 104 * 1024;  // lists of a CTA; two CTAs an SM

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

// The slot of token t: of the table's array from `base` on (dense), or where its key is or goes.
ZWG_DEV int slot_of(uint32_t* keys, int log_slots, int t, int base, bool dense) {
    if (dense) return t - base;
    uint32_t s = (uint32_t)t * 2654435761u >> (32 - log_slots);
    for (;;) {  // at most half of the slots are taken
        const uint32_t had = atomicCAS(keys + s, EMPTY, (uint32_t)t);
        if (had == EMPTY || had == (uint32_t)t) return (int)s;
        s = (s + 1) & ((1u << log_slots) - 1);
    }
}

__global__ void __launch_bounds__(THREADS)
    logit_rules_kernel(float* logits, int n_vocab, size_t stride, LogitRules r, int32_t* out, size_t out_stride,
                       int log_slots, int vec, int* err) {
    chain_release();
    const int z = chain_wait();
    const int slots = 1 << log_slots;
    extern __shared__ __align__(16) uint32_t words[];      // where there are lists: [slots]
    uint32_t* keys = words + slots;                        // [slots]
    uint16_t* used = reinterpret_cast<uint16_t*>(keys + slots);  // [slots], those whose word is not 0
    int* ids = reinterpret_cast<int*>(used + slots);       // [n_bias]
    float* sums = reinterpret_cast<float*>(ids + r.n_bias);  // [n_bias], at first the biases
    int* turn = reinterpret_cast<int*>(sums + r.n_bias);   // [n_bias]
    __shared__ Best warp_best[THREADS / 32], cta_best[MAX_CTAS];
    __shared__ int n_used;
    const int row = blockIdx.y, rank = blockIdx.x, n_ctas = gridDim.x, tid = threadIdx.x;
    float* x = logits + (size_t)row * stride + z;
    const int share = ((n_vocab + n_ctas - 1) / n_ctas + 31) & ~31;  // whole mask words
    const int begin = min(n_vocab, rank * share), end = min(n_vocab, begin + share), n = end - begin;
    const uint32_t* allow = r.allow ? r.allow + (size_t)row * r.allow_stride + z : nullptr;
    if (vec && tid == 0 && n >= 4)
        sm100::bulk_hint(x + begin, n / 4 * 16);

    int n_recent = r.n_recent;
    if (r.n_recents) {
        const int have = __ldcg(r.n_recents + row + z);
        if (have < 0 || have > n_recent) {
            if (tid == 0) set_error(err, kErrBounds);
            n_recent = have < 0 ? 0 : n_recent;
        } else {
            n_recent = have;
        }
    }
    const int oldest = n_recent > r.window ? n_recent - r.window : 0, in_window = n_recent - oldest;
    const int32_t* recent = r.recent + (size_t)row * r.recent_stride + oldest + z;
    if (in_window > 0 || r.n_bias > 0) {
        const bool dense = in_window + r.n_bias > MOST_HASHED;  // then there are MOST_SLOTS
        for (int j = tid; j < r.n_bias; j += THREADS) {
            const int t = __ldcg(r.bias_ids + (size_t)row * r.bias_stride + j + z);
            if (t < 0 || t >= n_vocab) set_error(err, kErrBounds);
            ids[j] = t;
            sums[j] = __ldcg(r.bias + (size_t)row * r.bias_stride + j + z);
            turn[j] = INT_MAX;
        }
        for (int base = begin; base < end; base += dense ? slots : n) {
            const int top = dense ? min(end, base + slots) : end;  // tokens of this turn
            if (tid == 0) n_used = 0;
            for (int j = tid; j < slots / 4; j += THREADS) {
                reinterpret_cast<uint4*>(words)[j] = make_uint4(0, 0, 0, 0);
                if (!dense) reinterpret_cast<uint4*>(keys)[j] = make_uint4(EMPTY, EMPTY, EMPTY, EMPTY);
            }
            __syncthreads();
            if (r.n_bias) {
                uint32_t mine = 0, todo = 0;  // entries tid + e * THREADS of the list in this turn
                for (int e = 0; e * THREADS + tid < r.n_bias; e++) {
                    const int j = e * THREADS + tid, t = ids[j];
                    if (t < base || t >= top) continue;
                    mine |= 1u << e;
                    const int s = ids[j] = slot_of(keys, log_slots, t, base, dense);  // from here on in this turn
                    if (atomicMax(words + s, (uint32_t)(1 + MAX_BIAS - j) << COUNT_BITS) == 0) used[atomicAdd(&n_used, 1)] = s;
                }
                __syncthreads();
                for (uint32_t w = mine; w; w &= w - 1) {
                    const int e = __ffs(w) - 1, j = e * THREADS + tid;
                    if ((words[ids[j]] >> COUNT_BITS) != (uint32_t)(1 + MAX_BIAS - j)) todo |= 1u << e;  // not the token's first
                }
                while (__syncthreads_or(todo != 0)) {
                    for (uint32_t w = todo; w; w &= w - 1) {
                        const int j = (__ffs(w) - 1) * THREADS + tid;
                        atomicMin(turn + (1 + MAX_BIAS - (words[ids[j]] >> COUNT_BITS)), j);
                    }
                    __syncthreads();
                    for (uint32_t w = todo; w; w &= w - 1) {
                        const int e = __ffs(w) - 1, j = e * THREADS + tid;
                        const int home = 1 + MAX_BIAS - (words[ids[j]] >> COUNT_BITS);
                        if (*(volatile int*)(turn + home) == j) {  // the first of the token's entries that are left
                            sums[home] = __fadd_rn(sums[home], sums[j]);
                            *(volatile int*)(turn + home) = INT_MAX;
                            todo &= ~(1u << e);
                        }
                    }
                }
                for (uint32_t w = mine; w; w &= w - 1) ids[(__ffs(w) - 1) * THREADS + tid] = -1;  // done
            }
            for (int j = tid; j < in_window; j += THREADS) {
                const int t = __ldcg(recent + j);
                if (t >= n_vocab) set_error(err, kErrBounds);
                if (t < base || t >= top) continue;
                const int s = slot_of(keys, log_slots, t, base, dense);
                if (atomicAdd(words + s, 1u) == 0) used[atomicAdd(&n_used, 1)] = s;
            }
            __syncthreads();
            // rules 1 and 2 on the tokens of the table
            for (int j = tid; j < n_used; j += THREADS) {
                const int s = used[j];
                const uint32_t word = words[s];
                const int t = dense ? base + s : (int)keys[s], c = word & ((1u << COUNT_BITS) - 1), place = word >> COUNT_BITS;
                float v = __ldcg(x + t);
                if (c > 0)
                    v = __fsub_rn(__fmul_rn(v, v > 0.f ? r.inv_repeat : r.repeat),
                                  __fadd_rn(__fmul_rn((float)c, r.frequency), r.presence));
                const float add = place ? sums[1 + MAX_BIAS - place] : 0.f;
                if (add != 0.f) v = __fadd_rn(v, add);
                __stcg(x + t, v);
            }
            __syncthreads();
        }
    }

    float bv = -INFINITY;
    int bi = INT_MAX;
    const int n4 = vec ? n / 4 : 0;
    constexpr int U = 8;
    float4* x4 = reinterpret_cast<float4*>(x + begin);
    for (int base = tid; base < n4; base += U * THREADS) {
        float4 v[U];
        uint32_t bits[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = base + u * THREADS;
            v[u] = j < n4 ? __ldcg(x4 + j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            bits[u] = allow && j < n4 ? __ldcg(allow + (begin + 4 * j) / 32) >> (4 * j & 31) : ~0u;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = base + u * THREADS;
            if ((bits[u] & 15) != 15) {
                v[u].x = bits[u] & 1 ? v[u].x : -INFINITY;
                v[u].y = bits[u] & 2 ? v[u].y : -INFINITY;
                v[u].z = bits[u] & 4 ? v[u].z : -INFINITY;
                v[u].w = bits[u] & 8 ? v[u].w : -INFINITY;
                __stcg(x4 + j, v[u]);
            }
            if (fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w)) > bv) {  // no search for the place otherwise
                const int t = begin + 4 * j;
                better(bv, bi, v[u].x, t);
                better(bv, bi, v[u].y, t + 1);
                better(bv, bi, v[u].z, t + 2);
                better(bv, bi, v[u].w, t + 3);
            }
        }
    }
    for (int t = begin + n4 * 4 + tid; t < end; t += THREADS) {
        float v = __ldcg(x + t);
        if (allow && !(__ldcg(allow + t / 32) >> (t & 31) & 1)) {
            v = -INFINITY;
            __stcg(x + t, v);
        }
        better(bv, bi, v, t);
    }
    if (!out) return;  // the same for every CTA of the cluster
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        better(bv, bi, __shfl_xor_sync(0xffffffffu, bv, o), __shfl_xor_sync(0xffffffffu, bi, o));
    if ((tid & 31) == 0) warp_best[tid >> 5] = Best{bv, bi};
    __syncthreads();
    cg::cluster_group cluster = cg::this_cluster();
    if (n_ctas > 1) cluster.sync();  // CTA 0 runs before its shared memory is written
    if (tid == 0) {
        for (int w = 1; w < THREADS / 32; w++) better(bv, bi, warp_best[w].v, warp_best[w].i);
        cluster.map_shared_rank(cta_best, 0)[rank] = Best{bv, bi};
    }
    if (n_ctas > 1) cluster.sync();
    if (rank == 0 && tid == 0) {
        for (int c = 0; c < n_ctas; c++) better(bv, bi, cta_best[c].v, cta_best[c].i);
        out[row * out_stride + z] = bv > -INFINITY ? bi : -1;
    }
}

// Clusters of n CTAs that run at once on the current device, asked once for each device and amount of
// shared memory (two CTAs an SM, or one).
int clusters_at_once(int n, bool one_an_sm) {
    static std::atomic<int> known[64][2][MAX_CTAS + 1];
    int dev = 0, count = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    std::atomic<int>& at = known[dev & 63][one_an_sm][n];
    if ((count = at.load(std::memory_order_relaxed))) return count;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = one_an_sm ? MOST_SMEM : SMEM_FOR_TWO;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)n;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&count, logit_rules_kernel, &cfg) != cudaSuccess) (void)cudaGetLastError();
    at.store(count = std::max(1, count), std::memory_order_relaxed);
    return count;
}

}  // namespace

int logit_rules_launch(float* logits, size_t m, int n_vocab, size_t stride, const LogitRules& r, int32_t* out,
                       size_t out_stride, int sm_count, int* err, cudaStream_t st) {
    static_assert(MAX_BIAS <= 32 * THREADS, "a thread's entries fit its mask");
    const int vec = ((uintptr_t)logits | (m > 1 ? stride * sizeof(float) : 0)) % 16 == 0;
    const int entries = std::min(r.window, r.n_recent) + r.n_bias;
    int log_slots = 8;  // twice the entries, at the least
    while ((1 << log_slots) < MOST_SLOTS && (1 << log_slots) < 2 * entries) log_slots++;
    const size_t smem = entries ? ((size_t)10 << log_slots) + 12 * (size_t)r.n_bias : 0;
    // two CTAs an SM, each with at least a round of its threads' loads
    const int worth = (n_vocab + 4 * THREADS - 1) / (4 * THREADS);
    int ctas = (int)std::max<size_t>(1, std::min<size_t>({2 * (size_t)sm_count / m, MAX_CTAS, (size_t)worth}));
    static std::atomic<uint64_t> done{0};
    if (allow_smem(done, (const void*)logit_rules_kernel, (int)MOST_SMEM, true) != cudaSuccess) return -1;
    // all rows' clusters at once: 16 rows in clusters of 16, of which 14 fit, 13.7 us, in smaller ones 9.4; 48 rows 21.2 and 14.8
    while (ctas > 1 && m <= (size_t)sm_count && (size_t)clusters_at_once(ctas, smem > SMEM_FOR_TWO) < m) ctas--;
    for (size_t row = 0; row < m; row += 65535) {  // rows are the grid's y
        const unsigned rows = (unsigned)std::min<size_t>(65535, m - row);
        LogitRules c = r;
        if (c.recent) c.recent += row * c.recent_stride;
        if (c.n_recents) c.n_recents += row;
        if (c.bias_ids) c.bias_ids += row * c.bias_stride;
        if (c.bias) c.bias += row * c.bias_stride;
        if (c.allow) c.allow += row * c.allow_stride;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)ctas, rows);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = (unsigned)ctas;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 2;
        if (cudaLaunchKernelEx(&cfg, logit_rules_kernel, logits + row * stride, n_vocab, stride, c,
                               out ? out + row * out_stride : out, out_stride, log_slots, vec, err) != cudaSuccess)
            return -1;
    }
    return 0;
}

}  // namespace zwg
