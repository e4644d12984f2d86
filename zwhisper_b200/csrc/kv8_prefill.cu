// Attention over a cache in 8 bits for many query rows of a kv head (prompt chunks), on the tcgen05
// tensor cores: the products, scales, pieces and softmax of kv8_attn.cu with 128 keys and 2 x 128
// query rows at a time.
//
// kv8_prefill_kernel. A CTA of 26 warps takes 256 rows (row = query * group + head) of one (sequence,
// kv head), or a cut of their keys. Warps 16-23 turn the int8 keys and values of 4 blocks into f16
// tiles in shared memory, in the 128-byte swizzle of a K-major operand, a tile ahead in registers: a
// cache row's bytes and a value column's 32 tokens are both contiguous along K, so neither is
// transposed. Warps 24 and 25 issue the products of one query tile each: S = Q K^T (Q from shared
// memory in its pieces) into TMEM, then O += P V (P from TMEM). Warps 0-15 are the softmax, two
// threads a row, each with two of a tile's four blocks, so that four warps of every scheduler hide
// one another's latencies; a row's two maxima meet in shared memory. They read S twice (the maximum,
// then the probabilities, 16 columns at a time) and write P over it, in its pieces, so that S, P and O
// of both query tiles fill the 512 columns of TMEM, and one tile's softmax runs while the other's
// products do. Keys have two buffers, so that neither tile waits for the other; values too, where
// there is room (not beside two pieces of d 128).
// O is rescaled in TMEM only where a row's maximum grows by more than 2^4 or the values' scale does:
// probabilities stay below 2^4 and P's pieces hold 2^11 p.
//
// 32 sequences x 256 tokens after 1744, 12 / 2 heads of d 128: 318 us in f32 (the products alone, of two
// pieces, take 113 us at the rate of large library products), 220 us in bf16 (57); 16 x 250 after 1750,
// 14 / 2 heads of d 64: 152 us in f32, 110 us in bf16 (16). Bound by the latency of a tile's chain (S, its maximum,
// P, P V) over only two tiles at a time. Copies with parts left out, in f32 without drains (261 us then, 271 now): an
// eighth of the products 208 us, no exponentials 252, no conversion of K and V 261. Tile 1 starts a softmax behind
// tile 0, so that the one's products run during the other's exponentials (294 us side by side). One key and two value
// buffers: 278 us. 26 warps leave 72 registers a thread, which every form exceeds: 52 to 352 bytes of spills are read
// back in a thread. CTAs of 256 rows also leave SMs empty at the end: 384 CTAs on 148 SMs are 2.6 waves.
#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv8_attn.cuh"
#include "seqs.cuh"
#include "sm100.cuh"

namespace zwg {
namespace {

using namespace kv8;
using namespace sm100;

constexpr int BM = 128, BN = 128;         // rows of a query tile, keys of a tile
constexpr int BLOCKS = BN / KV8_BLOCK;    // blocks of a key tile
constexpr int SOFTMAX = 512, CONVERTERS = 256;  // threads; then the two issuing warps
constexpr int THREADS = SOFTMAX + CONVERTERS + 64;
constexpr float kUnit = 2048.f;   // P's pieces hold 2^11 p, and p < 2^4
constexpr float kStale = 4.f;
constexpr uint32_t TMEM_COLS = 512;
// With one piece of d 64 there is room for P beside S: the next S is computed while the probabilities are.
template <int D, int P>
constexpr bool BESIDE = D == 64 && P == 1;
__host__ __device__ constexpr uint32_t s_col(int t) { return t * 128u; }
__host__ __device__ constexpr uint32_t beside_col(int t) { return 384u + t * 64u; }
template <int D>
__host__ __device__ constexpr uint32_t o_col(int t) { return 256u + t * D; }

// The tensor cores truncate their sums, 2 x 128 / 16 of them to a key tile, which shrinks O by 2e-9 of it
// for each key: 1.6e-5 after 8000 keys. So where two pieces ask for f32's accuracy, the sums of MOST_RUN
// tiles at the most are drained into f32 sums that wait in the output's own place. 32 x 256 tokens after 1744
// at d 128, keys with a few strong channels: 271 us and off by 4.4e-6 without, 292 us and 2.4e-6 in runs of 8, 309 us
// and 1.8e-6 of 6, 318 us and 1.6e-6 of 5, 324 us and 1.45e-6 of 4 (the f32 library form of the same sums: 1.2e-6).
// From 500 to 32000 keys, d 64 and 128: 1.5e-6 to 1.75e-6, and 1.1e-6 to 1.3e-6 where all channels are alike (library
// form 0.6e-6 to 1.3e-6). What stays are the truncated sums of the scores and of a run. (The small query pieces go
// first for the same reason: 3e-7 less.)
constexpr int MOST_RUN = 5;
// Key tiles from one drain to the next, of n in all.
template <int P>
ZWG_DEV int run_of(int n) {
    const int runs = (n + MOST_RUN - 1) / MOST_RUN;
    return P == 1 || runs < 2 ? n : (n + runs - 1) / runs;
}

template <int D, int P>
struct Smem {
    static constexpr int KS = 2, VS = D * P > 128 ? 1 : 2;  // buffers of keys and values
    uint8_t q[2][P][D / 64][BM * 128];   // query tiles: [row][64 f16], swizzled
    uint8_t k[KS][D / 64][BN * 128];     // keys: [key][64 f16]
    uint8_t v[VS][BN / 64][D * 128];     // value columns: [d][64 f16 of tokens]
    float2 scale[4][BLOCKS];             // (ks, vs) of a tile's blocks: a tile's are read until its P is there
    float part[2][2][BM];                // what a row's two threads tell each other: [query tile][half]
    uint64_t q_full[2], k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], s_full[2], s_free[2], p_full[2], pv_done[2], drained[2];
    uint64_t started;  // tile 0's first P is there
    uint32_t tmem_base;
};

// Packed products and sums, each rounded: written out, since the compiler may contract the intrinsics.
ZWG_DEV float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}
ZWG_DEV float2 add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(r)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
    return r;
}

// Barrier `id` of n threads, and whether all of them say yes: warps that wait for one another agree on
// whether one of them gave up.
ZWG_DEV bool all_of(int id, int n, bool ok) {
    uint32_t all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, %3, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(ok ? 1u : 0u), "r"(id), "r"(n)
        : "memory");
    return all != 0;
}

// o f + (had g) h
ZWG_DEV float4 summed(const uint32_t* o, float f, float4 had, float g, float h) {
    return make_float4(__uint_as_float(o[0]) * f + had.x * g * h, __uint_as_float(o[1]) * f + had.y * g * h,
                       __uint_as_float(o[2]) * f + had.z * g * h, __uint_as_float(o[3]) * f + had.w * g * h);
}
ZWG_DEV float4 had_at(const float* p, bool whole) {
    return whole ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3]);
}

// 16 int8 -> two 16-byte units of f16.
ZWG_DEV void widen(uint4 w, uint4& lo, uint4& hi) {
    ints_to_f16(w.x, lo.x, lo.y);
    ints_to_f16(w.y, lo.z, lo.w);
    ints_to_f16(w.z, hi.x, hi.y);
    ints_to_f16(w.w, hi.z, hi.w);
}

// vec: bit 0 queries, bit 1 outputs can be moved 16 bytes of f32 at a time.
template <typename T, int D, int P>
__global__ void __launch_bounds__(THREADS, 1) kv8_prefill_kernel(Kv8Attn p, int splits, int vec, float scale) {
    chain_release();
    const int z = chain_wait();
    extern __shared__ __align__(1024) uint8_t smem_raw[];  // the swizzle goes by address: checked below
    Smem<D, P>& sm = *reinterpret_cast<Smem<D, P>*>(smem_raw);
    if (smem_u32(smem_raw) & 1023) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    constexpr int BYTES = KV8_BLOCK * D;
    const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = p.n_head / p.c.n_head_kv;
    const Place at = place_of(p.s, b, p.c.blocks * KV8_BLOCK, threadIdx.x == 0 && blockIdx.x == 0 && h == 0 ? p.err : nullptr);
    const int rows = at.count * group, row0 = tile * 2 * BM;
    if (row0 >= rows) return;
    const int first = p.s.first ? __ldcg(p.s.first + b + z) : 0;
    if (first < 0) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    const int n_t = row0 + BM < rows ? 2 : 1;  // query tiles with rows
    const int seen = at.past + (min(rows, row0 + 2 * BM) - 1) / group + 1;  // keys the last row sees
    const int blk_hi = (seen + KV8_BLOCK - 1) / KV8_BLOCK;
    const int all = max(0, (blk_hi - first / KV8_BLOCK + BLOCKS - 1) / BLOCKS);
    const int from = (int)((long long)all * split / splits), n_tiles = (int)((long long)all * (split + 1) / splits) - from;
    const int blk0 = first / KV8_BLOCK + from * BLOCKS;
    int* err = p.err;

    using S = Smem<D, P>;
    constexpr int ISSUER = (SOFTMAX + CONVERTERS) / 32;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; t++) {
            mbar_init(&sm.q_full[t], 8);
            mbar_init(&sm.s_full[t], 2);  // the products' completion, and the issuer's own: it has seen the scales
            mbar_init(&sm.s_free[t], 8);
            mbar_init(&sm.p_full[t], 8);
            mbar_init(&sm.pv_done[t], 1);
            mbar_init(&sm.drained[t], 1);
        }
        for (int i = 0; i < S::KS; i++) {
            mbar_init(&sm.k_full[i], CONVERTERS / 32);
            mbar_init(&sm.k_empty[i], n_t);
        }
        for (int i = 0; i < S::VS; i++) {
            mbar_init(&sm.v_full[i], CONVERTERS / 32);
            mbar_init(&sm.v_empty[i], n_t);
        }
        mbar_init(&sm.started, 1);
        fence_mbar_init();
    }
    if (warp == ISSUER) {
        tmem_alloc(&sm.tmem_base, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp >= ISSUER) {
        // ---------------------------------------------------- the products of query tile t
        const int t = warp - ISSUER;
        if (t < n_t && lane == 0 && n_tiles > 0) {
            constexpr uint32_t idesc_s = idesc_f16(BM, BN, false, false, false);
            constexpr uint32_t idesc_o = idesc_f16(BM, D, false, false, false);
            bool ok = mbar_wait(&sm.q_full[t], 0, err);
            // tile 1 starts a softmax behind tile 0, so that the one's exponentials run during the other's products
            // (a barrier of its own: p_full's phases go on, and one that is two ahead looks like none)
            if (t == 1) ok = ok && mbar_wait(&sm.started, 0, err);
            const auto scores = [&](int j) {
                const int ks = j % S::KS;
                if (!mbar_wait(&sm.k_full[ks], j / S::KS & 1, err)) return false;
                // S goes where the last S was read from, or its P, which the PV reads
                if (j > 0 && !mbar_wait(BESIDE<D, P> ? &sm.s_free[t] : &sm.pv_done[t], (j - 1) & 1, err)) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < P; c++)
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++) {
                        const uint64_t qa = smem_desc_sw128(smem_u32(sm.q[t][P - 1 - c][kk / 4]) + kk % 4 * 32, 16, 1024);
                        const uint64_t kb = smem_desc_sw128(smem_u32(sm.k[ks][kk / 4]) + kk % 4 * 32, 16, 1024);
                        mma_f16_ss(tmem + s_col(t), qa, kb, idesc_s, c > 0 || kk > 0);
                    }
                mma_commit(&sm.s_full[t]);
                mma_commit(&sm.k_empty[ks]);
                mbar_arrive(&sm.s_full[t]);
                return true;
            };
            if (BESIDE<D, P>) ok = ok && scores(0);
            const int run = run_of<P>(n_tiles);
            int started = 0;  // the tile that O starts with
            for (int j = 0; ok && j < n_tiles; j++) {
                if (j == started + run) started = j;
                const int vs = j % S::VS;
                if (!BESIDE<D, P>) ok = scores(j);
                else if (j + 1 < n_tiles) ok = scores(j + 1);
                if (!ok || !(ok = mbar_wait(&sm.p_full[t], j & 1, err))) break;
                if (t == 0 && j == 0) mbar_arrive(&sm.started);
                if (!(ok = mbar_wait(&sm.v_full[vs], j / S::VS & 1, err))) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < P; c++)
#pragma unroll
                    for (int kk = 0; kk < BN / 16; kk++) {
                        const uint64_t vb = smem_desc_sw128(smem_u32(sm.v[vs][kk / 4]) + kk % 4 * 32, 16, 1024);
                        const uint32_t pa = BESIDE<D, P> ? beside_col(t) + kk * 8 : s_col(t) + kk * 16 + c * 8;
                        mma_f16_ts(tmem + o_col<D>(t), tmem + pa, vb, idesc_o, j > started || c > 0 || kk > 0);
                    }
                mma_commit(&sm.pv_done[t]);
                mma_commit(&sm.v_empty[vs]);
            }
            if (!ok) {  // gave up: the products on their way end before TMEM is given back
                mma_commit(&sm.drained[t]);
                mbar_wait_drain(&sm.drained[t], 0);
            }
        }
    } else if (warp >= SOFTMAX / 32) {
        // ---------------------------------------------------- int8 blocks to f16 tiles
        const int tid = threadIdx.x - SOFTMAX;
        constexpr int SEGS = D / 16;               // 16-byte pieces of a key's row
        constexpr int N = BN * SEGS / CONVERTERS;  // pieces of a tile for each thread, in their order in memory
        const size_t head = (size_t)bh * p.c.blocks;
        uint4 kb[N], vb[N];
        float2 sc = make_float2(0.f, 0.f);
        const auto load = [&](uint4 (&buf)[N], const int8_t* from, int j) {
            const int blk = blk0 + j * BLOCKS, pieces = min(blk_hi - blk, BLOCKS) * (BYTES / 16);  // behind them: masked, but finite
            const uint4* src = reinterpret_cast<const uint4*>(from + (head + blk) * BYTES + z);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = tid + i * CONVERTERS;
                buf[i] = e < pieces ? __ldcg(src + e) : make_uint4(0, 0, 0, 0);
            }
        };
        const auto load_k = [&](int j) {
            load(kb, p.c.k, j);
            const int blk = blk0 + j * BLOCKS + tid;
            sc = make_float2(0.f, 0.f);
            if (tid < BLOCKS && blk < blk_hi)
                sc = make_float2(__ldcg(p.c.k_scale + head + blk + z), __ldcg(p.c.v_scale + head + blk + z));
        };
        const auto store = [&](uint8_t* row, int r, int unit, uint4 w) {
            uint4 lo, hi;
            widen(w, lo, hi);
            *reinterpret_cast<uint4*>(row + ((unit ^ (r & 7)) << 4)) = lo;
            *reinterpret_cast<uint4*>(row + (((unit + 1) ^ (r & 7)) << 4)) = hi;
        };
        if (n_tiles > 0) {
            load_k(0);
            load(vb, p.c.v, 0);
        }
        for (int j = 0; j < n_tiles; j++) {
            const int ks = j % S::KS, vs = j % S::VS;
            if (j >= S::KS && !mbar_wait_warp(&sm.k_empty[ks], (j / S::KS - 1) & 1, err)) break;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = tid + i * CONVERTERS, r = e / SEGS, seg = e % SEGS;
                store(sm.k[ks][seg / 4] + r * 128, r, (seg & 3) * 2, kb[i]);
            }
            if (tid < BLOCKS) {
                if (sc.y != sc.y) sc = make_float2(sc.y, 0.f);  // values that read as NaN: through the scores
                sm.scale[j & 3][tid] = sc;
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.k_full[ks]);
            if (j + 1 < n_tiles) load_k(j + 1);
            if (j >= S::VS && !mbar_wait_warp(&sm.v_empty[vs], (j / S::VS - 1) & 1, err)) break;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int e = tid + i * CONVERTERS, blk = e / (D * 2), r = e / 2 % D;
                store(sm.v[vs][blk / 2] + r * 128, r, (blk & 1) * 4 + (e & 1) * 2, vb[i]);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.v_full[vs]);
            if (j + 1 < n_tiles) load(vb, p.c.v, j + 1);
        }
    } else {
        // ---------------------------------------------------- softmax of query tile t, half of each tile's keys
        const int t = warp >> 3, half = warp >> 2 & 1, quarter = warp & 3, r = quarter * 32 + lane;
        const int row = row0 + t * BM + r, pair = 1 + t * 4 + quarter;  // the barrier of a row's two threads
        const bool live = row < rows;
        const int i = live ? row / group : 0;
        const size_t in_token = (size_t)(h * group + (live ? row - i * group : 0)) * D;
        const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
        if (t < n_t) {
            // queries: the warp takes half of its quarter's rows, whole ones, a lane four elements
            constexpr int LANES = D / 4, AT_ONCE = 32 / LANES, BATCH = 8;  // BATCH loads on their way
            const T* q = static_cast<const T*>(p.q.data) + z + b * p.q.bs + lane % LANES * 4;
            const size_t q_off = i * p.q.ts + in_token;
#pragma unroll 1
            for (int n0 = half * 16; n0 < half * 16 + 16; n0 += BATCH * AT_ONCE) {
                Four<T> xs[BATCH];
                size_t off[BATCH];
#pragma unroll
                for (int c = 0; c < BATCH; c++) off[c] = __shfl_sync(0xffffffffu, q_off, n0 + c * AT_ONCE + lane / LANES);
                if (vec & 1) {  // (a row behind the last one: the first token's)
#pragma unroll
                    for (int c = 0; c < BATCH; c++) xs[c] = load_four(q + off[c], true);
                } else {
#pragma unroll
                    for (int c = 0; c < BATCH; c++) xs[c] = load_four(q + off[c], false);
                }
#pragma unroll
                for (int c = 0; c < BATCH; c++) {
                    const int rr = n0 + c * AT_ONCE + lane / LANES, qr = quarter * 32 + rr;
                    float4 x = value_of(xs[c]);
                    if (!(live_rows >> rr & 1)) x = make_float4(0.f, 0.f, 0.f, 0.f);
                    uint32_t top = max(max(__float_as_uint(fabsf(x.x)), __float_as_uint(fabsf(x.y))),
                                       max(__float_as_uint(fabsf(x.z)), __float_as_uint(fabsf(x.w))));
                    top = __reduce_max_sync(LANES == 32 ? 0xffffffffu : lane < 16 ? 0xffffu : 0xffff0000u, top);
                    float p2, inv;
                    power_of(__uint_as_float(top), p2, inv);
                    if (lane % LANES == 0) sm.part[t][0][qr] = p2 * scale;
                    uint32_t w[2][P];
                    pieces_of<P>(x.x * inv, x.y * inv, w[0]);
                    pieces_of<P>(x.z * inv, x.w * inv, w[1]);
                    const int e = lane % LANES * 4;
#pragma unroll
                    for (int k = 0; k < P; k++)
                        *reinterpret_cast<uint2*>(sm.q[t][k][e / 64] + qr * 128 + (((e % 64 / 8) ^ (qr & 7)) << 4) + e / 4 % 2 * 8) =
                            make_uint2(w[0][k], w[1][k]);
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full[t]);
            all_of(pair, 64, true);
            const float unit = sm.part[t][0][r];  // of the row's scores
            bool ok = all_of(pair, 64, true);

            constexpr int MINE = BLOCKS / 2;                                   // blocks of a tile
            const int lim = live ? at.past + i + 1 : 0;                        // keys below it are seen
            const int seen_by_all = at.past + (row0 + t * BM) / group + 1;     // by the tile's first row
            const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
            const uint32_t s_addr = tmem + lanes + s_col(t) + half * 64, o_addr = tmem + lanes + o_col<D>(t) + half * (D / 2);
            const uint32_t p_addr = tmem + lanes + beside_col(t) + half * 32;
            float m = -INFINITY, l = 0.f;
            uint32_t ref = 0x00800000u;  // bits of a power of two above every vs so far
            const int run = run_of<P>(n_tiles);
            float m_out = -INFINITY;  // the maximum that drained sums refer to
            for (int j = 0, stop = min(run, n_tiles);; stop = min(stop + run, n_tiles)) {
                for (; j < stop; j++) {
                    ok = ok && mbar_wait_warp(&sm.s_full[t], j & 1, err);
                    tc_fence_after();
                    float4 sc01 = *reinterpret_cast<const float4*>(sm.scale[j & 3]);
                    float4 sc23 = *reinterpret_cast<const float4*>(sm.scale[j & 3] + 2);
                    const int key0 = (blk0 + j * BLOCKS) * KV8_BLOCK;
                    const bool masked = key0 + BN > seen_by_all || key0 < first;
                    if (masked) {  // blocks that only later rows see have no part in the row's reference: their values may be far larger
                        if (key0 >= lim) sc01.y = 0.f;
                        if (key0 + KV8_BLOCK >= lim) sc01.w = 0.f;
                        if (key0 + 2 * KV8_BLOCK >= lim) sc23.y = 0.f;
                        if (key0 + 3 * KV8_BLOCK >= lim) sc23.w = 0.f;
                    }
                    const uint32_t top_vs = max(max(__float_as_uint(sc01.y), __float_as_uint(sc01.w)),
                                                max(__float_as_uint(sc23.y), __float_as_uint(sc23.w)));
                    const uint32_t top_ref = max(ref, (top_vs & 0x7f800000u) + 0x00800000u);
                    const float inv_ref = __uint_as_float(0x7f000000u - top_ref);
                    const float ks[MINE] = {half ? sc23.x : sc01.x, half ? sc23.z : sc01.z};
                    const float vs[MINE] = {half ? sc23.y : sc01.y, half ? sc23.w : sc01.w};
                    // scores in base-2 units, from column c of the thread's 64; -inf where a mask covers them
                    const auto scores = [&](auto& s, int c) {
                        const float f = ks[c / KV8_BLOCK] * unit;
                        constexpr int n = sizeof(s) / 4;
#pragma unroll
                        for (int e = 0; e < n; e += 2) {
                            const float2 x = mul2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), make_float2(f, f));
                            s[e] = __float_as_uint(x.x);
                            s[e + 1] = __float_as_uint(x.y);
                        }
                        if (masked) {
                            const int key = key0 + half * 64 + c;
#pragma unroll
                            for (int e = 0; e < n; e++)
                                if (key + e >= lim || key + e < first) s[e] = __float_as_uint(-INFINITY);
                        }
                    };
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < MINE; k++) {
                        uint32_t s[32];
                        tmem_ld32(s_addr + k * 32, s);
                        tmem_ld_wait();
                        scores(s, k * 32);
#pragma unroll
                        for (int e = 0; e < 32; e += 8)
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                mx[c] = fmax3(mx[c], __uint_as_float(s[e + c]), __uint_as_float(s[e + 4 + c]));
                    }
                    float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    // (the next tile's S waits for both threads' P, so for both reads)
                    sm.part[t][half][r] = top;
                    ok = all_of(pair, 64, ok);
                    if (!ok) break;
                    top = fmaxf(top, sm.part[t][half ^ 1][r]);
                    const bool grow = top > m + kStale;  // from nothing, too
                    const float was = m;
                    if (grow) m = top;
                    const float base = m == -INFINITY ? 0.f : m;
                    const float alpha = grow ? exp2_approx(was - base) : 1.f;
                    const float keep = alpha * (__uint_as_float(ref) * inv_ref);
                    ref = top_ref;
                    // O is complete (and the last P read): S was computed after that PV, or waits for it here
                    if (BESIDE<D, P> && j > 0) {
                        ok = mbar_wait_warp(&sm.pv_done[t], (j - 1) & 1, err);
                        tc_fence_after();
                    }
                    if (j > 0 && __any_sync(0xffffffffu, keep != 1.f)) {
#pragma unroll
                        for (int c = 0; c < D / 64; c++) {
                            uint32_t o[32];
                            tmem_ld32(o_addr + c * 32, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tmem_st32(o_addr + c * 32, o);
                        }
                    }
                    const float2 nb = make_float2(-base, -base);
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < 64; c += 16) {
                        const float u = vs[c / KV8_BLOCK] * inv_ref * kUnit;
                        uint32_t s[16], w[8][P];
                        tmem_ld16(s_addr + c, s);
                        tmem_ld_wait();
                        scores(s, c);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            float2 x = add2(make_float2(__uint_as_float(s[e]), __uint_as_float(s[e + 1])), nb);
                            x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                            sum = add2(sum, x);
                            x = mul2(x, make_float2(u, u));
                            pieces_of<P>(x.x, x.y, w[e / 2]);
                        }
                        // over the same 16 keys' scores
#pragma unroll
                        for (int k = 0; k < P; k++) {
                            uint32_t o[8];
#pragma unroll
                            for (int e = 0; e < 8; e++) o[e] = w[e][k];
                            tmem_st8(BESIDE<D, P> ? p_addr + c / 2 : s_addr + c + k * 8, o);
                        }
                    }
                    if (BESIDE<D, P>) {  // S has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.s_free[t]);
                    }
                    l = l * alpha + (sum.x + sum.y);
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.p_full[t]);
                }
                if (!ok) break;  // both threads of a row know
                if (P == 2 && n_tiles > run) {
                    // O's sums of the run: to where they wait, on top of those that wait there; the last run's O is
                    // completed by them. They wait in their own columns, 16 at a time, of the tile's rows, 4 lanes to
                    // 64 bytes of a row if all of the warp's rows are live (a thread finds its own again, in
                    // whatever row), else each thread in its own.
                    const bool spread = splits > 1 || live_rows == 0xffffffffu, whole = splits > 1 || (vec & 2), last = stop == n_tiles;
                    float* at[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const int rr = spread ? u * 8 + lane / 4 : lane, c = half * (D / 2) + (spread ? lane & 3 : u) * 4;
                        const size_t off = __shfl_sync(0xffffffffu, i * p.out.ts + in_token, rr);
                        at[u] = (splits > 1 ? p.ws + z + (((size_t)bh * gridDim.x + blockIdx.x) * 2 * BM + t * BM + quarter * 32 + rr) * (D + 4) + 4
                                            : static_cast<float*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + off) + c;
                    }
                    const float old_f = m_out == m ? 1.f : exp2_approx(m_out - m);
                    const float f = last ? 1.f : __uint_as_float(ref) * (1.f / kUnit), to_f = last ? __uint_as_float(0x7f000000u - ref) : 1.f;
                    m_out = m;
                    ok = mbar_wait_warp(&sm.pv_done[t], (stop - 1) & 1, err);
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 16) {
                        float4 had[4] = {};
                        uint32_t o[16];
                        if (stop > run && live) {
#pragma unroll
                            for (int u = 0; u < 4; u++) had[u] = had_at(at[u] + c, whole);
                        }
                        tmem_ld16(o_addr + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const float4 y = summed(o + u * 4, f, had[u], to_f, last ? old_f * kUnit : old_f);
                            o[u * 4] = __float_as_uint(y.x);
                            o[u * 4 + 1] = __float_as_uint(y.y);
                            o[u * 4 + 2] = __float_as_uint(y.z);
                            o[u * 4 + 3] = __float_as_uint(y.w);
                            if (ok && live && !last) store4(at[u] + c, y, 1.f, whole);
                        }
                        if (last) tmem_st16(o_addr + c, o);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                }
                if (stop == n_tiles) break;  // (a wait that gave up here is known to both after the next exchange)
            }
            // the rows' outputs, or their part of the keys' cuts: the two threads' sums, then O through the warp's
            // part of the queries' shared memory, 16 columns at a time, so that 4 lanes write 64 consecutive bytes
            // (of f32) of a row
            if (ok && n_tiles > 0) ok = mbar_wait_warp(&sm.pv_done[t], (n_tiles - 1) & 1, err);
            tc_fence_after();
            sm.part[t][half][r] = l;
            ok = all_of(pair, 64, ok);
            l += sm.part[t][half ^ 1][r];
            const float units = __uint_as_float(ref) * (1.f / kUnit);
            const float f = splits > 1 ? units : l == 0.f ? 0.f : units / l;
            T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs;
            const size_t out_off = i * p.out.ts + in_token;
            float* ws = p.ws + z + (((size_t)bh * gridDim.x + blockIdx.x) * 2 * BM + t * BM + quarter * 32) * (D + 4);
            uint8_t* stage = &sm.q[t][0][0][0] + (quarter * 2 + half) * 2048;
#pragma unroll 1
            for (int c = 0; c < D / 2; c += 16) {
                uint32_t o[16] = {};
                if (n_tiles > 0) {
                    tmem_ld16(o_addr + c, o);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int u = 0; u < 4; u++)
                    *reinterpret_cast<float4*>(stage + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) =
                        make_float4(__uint_as_float(o[u * 4]) * f, __uint_as_float(o[u * 4 + 1]) * f,
                                    __uint_as_float(o[u * 4 + 2]) * f, __uint_as_float(o[u * 4 + 3]) * f);
                __syncwarp();
#pragma unroll
                for (int n = 0; n < 32; n += 8) {
                    const int rr = n + lane / 4, u = lane & 3, col = half * (D / 2) + c + u * 4;
                    const float4 y = *reinterpret_cast<const float4*>(stage + rr * 64 + ((u ^ (rr >> 1 & 3)) << 4));
                    const size_t off = __shfl_sync(0xffffffffu, out_off, rr);
                    if (ok && (live_rows >> rr & 1)) {
                        if (splits > 1) store4(ws + rr * (D + 4) + 4 + col, y, 1.f, true);
                        else store4(out + off + col, y, 1.f, vec & 2);
                    }
                }
                __syncwarp();
            }
            if (splits > 1 && live && ok && half == 0) *reinterpret_cast<float2*>(ws + lane * (D + 4)) = make_float2(m, l);
            __syncwarp();
            tc_fence_before();
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == ISSUER) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

template <typename T, int D, int P>
int launch(const Kv8Attn& p, int splits, cudaStream_t st) {
    const auto kern = kv8_prefill_kernel<T, D, P>;
    constexpr int smem = sizeof(Smem<D, P>);
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    static std::atomic<uint64_t> done{0};
    if (allow_smem(done, (const void*)kern, smem) != cudaSuccess) return -1;
    const int rows = p.s.n * (p.n_head / p.c.n_head_kv), tiles = (rows + KV8_PREFILL_ROWS - 1) / KV8_PREFILL_ROWS;
    const float scale = (float)(1.0 / sqrt((double)D)) * kLog2e;
    const int vec = (wide(p.q, sizeof(T), 16) ? 1 : 0) | (wide(p.out, sizeof(T), 4 * sizeof(T)) ? 2 : 0);
    return launch_chained_smem(kern, dim3((unsigned)(tiles * splits), (unsigned)(p.s.n_batch * p.c.n_head_kv)), dim3(THREADS),
                               smem, st, p, splits, vec, scale) == cudaSuccess
               ? 0
               : -1;
}

}  // namespace

int kv8_prefill_launch(const Kv8Attn& p, int type, int pieces, int splits, cudaStream_t st) {
    static_assert(KV8_PREFILL_ROWS == 2 * BM && KV8_PREFILL_KEYS == BN, "the plan's tiles are the kernel's");
    if (type == TYPE_BF16) return p.c.d == 64 ? launch<__nv_bfloat16, 64, 1>(p, splits, st) : launch<__nv_bfloat16, 128, 1>(p, splits, st);
    if (pieces == 1) return p.c.d == 64 ? launch<float, 64, 1>(p, splits, st) : launch<float, 128, 1>(p, splits, st);
    return p.c.d == 64 ? launch<float, 64, 2>(p, splits, st) : launch<float, 128, 2>(p, splits, st);
}

}  // namespace zwg
