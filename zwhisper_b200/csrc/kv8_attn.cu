// Attention over a cache in 8 bits (zwg_kv8_attn): softmax(q . (ks K) / sqrt(d)) (vs V), K and V
// int8 with a scale for each block of 32 tokens and kv head.
//
// kv8_split_kernel. The int8 values are exact in f16, so both products run on the tensor cores
// (mma.sync m16n8k16, f32 sums) with the scales outside of them: a query is one or two f16
// pieces of q / 2^e (e the exponent of its largest element), a score is the integer dot product
// times ks * 2^e / sqrt(d), a probability is one or two f16 pieces of 2^15 p vs / (the largest vs
// so far), and the sum of products is scaled by that largest vs in the end. Two pieces hold 22
// bits, so the result has the accuracy of f32 sums; one holds the 11 bits of the tf32 math mode,
// and of bf16 rows more than they have.
// The keys are the M side: S^T = K Q^T and O^T = V^T P^T, so the 8-wide N side is the rows of a
// kv head's query group (6 to 8 rows waste little), and S^T turns into the operand P^T by four
// 8x8 register transposes (movmatrix). A lane's operands are contiguous bytes of the cache: the
// order of the d elements inside a dot product and of the tokens inside a sum is free, so lane
// (g, t) takes 16 consecutive bytes of a key's row and 8 consecutive tokens of a value's column,
// and no shared memory or shuffle stands between memory and the tensor cores.
// A warp takes whole blocks of the split's range, each one bulk copy of its keys and one of its
// values into the warp's own ring in shared memory, so a warp never waits for another one before the
// merge, and loads run ahead of the arithmetic.
// The splits of a (sequence, kv head, tile of query rows) that fit a cluster (8 CTAs) meet in each
// other's shared memory; more of them write partials (m, l, O) for kv8_combine_kernel.
//
// A decode step is bound by the cache's bytes: 64 sequences, 12 / 2 heads of d 128, f32 queries, in a graph
// 17.5 us at 2256 tokens (75 MB, 4.3 TB/s), 30.1 at 4512, 52.4 at 9024 (298 MB, 5.7 TB/s; 6.6 TB/s from one
// length to the next, so what is left is the start, the merge and the launch, 5 us). Few sequences are bound
// by latency: one of 2256 tokens 7.5 us, of 65536 16.3 us. Two of 131001 in bf16 31.2 us: 6.0 TB/s to the next length,
// so 22 us of bytes and 9 of start, partials and second kernel. A block's products start from zero and are added to O
// rounded, since the tensor cores truncate their sums: off by 2.3e-7 to 2.6e-7 from 500 to 100000 keys, by 2.9e-7 to
// 5.7e-7 where the keys have a few strong channels (the f32 library form: 0.4e-6 to 1.6e-6); summed in O itself 1.4e-6
// after 100000 keys, and 0 to 4 % faster at d 128, 2 to 4 % slower at d 64 (O was rescaled apart).
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv8_attn.cuh"
#include "seqs.cuh"
#include "sm100.cuh"

namespace zwg {
namespace {

namespace cg = cooperative_groups;
using namespace kv8;

constexpr float kUnit = 32768.f;  // P's f16 pieces hold 2^15 p: small probabilities stay normal

ZWG_DEV void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

ZWG_DEV uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

constexpr int SMALL = 4;            // warps of a small CTA, three of which share an SM
constexpr int MAX_CLUSTER = 8;
constexpr int MOST_SPLIT_ROWS = 48;  // query rows of a kv head above which the tcgen05 kernel may run
constexpr int WARP_RING = 16 * 1024;  // bytes a warp has for blocks on their way

struct Plan {
    int tile_rows, tiles;  // query rows of a tile, tiles of a (sequence, kv head)
    int warps;   // of a CTA; 0: the tcgen05 kernel's
    int splits;  // cuts of the keys
    size_t ws;   // floats of workspace for this and shorter caches: a long cache's serves shorter ones
    float us;    // about how long it takes, for a choice between the kernels
    int in_place() const { return warps ? MAX_CLUSTER : 1; }  // cuts that need no workspace
};

// Warps of a CTA that has an SM to itself; the registers of two N tiles leave room for 8.
constexpr int big_warps(int tile_rows) { return tile_rows == 8 ? 12 : 8; }

// Clusters of n CTAs that run at once on the current device: a cluster lives in one GPC, and the GPCs
// have different numbers of SMs (n 4: 33 of 148 SMs, n 8: 15). Asked once for each device.
int clusters_of(int tile_rows, bool big, int n);
int clusters_at_once(int tile_rows, bool big, int n) {
    static std::atomic<int> known[64][2][2][MAX_CLUSTER + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    std::atomic<int>& at = known[dev & 63][tile_rows == 8][big][n];
    int count = at.load(std::memory_order_relaxed);
    if (count == 0) at.store(count = std::max(1, clusters_of(tile_rows, big, n)), std::memory_order_relaxed);
    return count;
}

// How the keys of `ctas` (sequence, kv head, tile of rows)s are cut for CTAs of one kind, and what it
// costs: the blocks that follow each other in a warp, and 0.7 of one for the second kernel.
struct Cut {
    int splits, most_splits;  // most: with any shorter cache
    float cost;
};
Cut cut_for(int tile_rows, bool big, long long ctas, int blocks, int combine_rows, int sm_count) {
    const int warps = big ? big_warps(tile_rows) : SMALL, per_sm = big_warps(tile_rows) / warps;
    const int useful = (blocks + warps - 1) / warps;
    const auto rounds = [&](int n) { return (useful + n - 1) / n; };
    // one wave of clusters: one that waits for a second wave doubles the time (8 sequences of 4512 tokens in
    // clusters of 8, of which 15 fit: 19.5 us, of 6: 11.3)
    int in_cluster = (int)std::min<long long>(std::min(MAX_CLUSTER, useful), std::max<long long>(1, (long long)per_sm * sm_count / ctas));
    while (in_cluster > 1 && ctas > clusters_at_once(tile_rows, big, in_cluster)) in_cluster--;
    // More splits than that, and the combining kernel, whose CTAs start early if places are left for them:
    // 8 to an SM, 2 beside two small CTAs (2 sequences of 20001 tokens: all SMs taken 14.4 us, 108 of them 12.2)
    const long long places = (long long)per_sm * sm_count - (combine_rows + 8 / per_sm - 1) / (8 / per_sm);
    const int most = (int)std::min<long long>(useful, places / ctas);
    Cut c{in_cluster, in_cluster, (float)rounds(in_cluster)};
    if (most > MAX_CLUSTER) {
        const int r = rounds(most);
        if (r + 0.7f < c.cost) c = {std::max(MAX_CLUSTER + 1, (useful + r - 1) / r), most, r + 0.7f};
        c.most_splits = most;
    }
    return c;
}

size_t workspace_of(const Kv8& c, const Seqs& s, const Plan& p, int most_splits) {
    if (most_splits <= p.in_place()) return 0;
    return (size_t)s.n_batch * c.n_head_kv * p.tiles * most_splits * p.tile_rows * (c.d + 4);
}

// Keys that the longest sequence can have at the call's end: no more than the cache, wherever n_past, the most
// that any past[b] may be, lies.
int keys_of(const Kv8& c, const Seqs& s) { return (int)std::min<long long>((long long)s.n_past + s.n, (long long)c.blocks * KV8_BLOCK); }

// Blocks of keys that a query sees, on average.
float blocks_seen(const Seqs& s) { return (s.n_past + 0.5f * s.n) / KV8_BLOCK + 1.f; }

// The tcgen05 kernel: keys are cut while SMs stay empty, two tiles of keys to a cut at least.
Plan plan_tc(const Kv8& c, const Seqs& s, int rows, int sm_count) {
    Plan p{KV8_PREFILL_ROWS, (rows + KV8_PREFILL_ROWS - 1) / KV8_PREFILL_ROWS, 0, 1, 0, 0.f};
    const long long ctas = (long long)s.n_batch * c.n_head_kv * p.tiles;
    const int key_tiles = (keys_of(c, s) + KV8_PREFILL_KEYS - 1) / KV8_PREFILL_KEYS;
    p.splits = (int)std::min<long long>(std::max<long long>(1, sm_count / ctas), std::max(1, key_tiles / 2));
    p.ws = workspace_of(c, s, p, p.splits);
    // a CTA's start and end and its key tiles, as measured with f32 queries; cuts go through memory twice
    const float turns = std::ceil(blocks_seen(s) / (KV8_PREFILL_KEYS / KV8_BLOCK) / p.splits), two = rows > KV8_PREFILL_ROWS / 2;
    const float cta = (two ? c.d == 64 ? 11.f : 13.f : c.d == 64 ? 8.5f : 9.5f) + turns * (two ? c.d == 64 ? 4.6f : 5.3f : c.d == 64 ? 3.f : 3.5f);
    p.us = (float)((ctas * p.splits + sm_count - 1) / sm_count) * cta;
    if (p.splits > 1) p.us += 3.f + 5.f * rows * s.n_batch * c.n_head_kv * p.splits * (c.d + 4) / 3e6f;
    return p;
}

// Splits of small CTAs with one block for each warp.
int one_each(int blocks) { return (blocks + SMALL - 1) / SMALL; }

Plan plan_split(const Kv8& c, const Seqs& s, int rows, int n_head, int sm_count) {
    Plan p{};
    p.tile_rows = rows <= 8 ? 8 : 16;  // one or two 8-wide N tiles
    p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
    const int big = big_warps(p.tile_rows);
    const long long ctas = (long long)s.n_batch * c.n_head_kv * p.tiles;
    const int blocks = (keys_of(c, s) + KV8_BLOCK - 1) / KV8_BLOCK;
    const int combine_rows = (int)std::min<long long>((long long)s.n_batch * s.n * n_head, 8 * sm_count);
    // most CTAs for which one block to each warp of small CTAs was the fastest plan: half the SMs
    const int few = (int)(sm_count / 2 / ctas);
    int most = 1;
    if (blocks <= 2 * big && ctas <= sm_count) {
        // no cut: merging two CTAs takes longer than a second block to each warp
        p.warps = blocks <= SMALL ? SMALL : big;
        p.splits = 1;
    } else if (one_each(blocks) <= few || (one_each(blocks) <= MAX_CLUSTER && ctas <= clusters_at_once(p.tile_rows, false, one_each(blocks)))) {
        p.warps = SMALL;
        p.splits = one_each(blocks);
    } else {
        // big CTAs (fewer states to merge) unless small ones leave fewer places empty
        const Cut small = cut_for(p.tile_rows, false, ctas, blocks, combine_rows, sm_count);
        const Cut large = cut_for(p.tile_rows, true, ctas, blocks, combine_rows, sm_count);
        const bool use_big = ctas <= sm_count && large.cost <= small.cost;
        p.warps = use_big ? big : SMALL;
        p.splits = use_big ? large.splits : small.splits;
        // big CTAs in clusters that put as many warps to work cost no more with any cache
        const int in_cluster = cut_for(p.tile_rows, true, ctas, big * MAX_CLUSTER, combine_rows, sm_count).splits;
        const int small_most = cut_for(p.tile_rows, false, ctas, 1 << 20, combine_rows, sm_count).most_splits;
        const bool always_big = ctas <= sm_count && large.most_splits <= MAX_CLUSTER && in_cluster * big >= small_most * SMALL;
        most = always_big ? 1 : std::max(large.most_splits, small.most_splits);
    }
    p.ws = workspace_of(c, s, p, std::max(most, std::max(p.splits, std::min(few, one_each(blocks)))));
    // waves of CTAs, each with its start, its merge and the blocks that follow each other in a warp
    const float turns = std::ceil(blocks_seen(s) / (p.splits * p.warps)), d64 = c.d == 64;
    const float waves = (float)(ctas * p.splits) / (sm_count * (big / p.warps)), whole = std::floor(waves);
    p.us = std::max(1.f, whole == waves ? waves : whole + 0.5f + 0.5f * (waves - whole)) * (d64 ? 3.5f + 1.2f * turns : 4.5f + 1.9f * turns);
    if (p.splits > MAX_CLUSTER) p.us += 2.f;
    return p;
}

// The tcgen05 kernel has four times the other one's rate, but 10 us of start and end for a CTA of 256 rows and
// 128 keys at a time. Both were timed for 24 to 1536 rows a head, 1 to 64 sequences, 200 to 8000 tokens, both d and
// f32, tf32 and bf16. Up to 48 rows the other one was at most 3 % the slower one (64 sequences of 200 tokens, 48 rows,
// d 128, bf16 14.6 us against 15.0; of 2000 62 against 86 in f32, 55 against 57 in bf16; one of 8000 13 against 24); above,
// the shorter estimate: 16 sequences of 2000 tokens, d 128, 288 rows 75 us against 69, 1536 rows 408 against 228; one
// of 200 tokens, 1536 rows 12.9 against 28.9. Its constants are f32's; with one piece both kernels take 0.6 to 0.85 of
// that, and the choice is as good: on average 1.4 % from the better in every type, at worst 1.5 times (f32) and 1.6 times
// (16 sequences of 8000 tokens, 144 rows, d 64, bf16: 98 us for 60).
Plan plan_for(const Kv8& c, const Seqs& s, int n_head, int sm_count) {
    const int rows = s.n * (n_head / c.n_head_kv);
    Plan split = plan_split(c, s, rows, n_head, sm_count);
    if (rows <= MOST_SPLIT_ROWS) return split;
    Plan tc = plan_tc(c, s, rows, sm_count);
    split.ws = tc.ws = std::max(split.ws, tc.ws);
    return split.us < tc.us ? split : tc;
}

// What each of n softmax states (m, l) weighs in their sum: f[i] = 2^(m_i - max), and the sum of l f.
struct Sum {
    float m, l;
};
template <typename M>
ZWG_DEV Sum weigh(int n, M state, float* f, int step) {
    Sum x{-INFINITY, 0.f};
    for (int i = 0; i < n; i++) x.m = fmaxf(x.m, state(i).x);
    const float base = x.m == -INFINITY ? 0.f : x.m;
    for (int i = 0; i < n; i++) {
        const float2 ml = state(i);
        f[i * step] = exp2_approx(ml.x - base);
        x.l += ml.y * f[i * step];
    }
    return x;
}

ZWG_DEV void add4(float4& a, float f, float4 x) {
    a.x += f * x.x;
    a.y += f * x.y;
    a.z += f * x.z;
    a.w += f * x.w;
}

// The blocks [from, to) of a split: the tile's keys first .. past + (the last row's query).
struct Range {
    int rows, row0, last_row, first, seen_by_all, from, to;
};
template <int R>
ZWG_DEV Range range_of(Place at, int first, int group, int tile, int split, int splits) {
    Range r;
    r.rows = at.count * group;
    r.row0 = tile * R;
    r.last_row = min(r.rows, r.row0 + R) - 1;
    r.first = first;
    const int q0 = r.row0 / group, q1 = r.last_row / group;
    r.seen_by_all = at.past + q0 + 1;  // keys the tile's first row sees
    const int lo = first / KV8_BLOCK, n = max(0, (at.past + q1 + KV8_BLOCK) / KV8_BLOCK - lo);
    const int each = n / splits, more = n - each * splits;
    r.from = lo + split * each + min(split, more);
    r.to = r.from + each + (split < more ? 1 : 0);
    return r;
}

template <typename T, int D, int NT, int P, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
    kv8_split_kernel(Kv8Attn p, int splits, int clustered, int vec, float scale) {
    chain_release();
    constexpr int R = 8 * NT, CH = D / 64, LDO = D + 4;
    constexpr int BYTES = KV8_BLOCK * D, STAGES = WARP_RING / (2 * BYTES);
    static_assert(R * LDO * sizeof(float) <= WARP_RING, "the merge fits the ring");
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ uint64_t full[WARPS][STAGES];
    __shared__ float2 state[WARPS][R], merged[R];
    __shared__ float weight[WARPS > MAX_CLUSTER ? WARPS : MAX_CLUSTER][R], inv_l[R];
    const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = p.n_head / p.c.n_head_kv, room = p.c.blocks * KV8_BLOCK;
    const size_t head = (size_t)bh * p.c.blocks;
    if (lane == 0) {
        for (int s = 0; s < STAGES; s++) sm100::mbar_init(&full[warp][s], 1);
        sm100::fence_mbar_init();
        sm100::fence_proxy_async_smem();
        // before the kernel ahead is through: a hint to L2 for the warp's first blocks, from places that
        // kernel may still be changing (held within the cache, and read again below)
        Place hint{p.s.past ? min(max(__ldcg(p.s.past + b), 0), room - 1) : p.s.n_past,
                   p.s.count ? min(max(__ldcg(p.s.count + b), 1), p.s.n) : p.s.n};
        const int f = p.s.first ? min(max(__ldcg(p.s.first + b), 0), room - 1) : 0;
        const Range r = range_of<R>(hint, f, group, tile, split, splits);
        for (int s = 0; s < STAGES; s++) {
            const int blk = r.from + warp + s * WARPS;
            if (blk < r.to && blk < p.c.blocks) {
                sm100::bulk_hint(p.c.k + (head + blk) * BYTES, BYTES);
                sm100::bulk_hint(p.c.v + (head + blk) * BYTES, BYTES);
            }
        }
    }
    const int z = chain_wait();
    const Place at = place_of(p.s, b, room, threadIdx.x == 0 && blockIdx.x == 0 && h == 0 ? p.err : nullptr);
    const int first = p.s.first ? __ldcg(p.s.first + b + z) : 0;
    const Range rg = range_of<R>(at, max(first, 0), group, tile, split, splits);
    const int rows = rg.rows, row0 = rg.row0, from = rg.from, to = rg.to;
    if (row0 >= rows) return;  // the same for every CTA of a cluster
    if (first < 0) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }

    unsigned char* mine = ring + warp * (STAGES * 2 * BYTES);
    const auto load = [&](int blk, int stage) {
        sm100::mbar_arrive_expect_tx(&full[warp][stage], 2 * BYTES);
        sm100::bulk_load(mine + stage * 2 * BYTES, p.c.k + (head + blk) * BYTES + z, BYTES, &full[warp][stage]);
        sm100::bulk_load(mine + stage * 2 * BYTES + BYTES, p.c.v + (head + blk) * BYTES + z, BYTES, &full[warp][stage]);
    };
    if (lane == 0)
        for (int s = 0; s < STAGES; s++)
            if (from + warp + s * WARPS < to) load(from + warp + s * WARPS, s);
    __syncwarp();
    float next_ks = 0.f, next_vs = 0.f;
    if (from + warp < to) {
        next_ks = __ldcg(p.c.k_scale + head + from + warp + z);
        next_vs = __ldcg(p.c.v_scale + head + from + warp + z);
    }

    // queries: the B operand, lane (g, t) holds row g's 16 consecutive elements of each 64
    uint32_t qf[NT][CH][4][P][2];
    float unit[NT][2];  // of the columns 2t, 2t + 1: 2^e * log2(e) / sqrt(d)
    int lim[NT][2];     // keys below it are seen
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int row = row0 + nt * 8 + g;
        float x[CH][16] = {};
        float top = 0.f;
        if (row < rows) {
            const int i = row / group;
            const T* q = static_cast<const T*>(p.q.data) + z + b * p.q.bs + i * p.q.ts + (size_t)(h * group + row - i * group) * D;
#pragma unroll
            for (int c = 0; c < CH; c++) load16(q + c * 64 + t * 16, x[c], vec & 1);
        }
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int e = 0; e < 16; e++) top = fmaxf(top, fabsf(x[c][e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float pw, inv;
        power_of(top, pw, inv);
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    uint32_t w[P];
                    pieces_of<P>(x[i][s * 4 + e * 2] * inv, x[i][s * 4 + e * 2 + 1] * inv, w);
#pragma unroll
                    for (int c = 0; c < P; c++) qf[nt][i][s][c][e] = w[c];
                }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            unit[nt][e] = __shfl_sync(0xffffffffu, pw, (2 * t + e) * 4) * scale;
            const int r = row0 + nt * 8 + 2 * t + e;
            lim[nt][e] = r < rows ? at.past + r / group + 1 : 0;
        }
    }

    float o[D / 16][NT][4] = {}, m[NT][2], l[NT][2];
    uint32_t ref = 0x00800000u;  // bits of a power of two above every vs so far (2^-126 at least)
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.f;
        }

    int stage = 0;
    uint32_t phase = 0;
    for (int blk = from + warp; blk < to; blk += WARPS) {
        float ks = next_ks, vs = next_vs;
        if (blk + WARPS < to) {
            next_ks = __ldcg(p.c.k_scale + head + blk + WARPS + z);
            next_vs = __ldcg(p.c.v_scale + head + blk + WARPS + z);
        }
        if (vs != vs) {  // values that read as NaN: through the scores, which a mask covers
            ks = vs;
            vs = 0.f;
        }
        if (!sm100::mbar_wait_warp(&full[warp][stage], phase, p.err)) {
            // gave up: no further copies; those on their way end before the ring is used again
            for (int s = 0; s < STAGES && blk + s * WARPS < to; s++) {
                const int at_stage = (stage + s) % STAGES;
                sm100::mbar_wait_drain(&full[warp][at_stage], at_stage < stage ? phase ^ 1 : phase);
            }
            break;
        }
        const unsigned char* kb = mine + stage * 2 * BYTES;
        const unsigned char* vb = kb + BYTES;
        // S^T: rows are tokens, logical row (mt, hf, r) is token (r / 2) * 8 + mt * 4 + hf * 2 + r % 2
        // (two sums for each: shorter chains of dependent products)
        float s[2][NT][4] = {}, s2[2][NT][4] = {};
        uint4 kw[2][2][CH];
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int i = 0; i < CH; i++)
                    kw[mt][hf][i] = *reinterpret_cast<const uint4*>(
                        kb + ((g >> 1) * 8 + mt * 4 + hf * 2 + (g & 1)) * D + i * 64 + t * 16);
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int st = 0; st < 4; st++)
#pragma unroll
                for (int mt = 0; mt < 2; mt++) {
                    uint32_t a0, a1, a2, a3;
                    ints_to_f16((&kw[mt][0][i].x)[st], a0, a2);
                    ints_to_f16((&kw[mt][1][i].x)[st], a1, a3);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int c = 0; c < P; c++)
                            mma((P == 2 ? c : i & 1) ? s2[mt][nt] : s[mt][nt], a0, a1, a2, a3, qf[nt][i][st][c][0],
                                qf[nt][i][st][c][1]);
                }
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[mt][nt][e] += s2[mt][nt][e];
        // softmax over the block, for the columns 2t and 2t + 1
        const uint32_t top = max(ref, (__float_as_uint(vs) & 0x7f800000u) + 0x00800000u);
        const float inv_top = __uint_as_float(0x7f000000u - top);
        const float ratio = vs * inv_top, shrink = __uint_as_float(ref) * inv_top;
        ref = top;
        uint32_t pt[2][2][NT][P];
        float keep[NT][2];
        const int key0 = blk * KV8_BLOCK;
        const bool masked = key0 + KV8_BLOCK > rg.seen_by_all || key0 < first;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float f = ks * unit[nt][e];
                float mx = m[nt][e];
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        const int key = key0 + (g >> 1) * 8 + mt * 4 + hf * 2 + (g & 1);
                        float& x = s[mt][nt][hf * 2 + e];
                        x *= f;
                        if (masked && (key >= lim[nt][e] || key < first)) x = -INFINITY;
                        mx = fmaxf(mx, x);
                    }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float base = mx == -INFINITY ? 0.f : mx;
                const float alpha = exp2_approx(m[nt][e] - base);
                m[nt][e] = mx;
                float sum = 0.f;
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float& x = s[mt][nt][hf * 2 + e];
                        x = exp2_approx(x - base);
                        sum += x;
                    }
                l[nt][e] = l[nt][e] * alpha + sum;
                keep[nt][e] = alpha * shrink;
            }
            const float f = ratio * kUnit;
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    uint32_t w[P];
                    pieces_of<P>(s[mt][nt][hf * 2] * f, s[mt][nt][hf * 2 + 1] * f, w);
#pragma unroll
                    for (int c = 0; c < P; c++) pt[mt][hf][nt][c] = transpose8x8(w[c]);
                }
        }
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
            uint2 vw[2];
            // a block's sums start from zero and are added rounded: the tensor cores truncate theirs
            float sum[NT][4] = {};
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
                vw[hf] = *reinterpret_cast<const uint2*>(vb + (j * 16 + hf * 8 + g) * KV8_BLOCK + t * 8);
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                uint32_t a0, a1, a2, a3;
                ints_to_f16(mt ? vw[0].y : vw[0].x, a0, a2);
                ints_to_f16(mt ? vw[1].y : vw[1].x, a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < P; c++) mma(sum[nt], a0, a1, a2, a3, pt[mt][0][nt][c], pt[mt][1][nt][c]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[j][nt][e] = o[j][nt][e] * keep[nt][e & 1] + sum[nt][e];
        }
        __syncwarp();  // every lane has read the stage
        if (lane == 0 && blk + STAGES * WARPS < to) load(blk + STAGES * WARPS, stage);
        if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
        }
    }

    // the warp's state: sums over the lanes, O in its true units
    __syncthreads();  // every warp is through with the ring
    float* sm_o = reinterpret_cast<float*>(ring);  // [WARPS][R][LDO]
    const float units = __uint_as_float(ref) * (1.f / kUnit);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float sum = l[nt][e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int r = nt * 8 + 2 * t + e;
            if (g == 0) state[warp][r] = make_float2(m[nt][e], sum);
            float* row = sm_o + (warp * R + r) * LDO;
#pragma unroll
            for (int j = 0; j < D / 16; j++) {
                row[j * 16 + g] = o[j][nt][e] * units;
                row[j * 16 + 8 + g] = o[j][nt][2 + e] * units;
            }
        }
    __syncthreads();
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        const Sum x = weigh(WARPS, [&](int w) { return state[w][r]; }, &weight[0][r], R);
        merged[r] = make_float2(x.m, x.l);
        inv_l[r] = x.l == 0.f ? 0.f : 1.f / x.l;
    }
    __syncthreads();
    // a thread has the same four columns of every row it takes
    constexpr int ROWS_AT_ONCE = 32 * WARPS / (D / 4);
    const int live = rg.last_row - row0 + 1, c4 = threadIdx.x % (D / 4) * 4, r0 = threadIdx.x / (D / 4);
    T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + (size_t)h * group * D + c4;
    for (int r = r0; r < live; r += ROWS_AT_ONCE) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < WARPS; w++)
            add4(acc, weight[w][r], *reinterpret_cast<const float4*>(sm_o + (w * R + r) * LDO + c4));
        if (splits == 1) {
            const int row = row0 + r, i = row / group;
            store4(out + i * p.out.ts + (size_t)(row - i * group) * D, acc, inv_l[r], vec & 2);
        } else if (clustered) {
            *reinterpret_cast<float4*>(sm_o + r * LDO + c4) = acc;  // warp 0's, which no other thread reads
        } else {
            float* ws = p.ws + z + (((size_t)bh * gridDim.x + blockIdx.x) * R + r) * (D + 4);
            *reinterpret_cast<float4*>(ws + 4 + c4) = acc;
            if (c4 == 0) *reinterpret_cast<float2*>(ws) = merged[r];
        }
    }
    if (splits == 1 || !clustered) return;
    // the cluster's CTAs: row r's outputs are the CTA's of rank r modulo their number
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x < R) {
        const int r = threadIdx.x;
        const Sum x = weigh(splits, [&](int s) { return *cluster.map_shared_rank(&merged[r], s); }, &weight[0][r], R);
        inv_l[r] = x.l == 0.f ? 0.f : 1.f / x.l;
    }
    __syncthreads();
    for (int r = split + splits * r0; r < live; r += splits * ROWS_AT_ONCE) {
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int s = 0; s < splits; s++)
            add4(acc, weight[s][r], *reinterpret_cast<const float4*>(cluster.map_shared_rank(sm_o, s) + r * LDO + c4));
        const int row = row0 + r, i = row / group;
        store4(out + i * p.out.ts + (size_t)(row - i * group) * D, acc, inv_l[r], vec & 2);
    }
    cluster.sync();  // the others have read this CTA's shared memory
}

// A CTA of 256 threads takes a query row: the splits' partials to the output. The weights of up to
// CHUNK splits at a time meet in shared memory, then each group of D / 4 threads sums every so many
// splits' O and the groups' sums are added.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_combine_kernel(Kv8Attn p, int splits, int R, int vec) {
    chain_release();
    const int z = chain_wait();
    constexpr int GROUPS = 256 / (D / 4);
    extern __shared__ float f[];  // [splits]
    __shared__ float part[8];
    __shared__ float4 sums[GROUPS][D / 4];
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv, row = blockIdx.x;
    const int group = p.n_head / p.c.n_head_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Place at = place_of(p.s, b, p.c.blocks * KV8_BLOCK, nullptr);
    if (row >= at.count * group || (p.s.first && __ldcg(p.s.first + b + z) < 0)) return;
    const int tiles = (p.s.n * group + R - 1) / R;
    const size_t step = (size_t)R * (D + 4);
    const float* ws = p.ws + z + ((size_t)bh * tiles + row / R) * splits * step + (row % R) * (D + 4);
    float mx = -INFINITY;
    for (int s = threadIdx.x; s < splits; s += 256) mx = fmaxf(mx, __ldcg(ws + s * step));
    mx = warp_max(mx);
    if (lane == 0) part[warp] = mx;
    __syncthreads();
    mx = part[0];
#pragma unroll
    for (int w = 1; w < 8; w++) mx = fmaxf(mx, part[w]);
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    for (int s = threadIdx.x; s < splits; s += 256) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(ws + s * step));
        f[s] = exp2_approx(ml.x - base);
        sum += ml.y * f[s];
    }
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) part[warp] = sum;
    __syncthreads();
    sum = part[0];
#pragma unroll
    for (int w = 1; w < 8; w++) sum += part[w];
    const int c = threadIdx.x % (D / 4), first = threadIdx.x / (D / 4);
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = first; s < splits; s += GROUPS)
        add4(acc, f[s], __ldcg(reinterpret_cast<const float4*>(ws + s * step + 4) + c));
    sums[first][c] = acc;
    __syncthreads();
    if (first > 0) return;
#pragma unroll
    for (int w = 1; w < GROUPS; w++) add4(acc, 1.f, sums[w][c]);
    const int i = row / group;
    T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + i * p.out.ts +
             (size_t)(h * group + row - i * group) * D + c * 4;
    store4(out, acc, sum == 0.f ? 0.f : 1.f / sum, vec & 2);
}

template <int NT, int WARPS>
int clusters_of_kind(int n) {
    const auto kern = kv8_split_kernel<float, 128, NT, 2, WARPS>;  // the others need no more than it
    static std::atomic<uint64_t> done{0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = WARPS * WARP_RING;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)n;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int count = 0;
    if (allow_smem(done, (const void*)kern, WARPS * WARP_RING) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&count, kern, &cfg) != cudaSuccess)
        (void)cudaGetLastError();
    return count;
}

int clusters_of(int tile_rows, bool big, int n) {
    if (tile_rows == 8) return big ? clusters_of_kind<1, big_warps(8)>(n) : clusters_of_kind<1, SMALL>(n);
    return big ? clusters_of_kind<2, big_warps(16)>(n) : clusters_of_kind<2, SMALL>(n);
}

// The same where rows are many: D / 4 threads take a row.
template <typename T, int D>
__global__ void __launch_bounds__(256) kv8_combine_rows_kernel(Kv8Attn p, int splits, int R, int vec) {
    chain_release();
    const int z = chain_wait();
    constexpr int GROUPS = 256 / (D / 4);
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv;
    const int group = p.n_head / p.c.n_head_kv, row = blockIdx.x * GROUPS + threadIdx.x / (D / 4), c = threadIdx.x % (D / 4);
    const Place at = place_of(p.s, b, p.c.blocks * KV8_BLOCK, nullptr);
    if (row >= at.count * group || (p.s.first && __ldcg(p.s.first + b + z) < 0)) return;
    const int tiles = (p.s.n * group + R - 1) / R;
    const size_t step = (size_t)R * (D + 4);
    const float* ws = p.ws + z + ((size_t)bh * tiles + row / R) * splits * step + (row % R) * (D + 4);
    float mx = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < splits; s++) mx = fmaxf(mx, __ldcg(ws + s * step));
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int s = 0; s < splits; s++) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(ws + s * step));
        const float f = exp2_approx(ml.x - base);
        sum += ml.y * f;
        add4(acc, f, __ldcg(reinterpret_cast<const float4*>(ws + s * step + 4) + c));
    }
    const int i = row / group;
    T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + i * p.out.ts +
             (size_t)(h * group + row - i * group) * D + c * 4;
    store4(out, acc, sum == 0.f ? 0.f : 1.f / sum, vec & 2);
}

template <typename T, int D, int NT, int P, int WARPS>
int split_launch(const Kv8Attn& p, const Plan& plan, int vec, cudaStream_t st) {
    constexpr int RING = WARPS * WARP_RING;
    const float scale = (float)(1.0 / sqrt((double)D)) * kLog2e;
    const unsigned segs = (unsigned)(p.s.n_batch * p.c.n_head_kv);
    const int clustered = plan.splits <= MAX_CLUSTER;
    const auto kern = kv8_split_kernel<T, D, NT, P, WARPS>;
    static std::atomic<uint64_t> done{0};
    if (allow_smem(done, (const void*)kern, RING) != cudaSuccess) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.tiles * plan.splits), segs);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = RING;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = clustered ? (unsigned)plan.splits : 1;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, p, plan.splits, clustered, vec, scale) == cudaSuccess ? 0 : -1;
}

template <typename T, int D, int NT, int P>
int split_of(const Kv8Attn& p, const Plan& plan, int vec, cudaStream_t st) {
    return plan.warps == SMALL ? split_launch<T, D, NT, P, SMALL>(p, plan, vec, st)
                               : split_launch<T, D, NT, P, big_warps(8 * NT)>(p, plan, vec, st);
}

template <typename T, int D>
int combine(const Kv8Attn& p, const Plan& plan, int rows, int vec, int sm_count, cudaStream_t st) {
    const unsigned segs = (unsigned)(p.s.n_batch * p.c.n_head_kv);
    cudaError_t e;
    if ((long long)rows * segs > 8 * sm_count) {  // more than a CTA to a row fits at once
        constexpr int GROUPS = 256 / (D / 4);
        e = launch_chained(kv8_combine_rows_kernel<T, D>, dim3((unsigned)(rows + GROUPS - 1) / GROUPS, segs), dim3(256), st, p,
                           plan.splits, plan.tile_rows, vec);
    } else {
        e = launch_chained_smem(kv8_combine_kernel<T, D>, dim3((unsigned)rows, segs), dim3(256), plan.splits * sizeof(float), st, p,
                                plan.splits, plan.tile_rows, vec);
    }
    return e == cudaSuccess ? 0 : -1;
}

template <typename T, int D>
int attn(const Kv8Attn& p, int pieces, int sm_count, cudaStream_t st) {
    const Plan plan = plan_for(p.c, p.s, p.n_head, sm_count);
    const int rows = p.s.n * (p.n_head / p.c.n_head_kv);
    const bool one = plan.tile_rows == 8, two_pieces = sizeof(T) == 4 && pieces == 2;  // bf16 queries are exact in one piece
    const int vec = (wide(p.q, sizeof(T), 16) ? 1 : 0) | (wide(p.out, sizeof(T), 4 * sizeof(T)) ? 2 : 0);
    int rc;
    if (plan.warps == 0) {
        rc = kv8_prefill_launch(p, sizeof(T) == 2 ? TYPE_BF16 : TYPE_F32, pieces, plan.splits, st);
    } else if (two_pieces) {
        if constexpr (sizeof(T) == 4) rc = one ? split_of<T, D, 1, 2>(p, plan, vec, st) : split_of<T, D, 2, 2>(p, plan, vec, st);
    } else {
        rc = one ? split_of<T, D, 1, 1>(p, plan, vec, st) : split_of<T, D, 2, 1>(p, plan, vec, st);
    }
    if (rc == 0 && plan.splits > plan.in_place()) rc = combine<T, D>(p, plan, rows, vec, sm_count, st);
    return rc;
}

}  // namespace

size_t kv8_attn_workspace_bytes(const Kv8& c, const Seqs& s, int n_head, int sm_count) {
    if (s.n_batch == 0 || s.n == 0) return 0;
    return plan_for(c, s, n_head, sm_count).ws * sizeof(float);
}

int kv8_attn_launch(const Kv8Attn& p, int type, int pieces, int sm_count, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    if (type == TYPE_BF16)
        return p.c.d == 64 ? attn<__nv_bfloat16, 64>(p, 1, sm_count, st) : attn<__nv_bfloat16, 128>(p, 1, sm_count, st);
    return p.c.d == 64 ? attn<float, 64>(p, pieces, sm_count, st) : attn<float, 128>(p, pieces, sm_count, st);
}

}  // namespace zwg
