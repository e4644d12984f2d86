// Attention over a cache in pages (zwg_paged_attn): softmax(q . K / sqrt(d)) V, K and V 16-bit floats in pages
// that a table names, for steps of a token, chunks of a prompt and trees of drafted tokens.
//
// paged_split_kernel. The keys are the M side of mma.sync m16n8k16: S^T = K Q^T and O^T = V^T P^T, so that the
// 8-wide N side is the rows (query * group + head) of a kv head's group, and S^T turns into the operand P^T by two
// 8x8 register transposes. A warp takes 16 keys of d 128 or 32 of d 64 at a time (4 KB of keys, 4 KB of values), 16 of
// which lie in one page. The order of the d elements in a dot product is free, so lane (g, t) loads 16 consecutive
// bytes of the rows of keys g and g + 8; the order of the rows of O^T is free, so it loads 16 consecutive bytes of the
// values of keys 2t, 2t + 1, 2t + 8 and 2t + 9 and pairs them up by byte permutes. So nothing but registers stands
// between memory and the tensor cores: a warp's next keys are on their way while this group's softmax runs, its next
// values from the end of this group's products.
// f32 rows: a query is one or two f16 pieces of q / 2^e (e the exponent of its largest element), a probability one or
// two of 2^15 p against f16 keys and values; two pieces hold 22 bits, so the result has the accuracy of f32 sums.
// bf16 rows: queries as they are, probabilities rounded to bf16, and the sum that divides takes the rounded ones, so
// that what a probability is off by weighs only how far its value is from the result.
// A CTA has 4 warps, or 12 (8 of two N tiles) and then an SM to itself: large ones merge more in their own shared memory,
// small ones start sooner and fill SMs evenly; the plan below weighs both. The splits of a (sequence, kv head, tile
// of rows) that fit a cluster (up to 16) push their parts into the shared memory of the CTA that ends the row, behind one
// barrier of the cluster; more of them write partials (m, l, O) for paged_combine_kernel. What the first two turns read is
// hinted to L2 while the kernel ahead still runs.
// Bound by HBM where there are many keys, by latency where there are few. 12 / 2 heads of d 128, bf16, in a graph:
// 64 sequences of 9024 tokens 92.1 us (6.4 TB/s), of 4512 50, of 2256 28.1; 2 of 131001 52.5 us (5.1 TB/s; 36 cuts,
// partials and the second kernel); one of 2256 5.8, of which the bytes are 0.35.
#include <algorithm>
#include <cmath>

#include <cooperative_groups.h>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv8_attn.cuh"
#include "paged.cuh"
#include "seqs.cuh"
#include "sm100.cuh"

namespace zwg {
namespace {

namespace cg = cooperative_groups;
using kv8::kLog2e;
using kv8::pieces_of;
using kv8::power_of;
using kv8::store4;
using kv8::wide;
using paged::finite;
using paged::Held;
using paged::page_of;
using paged::read_tree;
using paged::row_at;

constexpr int SMALL = 4;         // warps of a small CTA; a big one has an SM to itself
constexpr int big_warps(int tile_rows) { return tile_rows == 8 ? 12 : 8; }  // (two N tiles take twice the registers)
constexpr int GROUP = 16;        // keys of a product, which lie in one page
template <int D>
constexpr int KEYS = GROUP * 128 / D;  // of a warp at a time: 4 KB of them and 4 KB of values
constexpr int MAX_CLUSTER = 16;

ZWG_DEV void mma(__half, float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
ZWG_DEV void mma(__nv_bfloat16, float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

ZWG_DEV uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

ZWG_DEV uint4 load_cached(const uint16_t* p) { return __ldcg(reinterpret_cast<const uint4*>(p)); }
ZWG_DEV uint32_t word(const uint4& w, int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }

ZWG_DEV void add4(float4& a, float f, float4 x) {
    a.x += f * x.x;
    a.y += f * x.y;
    a.z += f * x.z;
    a.w += f * x.w;
}

// The sum of n partial results of a row: their states (m, l) and a piece of each one's O, weighed by 2^(m - the largest).
struct Sum {
    float m, l;
    float4 o;
};
template <typename M, typename O>
ZWG_DEV Sum sum_of(int n, M state, O piece) {
    Sum x{-INFINITY, 0.f, make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int i = 0; i < n; i++) x.m = fmaxf(x.m, state(i).x);
    const float base = x.m == -INFINITY ? 0.f : x.m;
#pragma unroll 4
    for (int i = 0; i < n; i++) {
        const float2 ml = state(i);
        const float f = exp2_approx(ml.x - base);
        x.l += ml.y * f;
        add4(x.o, f, piece(i));
    }
    return x;
}

// The turns [from, to) of a split, KEYS slots each: the tile's keys first .. past + (the last row's token).
struct Range {
    int rows, row0, seen_by_all, end, from, to;
};
template <int R, int KEYS>
ZWG_DEV Range range_of(Place at, int first, int group, int tile, int split, int splits, bool tree) {
    Range r;
    r.rows = at.count * group;
    r.row0 = tile * R;
    const int q0 = r.row0 / group, q1 = (min(r.rows, r.row0 + R) - 1) / group;
    r.seen_by_all = tree ? at.past : at.past + q0 + 1;  // slots below it: by every row of the tile
    r.end = at.past + q1 + 1;                           // slots from it on: by none
    const int lo = first / KEYS, n = first < r.end ? (r.end + KEYS - 1) / KEYS - lo : 0;
    const int each = n / splits, more = n - each * splits;
    r.from = lo + split * each + min(split, more);
    r.to = r.from + each + (split < more ? 1 : 0);
    return r;
}

// Rows of a cluster's merge: row r's is CTA r % splits, which has a place for every CTA's part of each of its own.
__host__ __device__ constexpr int rows_of_rank(int R, int splits) { return (R + splits - 1) / splits; }

template <typename T, int D, int NT, int P, int WARPS>
__global__ void __launch_bounds__(32 * WARPS, big_warps(8 * NT) / WARPS)
    paged_split_kernel(PagedAttn p, int splits, int clustered, int vec, float scale) {
    chain_release();
    using H = typename Held<T>::type;
    constexpr int R = 8 * NT, LDO = D + 4, KC = D / 32, VC = D / 64, TURN = KEYS<D>, U = TURN / GROUP;
    constexpr bool RAW = sizeof(T) == 2;        // queries as they are
    constexpr float SHIFT = RAW ? 0.f : 15.f;   // probabilities in units of 2^-15: their f16 pieces stay normal
    constexpr uint32_t EXP = Held<T>::exponent;
    extern __shared__ __align__(16) float sm_o[];  // [WARPS][R][LDO], then a cluster's inbox [splits][its rows][LDO]
    __shared__ float2 state[WARPS][R];
    __shared__ int parent[MOST_TREE];
    __shared__ uint32_t above[R][MOST_TREE / 32];  // a row's token and its ancestors
    const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = p.n_head / p.c.n_head_kv;
    const bool lead = threadIdx.x == 0 && blockIdx.x == 0 && h == 0, tree = p.tree.parent != nullptr;
    if (lane < 2 * U) {
        // before the kernel ahead is through: a hint to L2 for the warp's first two turns, from places that
        // kernel may still be changing (held within the cache, and read again below)
        const Place hint{p.s.past ? min(max(__ldcg(p.s.past + b), 0), p.c.room - 1) : p.s.n_past,
                         p.s.count ? min(max(__ldcg(p.s.count + b), 1), p.s.n) : p.s.n};
        const Range r = range_of<R, TURN>(hint, p.s.first ? min(max(__ldcg(p.s.first + b), 0), p.c.room - 1) : 0, group, tile, split, splits, tree);
        const int turn = r.from + warp + lane / U * WARPS, slot = turn * TURN + lane % U * GROUP;
        const int page = turn < r.to && slot < p.c.room ? page_of(p.c, b, slot) : -1;
        if (page >= 0) {
            const size_t at = row_at(p.c, page, h, slot) * 2;
            sm100::bulk_hint(static_cast<const char*>(p.c.k) + at, GROUP * D * 2);
            sm100::bulk_hint(static_cast<const char*>(p.c.v) + at, GROUP * D * 2);
        }
    }
    const int z = chain_wait();
    const Place at = place_of(p.s, b, p.c.room, lead ? p.err : nullptr);
    const int first = p.s.first ? __ldcg(p.s.first + b + z) : 0;
    const Range rg = range_of<R, TURN>(at, max(first, 0), group, tile, split, splits, tree);
    const int rows = rg.rows, row0 = rg.row0, to = rg.to;
    if (row0 >= rows) return;  // the same for every CTA of a cluster, as the next two
    if (first < 0) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    if (tree) {
        if (!read_tree(p.tree, b, at.count, z, parent)) {
            if (threadIdx.x == 0) set_error(p.err, kErrBounds);
            return;
        }
        if (threadIdx.x < R) {
            const int r = threadIdx.x;
            for (int w = 0; w < MOST_TREE / 32; w++) above[r][w] = 0;
            if (row0 + r < rows)
                for (int a = (row0 + r) / group; a >= 0; a = parent[a]) above[r][a >> 5] |= 1u << (a & 31);
        }
        __syncthreads();
    }
    __syncwarp();  // (the lanes of the hint: what follows is for whole warps)
    if (clustered) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // (waited for before the merge)

    // the pages of the warp's next 32 groups of keys, one in each lane
    int turn = rg.from + warp, pages = 0, it = 0;
    const auto look = [&](int from) {
        const int mine = from + lane / U * WARPS, slot = mine * TURN + lane % U * GROUP;
        // (a turn of two pages may begin with one before the first key, which may have been given back)
        pages = mine < to && slot < rg.end && (U == 1 || slot + GROUP > first) ? page_of(p.c, b, slot + z) : 0;
        if (pages < 0) set_error(p.err, kErrBounds);  // its keys are not seen
    };
    const auto page_in = [&](int (&page)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++) page[u] = __shfl_sync(0xffffffffu, pages, it * U + u);
    };
    uint4 kr[U][2][KC], vr[U][VC][4];
    const uint16_t* const kd = static_cast<const uint16_t*>(p.c.k) + z;
    const uint16_t* const vd = static_cast<const uint16_t*>(p.c.v) + z;
    const auto load_k = [&](const int (&page)[U], int slot) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint16_t* src = kd + row_at(p.c, max(page[u], 0), h, slot + u * GROUP) + g * D + t * 8;
#pragma unroll
            for (int m = 0; m < KC; m++) {
                kr[u][0][m] = load_cached(src + m * 32);
                kr[u][1][m] = load_cached(src + 8 * D + m * 32);
            }
        }
    };
    const auto load_v = [&](const int (&page)[U], int slot) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint16_t* src = vd + row_at(p.c, max(page[u], 0), h, slot + u * GROUP) + 2 * t * D + g * 8;
#pragma unroll
            for (int c = 0; c < VC; c++)
#pragma unroll
                for (int k = 0; k < 4; k++) vr[u][c][k] = load_cached(src + ((k & 1) + (k >> 1) * 8) * D + c * 64);
        }
    };
    look(turn);
    int page[U];
    page_in(page);
    if (turn < to) {
        load_k(page, turn * TURN);
        load_v(page, turn * TURN);
    }

    // queries: the B operand, lane (g, t) holds row g's elements 8 t .. 8 t + 7 of each 32
    uint32_t qf[NT][KC][2][P][2];
    float unit[NT][2];  // of the columns 2t, 2t + 1: 2^e * log2(e) / sqrt(d)
    int lim[NT][2];     // slots below it may be seen
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int row = row0 + nt * 8 + g, i = min(row, rows - 1) / group;
        const T* q = static_cast<const T*>(p.q.data) + z + b * p.q.bs + i * p.q.ts + (size_t)(h * group + min(row, rows - 1) - i * group) * D + t * 8;
        if constexpr (RAW) {
            unit[nt][0] = unit[nt][1] = scale;
#pragma unroll
            for (int m = 0; m < KC; m++) {
                uint32_t w[4];
                if (vec & 1) {
                    const uint4 x = *reinterpret_cast<const uint4*>(q + m * 32);
                    w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
                } else {
                    const uint16_t* u = reinterpret_cast<const uint16_t*>(q + m * 32);
#pragma unroll
                    for (int e = 0; e < 4; e++) w[e] = u[2 * e] | (uint32_t)u[2 * e + 1] << 16;
                }
#pragma unroll
                for (int e = 0; e < 4; e++) qf[nt][m][e >> 1][0][e & 1] = w[e];
            }
        } else {
            float x[KC][8];
            uint32_t top = 0;
#pragma unroll
            for (int m = 0; m < KC; m++) {
                if (vec & 1) {
                    *reinterpret_cast<float4*>(&x[m][0]) = *reinterpret_cast<const float4*>(q + m * 32);
                    *reinterpret_cast<float4*>(&x[m][4]) = *reinterpret_cast<const float4*>(q + m * 32 + 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) x[m][e] = q[m * 32 + e];
                }
#pragma unroll
                for (int e = 0; e < 8; e++) top = max(top, __float_as_uint(fabsf(x[m][e])));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float p2, inv;
            power_of(__uint_as_float(top), p2, inv);
#pragma unroll
            for (int e = 0; e < 2; e++) unit[nt][e] = __shfl_sync(0xffffffffu, p2 * scale, (2 * t + e) * 4);
#pragma unroll
            for (int m = 0; m < KC; m++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t w[P];
                    pieces_of<P>(x[m][2 * e] * inv, x[m][2 * e + 1] * inv, w);
#pragma unroll
                    for (int c = 0; c < P; c++) qf[nt][m][e >> 1][c][e & 1] = w[c];
                }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = row0 + nt * 8 + 2 * t + e;
            lim[nt][e] = r < rows ? at.past + r / group + 1 : 0;
        }
    }
    // whether the row of column e sees a slot of the tile's range
    const auto sees = [&](int nt, int e, int slot) {
        const int j = slot - at.past;
        bool ok = slot >= first && slot < lim[nt][e];
        if (tree && ok && j >= 0) ok = above[nt * 8 + 2 * t + e][j >> 5] >> (j & 31) & 1;
        return ok;
    };

    float o[VC][4][NT][4] = {}, m[NT][2], l[NT][2] = {};
#pragma unroll
    for (int nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -INFINITY;
    for (; turn < to; turn += WARPS) {
        const int slot = turn * TURN, next = turn + WARPS;
        int here[U];
        float s[U][NT][4] = {};
#pragma unroll
        for (int u = 0; u < U; u++) {
            here[u] = page[u];
#pragma unroll
            for (int c = P - 1; c >= 0; c--)  // (the small pieces first)
#pragma unroll
                for (int k = 0; k < KC; k++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++)
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
                            mma(H(), s[u][nt], word(kr[u][0][k], 2 * hf), word(kr[u][1][k], 2 * hf), word(kr[u][0][k], 2 * hf + 1),
                                word(kr[u][1][k], 2 * hf + 1), qf[nt][k][hf][c][0], qf[nt][k][hf][c][1]);
        }
        if (++it == 32 / U) {
            it = 0;
            look(next);
        }
        page_in(page);
        if (next < to) load_k(page, next * TURN);

        bool edge = slot < first || slot + TURN > rg.seen_by_all, dirty = false;
#pragma unroll
        for (int u = 0; u < U; u++) edge |= here[u] < 0;
        if (edge) {
            // values that no row sees count for nothing, whatever they are; of those that some see, what is infinite
            // or NaN comes in by itself below
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int key = slot + u * GROUP + 2 * t + (k & 1) + (k >> 1) * 8;
                    const bool none = key < first || key >= rg.end || here[u] < 0;
#pragma unroll
                    for (int c = 0; c < VC; c++) {
                        uint4& w = vr[u][c][k];
                        if (none) w = make_uint4(0, 0, 0, 0);
                        const uint4 f = make_uint4(finite(w.x, EXP), finite(w.y, EXP), finite(w.z, EXP), finite(w.w, EXP));
                        dirty |= f.x != w.x || f.y != w.y || f.z != w.z || f.w != w.w;
                        w = f;
                    }
                }
            dirty = __any_sync(0xffffffffu, dirty);
        }
        uint32_t pt[U][NT][2][P];
        float keep[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[u][nt][e] *= unit[nt][e & 1];
                    if (edge && (here[u] < 0 || !sees(nt, e & 1, slot + u * GROUP + g + (e >> 1) * 8))) s[u][nt][e] = -INFINITY;
                }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float top = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                for (int u = 1; u < U; u++) top = fmax3(top, s[u][nt][e], s[u][nt][2 + e]);
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                top = fmaxf(top, m[nt][e]);
                const float base = top == -INFINITY ? 0.f : top;
                keep[nt][e] = exp2_approx(m[nt][e] - base);
                m[nt][e] = top;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    s[u][nt][e] = exp2_approx(s[u][nt][e] - base + SHIFT);
                    s[u][nt][2 + e] = exp2_approx(s[u][nt][2 + e] - base + SHIFT);
                }
            }
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    uint32_t w[P];
                    if constexpr (RAW) {
                        __nv_bfloat162 x = __floats2bfloat162_rn(s[u][nt][hf * 2], s[u][nt][hf * 2 + 1]);
                        w[0] = *reinterpret_cast<uint32_t*>(&x);
                        s[u][nt][hf * 2] = __uint_as_float(w[0] << 16);
                        s[u][nt][hf * 2 + 1] = __uint_as_float(w[0] & 0xffff0000u);
                    } else {
                        pieces_of<P>(s[u][nt][hf * 2], s[u][nt][hf * 2 + 1], w);
                    }
#pragma unroll
                    for (int c = 0; c < P; c++) pt[u][nt][hf][c] = transpose8x8(w[c]);
                }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float sum = s[0][nt][e] + s[0][nt][2 + e];
#pragma unroll
                for (int u = 1; u < U; u++) sum += s[u][nt][e] + s[u][nt][2 + e];
                l[nt][e] = l[nt][e] * keep[nt][e] + sum;
            }
        }
#pragma unroll
        for (int c = 0; c < VC; c++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    // a turn's sums start from zero and are added rounded: the tensor cores truncate theirs
                    float sum[4] = {};
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const uint32_t w0 = word(vr[u][c][0], r), w1 = word(vr[u][c][1], r), w2 = word(vr[u][c][2], r), w3 = word(vr[u][c][3], r);
#pragma unroll
                        for (int k = P - 1; k >= 0; k--)
                            mma(H(), sum, __byte_perm(w0, w1, 0x5410), __byte_perm(w0, w1, 0x7632), __byte_perm(w2, w3, 0x5410),
                                __byte_perm(w2, w3, 0x7632), pt[u][nt][0][k], pt[u][nt][1][k]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) o[c][r][nt][e] = o[c][r][nt][e] * keep[nt][e & 1] + sum[e];
                }
        if (next < to) load_v(page, next * TURN);
        if (dirty) {
            // an infinity or a NaN ends in the sums of all that see it
#pragma unroll 1
            for (int key = max(slot, first); key < min(slot + TURN, rg.end); key++) {
                const int in = U > 1 && key - slot >= GROUP ? here[U - 1] : here[0];
                if (in < 0) continue;
                const uint16_t* src = vd + row_at(p.c, in, h, key) + g * 8;
#pragma unroll
                for (int c = 0; c < VC; c++) {
                    const uint4 w = load_cached(src + c * 64);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t x = word(w, r);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const uint16_t bits = e >> 1 ? x >> 16 : x & 0xffffu;
                            if ((bits & EXP) != EXP) continue;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
                                if (sees(nt, e & 1, key)) o[c][r][nt][e] += paged::up(*reinterpret_cast<const H*>(&bits));
                        }
                    }
                }
            }
            __syncwarp();
        }
    }

    // the warp's state: sums over the lanes; O in units of 2^-SHIFT, as l
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
#pragma unroll
            for (int c = 0; c < VC; c++)
#pragma unroll
                for (int k = 0; k < 4; k += 2)
                    *reinterpret_cast<float4*>(sm_o + (warp * R + r) * LDO + c * 64 + g * 8 + k * 2) =
                        make_float4(o[c][k][nt][e], o[c][k][nt][2 + e], o[c][k + 1][nt][e], o[c][k + 1][nt][2 + e]);
        }
    __syncthreads();
    if (clustered) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA of the cluster runs
    cg::cluster_group cluster = cg::this_cluster();
    // a thread has the same four columns of every row it takes
    constexpr int ROWS_AT_ONCE = 32 * WARPS / (D / 4);
    const int live = min(R, rows - row0), c4 = threadIdx.x % (D / 4) * 4, r0 = threadIdx.x / (D / 4), per = rows_of_rank(R, splits);
    T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + (size_t)h * group * D + c4;
    float* inbox = sm_o + WARPS * R * LDO;
    for (int r = r0; r < live; r += ROWS_AT_ONCE) {
        const Sum x = sum_of(WARPS, [&](int w) { return state[w][r]; },
                             [&](int w) { return *reinterpret_cast<const float4*>(sm_o + (w * R + r) * LDO + c4); });
        if (splits == 1) {
            const int row = row0 + r, i = row / group;
            store4(out + i * p.out.ts + (size_t)(row - i * group) * D, x.o, x.l == 0.f ? 0.f : 1.f / x.l, vec & 2);
        } else {
            const int k = r / splits;
            float* to = clustered ? cluster.map_shared_rank(inbox, r - k * splits) + (split * per + k) * LDO
                                  : p.ws + z + (((size_t)bh * gridDim.x + blockIdx.x) * R + r) * LDO;
            *reinterpret_cast<float4*>(to + 4 + c4) = x.o;
            if (c4 == 0) *reinterpret_cast<float2*>(to) = make_float2(x.m, x.l);
        }
    }
    if (!clustered) return;
    __syncwarp();
    cluster.sync();
    for (int k = r0; k * splits + split < live; k += ROWS_AT_ONCE) {
        const Sum x = sum_of(splits, [&](int s) { return *reinterpret_cast<const float2*>(inbox + (s * per + k) * LDO); },
                             [&](int s) { return *reinterpret_cast<const float4*>(inbox + (s * per + k) * LDO + 4 + c4); });
        const int row = row0 + k * splits + split, i = row / group;
        store4(out + i * p.out.ts + (size_t)(row - i * group) * D, x.o, x.l == 0.f ? 0.f : 1.f / x.l, vec & 2);
    }
}

// The splits' partials to the output, G * D / 4 threads to a row: each of the G groups sums every G-th split, and the
// groups' sums meet in shared memory.
template <typename T, int D, int G>
__global__ void __launch_bounds__(256) paged_combine_kernel(PagedAttn p, int splits, int R, int vec) {
    chain_release();
    const int z = chain_wait();
    constexpr int TO_ROW = G * D / 4, ROWS = 256 / TO_ROW;
    static_assert(ROWS >= 1 && (G == 1 || ROWS == 1), "whole rows, or one to the CTA");
    __shared__ int parent[MOST_TREE];
    __shared__ float top_of[G];
    __shared__ float sum_of_group[G];
    __shared__ float4 sums[G][D / 4];
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv, group = p.n_head / p.c.n_head_kv;
    const int row = blockIdx.x * ROWS + threadIdx.x / TO_ROW, sub = threadIdx.x % TO_ROW / (D / 4), c = threadIdx.x % (D / 4);
    const Place at = place_of(p.s, b, p.c.room, nullptr);
    if (p.s.first && __ldcg(p.s.first + b + z) < 0) return;
    if (p.tree.parent && !read_tree(p.tree, b, at.count, z, parent)) return;
    const bool live = row < at.count * group;
    if (G > 1 ? !live : blockIdx.x * ROWS >= at.count * group) return;
    const int tiles = (p.s.n * group + R - 1) / R;
    const size_t step = (size_t)R * (D + 4);
    const float* ws = p.ws + z + ((size_t)bh * tiles + row / R) * splits * step + (row % R) * (D + 4);
    // in batches whose loads are all on their way before the first is used
    constexpr int BATCH = 8;
    float mx = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (live)
#pragma unroll 1
        for (int s0 = sub; s0 < splits; s0 += BATCH * G) {
            float2 ml[BATCH];
            float4 o[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const float* at = ws + min(s0 + k * G, splits - 1) * step;
                ml[k] = __ldcg(reinterpret_cast<const float2*>(at));
                o[k] = __ldcg(reinterpret_cast<const float4*>(at + 4) + c);
            }
            float top = mx;
#pragma unroll
            for (int k = 0; k < BATCH; k++)
                if (s0 + k * G < splits) top = fmaxf(top, ml[k].x);
            const float base = top == -INFINITY ? 0.f : top, keep = exp2_approx(mx - base);
            sum *= keep;
            acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                if (s0 + k * G >= splits) continue;
                const float f = exp2_approx(ml[k].x - base);
                sum += ml[k].y * f;
                add4(acc, f, o[k]);
            }
            mx = top;
        }
    if (G > 1) {
        if (c == 0) {
            top_of[sub] = mx;
            sum_of_group[sub] = sum;
        }
        sums[sub][c] = acc;
        __syncthreads();
        if (sub > 0) return;
        const Sum x = sum_of(G, [&](int w) { return make_float2(top_of[w], sum_of_group[w]); }, [&](int w) { return sums[w][c]; });
        sum = x.l;
        acc = x.o;
    }
    if (!live) return;
    const int i = row / group;
    T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + i * p.out.ts +
             (size_t)(h * group + row - i * group) * D + c * 4;
    store4(out, acc, sum == 0.f ? 0.f : 1.f / sum, vec & 2);
}

struct Plan {
    int tile_rows, tiles;  // query rows of a tile, tiles of a (sequence, kv head)
    int splits;            // cuts of the keys
    int warps;             // of a CTA; 0: the tcgen05 kernel's
    size_t ws;             // floats of workspace, for this and shorter caches
    float us;              // about how long it takes, for the choice between the kernels
    int in_place() const { return warps ? MAX_CLUSTER : 1; }  // cuts that need no workspace
};

// Shared memory of a CTA: its warps' O, and a cluster's inbox.
int smem_of(int d, int tile_rows, int warps, int splits) {
    const int inbox = splits > 1 && splits <= MAX_CLUSTER ? splits * rows_of_rank(tile_rows, splits) : 0;
    return (warps * tile_rows + inbox) * (d + 4) * (int)sizeof(float);
}

// The most of it: splits * rows_of_rank is below R + splits.
constexpr int most_smem(int d, int tile_rows, int warps) { return (warps * tile_rows + tile_rows + MAX_CLUSTER) * (d + 4) * (int)sizeof(float); }

// Clusters of n CTAs that run at once on the current device: a cluster lives in one GPC, and the GPCs have different
// numbers of SMs. Asked once for each device.
template <int NT, int WARPS>
int ask_clusters(int n) {
    const auto kern = paged_split_kernel<float, 128, NT, 2, WARPS>;  // the others need no more than it
    static std::atomic<uint64_t> done{0};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n);
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = smem_of(128, 8 * NT, WARPS, n);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)n;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int count = 0;
    if (allow_smem(done, (const void*)kern, most_smem(128, 8 * NT, WARPS), true) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&count, kern, &cfg) != cudaSuccess)
        (void)cudaGetLastError();
    return count;
}
int clusters_at_once(int tile_rows, bool big, int n) {
    static std::atomic<int> known[64][2][2][MAX_CLUSTER + 1];
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 1;
    std::atomic<int>& at = known[dev & 63][tile_rows == 8][big][n];
    int count = at.load(std::memory_order_relaxed);
    if (count == 0) {
        count = tile_rows == 8 ? big ? ask_clusters<1, big_warps(8)>(n) : ask_clusters<1, SMALL>(n)
                               : big ? ask_clusters<2, big_warps(16)>(n) : ask_clusters<2, SMALL>(n);
        at.store(count = std::max(1, count), std::memory_order_relaxed);
    }
    return count;
}

// Slots that the longest sequence can have at the call's end.
int keys_of(const Paged& c, const Seqs& s) { return (int)std::min<long long>((long long)s.n_past + s.n, c.room); }

// How often SMs are filled: the last time counts half of itself and half of a whole one.
float waves_of(long long ctas, long long places) {
    const float w = (float)ctas / places, whole = std::floor(w);
    return w <= 1.f ? 1.f : whole == w ? w : whole + 0.5f + 0.5f * (w - whole);
}

Plan plan_split(const Paged& c, const Seqs& s, int rows, bool raw, int sm_count) {
    Plan p{};
    p.tile_rows = rows <= 8 ? 8 : 16;  // one or two 8-wide N tiles
    p.tiles = (rows + p.tile_rows - 1) / p.tile_rows;
    const long long ctas = (long long)s.n_batch * c.n_head_kv * p.tiles;
    const int key_turns = (keys_of(c, s) + GROUP * 128 / c.d - 1) / (GROUP * 128 / c.d);
    const float turn = c.d == 64 ? raw ? 1.5f : 1.8f : raw ? 1.5f : 2.f;  // us of a turn, of which a warp has some
    for (const bool big : {true, false}) {
        const int warps = big ? big_warps(p.tile_rows) : SMALL;
        const long long places = (long long)sm_count * (big_warps(p.tile_rows) / warps);
        const int useful = (key_turns + warps - 1) / warps;
        const auto turns = [&](int n) { return (useful + n - 1) / n; };  // that follow each other in a warp
        const int most = (int)std::min<long long>(useful, std::max<long long>(1, places / ctas));
        // a cluster that waits for a place doubles the time
        int splits = std::min(MAX_CLUSTER, most);
        while (splits > 1 && ctas > clusters_at_once(p.tile_rows, big, splits)) splits--;
        // more cuts than that where they save more turns than the second kernel costs
        const int in_cluster = splits;
        if (most > MAX_CLUSTER && turns(most) + 2 < turns(splits)) splits = most;
        // that takes more than 3 turns in the cluster, with these keys or fewer
        if (most > MAX_CLUSTER && useful > 3 * in_cluster) p.ws = std::max(p.ws, (size_t)ctas * most * p.tile_rows * (c.d + 4));
        // merges: of a cluster the longer the more CTAs it has (one sequence of 2256 tokens, 150 rows, in 7 big CTAs 14.1 us,
        // in 14 small ones 18.6), of a big CTA's warps
        const float merge = splits > MAX_CLUSTER ? 4.f : splits > 1 ? 2.f + 0.15f * splits : 0.f;
        const float us = waves_of(ctas * splits, places) * (5.f + turn * turns(splits)) + merge + (big ? 0.5f : 0.f);
        if (big || us < p.us) {
            p.us = us;
            p.splits = splits;
            p.warps = warps;
        }
    }
    return p;
}

// The tcgen05 kernel: keys are cut while SMs stay empty, two tiles of keys to a cut at least. Where sequences have lengths
// of their own, one cut more, so that all SMs have work and the longest sequence holds up less, if the cuts still take
// five times a CTA's start and end: 64 sequences of up to 8001 tokens, 96 rows, d 128, bf16: 141 us in one cut, 105
// in two where lengths lie between 0 and that, 141 and 135 from half of it on, 144 and 166 if all are alike; of up to
// 2000 (not cut): 42 and 49, 45 and 58, 46 and 65.
Plan plan_chunk(const Paged& c, const Seqs& s, int rows, bool raw, int sm_count) {
    Plan p{};
    p.warps = 0;
    p.tile_rows = PAGED_CHUNK_ROWS;
    p.tiles = (rows + PAGED_CHUNK_ROWS - 1) / PAGED_CHUNK_ROWS;
    const long long ctas = (long long)s.n_batch * c.n_head_kv * p.tiles;
    const int key_tiles = (keys_of(c, s) + PAGED_CHUNK_KEYS - 1) / PAGED_CHUNK_KEYS;
    const bool two = rows > PAGED_CHUNK_ROWS / 2;
    const float start = c.d == 64 ? raw ? 9.f : 11.f : raw ? 11.f : 16.f;
    const float turn = c.d == 64 ? two ? raw ? 1.9f : 2.5f : raw ? 1.1f : 1.4f : two ? raw ? 2.5f : 5.4f : raw ? 1.9f : 2.5f;
    p.splits = (int)std::min<long long>(std::max<long long>(1, sm_count / ctas), std::max(1, key_tiles / 2));
    const bool more = ctas * p.splits < sm_count && turn * (key_tiles / (p.splits + 1)) >= 5.f * start;
    const int most = p.splits + (more ? 1 : 0);  // the workspace is asked for with lengths of their own or without
    if (s.past && more) p.splits++;
    if (most > 1) p.ws = (size_t)ctas * most * p.tile_rows * (c.d + 4);
    p.us = waves_of(ctas * p.splits, sm_count) * (start + turn * ((key_tiles + p.splits - 1) / p.splits)) + (p.splits > 1 ? 2.f : 0.f);
    return p;
}

// The tcgen05 kernel has four times the other one's rate and reads the keys once for 256 rows, not 16, but a CTA of it
// takes 9 to 18 us to start and end. Above 16 rows the shorter estimate runs, its constants read off both kernels'
// times for 24 to 256 rows a head, 1 to 64 sequences of 200 to 8000 tokens, both d, bf16 and f32: 16 sequences of 2000
// tokens, d 128, bf16: 24 rows 16.4 us against this one's 20.0, 48 rows 26.4 against 18.4, 128 rows 45.5 against 20.9; one
// of 2000 tokens: 128 rows 10.4 against 14.9. Over 288 calls (18 to 258 rows, 1 to 64 sequences of
// 200 to 8000 tokens, both d and types) the one that runs takes 1.00 of the better one's time in the middle, 1.02 at the
// 95th of a hundred, 1.33 at the most (4 sequences of 2000 tokens, 96 rows, d 64, bf16: 14.8 us for 11.2). Up to 16
// rows, where the other kernel reads the keys once too, it was never the slower one by more than 5 %.
Plan plan_for(const Paged& c, const Seqs& s, int n_head, bool raw, int sm_count) {
    const int rows = s.n * (n_head / c.n_head_kv);
    Plan split = plan_split(c, s, rows, raw, sm_count);
    if (rows <= 16) return split;
    Plan chunk = plan_chunk(c, s, rows, raw, sm_count);
    split.ws = chunk.ws = std::max(split.ws, chunk.ws);
    return split.us < chunk.us ? split : chunk;
}

template <typename T, int D, int NT, int P, int WARPS>
int split_launch(const PagedAttn& p, const Plan& plan, int vec, cudaStream_t st) {
    const float scale = (float)(1.0 / sqrt((double)D)) * kLog2e;
    const int clustered = plan.splits > 1 && plan.splits <= MAX_CLUSTER;
    const auto kern = paged_split_kernel<T, D, NT, P, WARPS>;
    static std::atomic<uint64_t> done{0};
    if (allow_smem(done, (const void*)kern, most_smem(D, 8 * NT, WARPS), true) != cudaSuccess) return -1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(plan.tiles * plan.splits), (unsigned)(p.s.n_batch * p.c.n_head_kv));
    cfg.blockDim = dim3(32 * WARPS);
    cfg.dynamicSmemBytes = smem_of(D, 8 * NT, WARPS, plan.splits);
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
int split_of(const PagedAttn& p, const Plan& plan, int vec, cudaStream_t st) {
    return plan.warps == SMALL ? split_launch<T, D, NT, P, SMALL>(p, plan, vec, st)
                               : split_launch<T, D, NT, P, big_warps(8 * NT)>(p, plan, vec, st);
}

template <typename T, int D>
int combine(const PagedAttn& p, const Plan& plan, int vec, int sm_count, cudaStream_t st) {
    const int rows = p.s.n * (p.n_head / p.c.n_head_kv);
    const unsigned segs = (unsigned)(p.s.n_batch * p.c.n_head_kv);
    constexpr int G = 1024 / D;
    cudaError_t e;
    if ((long long)rows * segs > 8 * sm_count)  // more than a CTA to a row fits at once
        e = launch_chained(paged_combine_kernel<T, D, 1>, dim3((unsigned)(rows + G - 1) / G, segs), dim3(256), st, p, plan.splits, plan.tile_rows, vec);
    else
        e = launch_chained(paged_combine_kernel<T, D, G>, dim3((unsigned)rows, segs), dim3(256), st, p, plan.splits, plan.tile_rows, vec);
    return e == cudaSuccess ? 0 : -1;
}

template <typename T, int D, int P>
int attn(const PagedAttn& p, int sm_count, cudaStream_t st) {
    const Plan plan = plan_for(p.c, p.s, p.n_head, sizeof(T) == 2, sm_count);
    const int vec = (wide(p.q, sizeof(T), 16) ? 1 : 0) | (wide(p.out, sizeof(T), 4 * sizeof(T)) ? 2 : 0);
    int rc = plan.warps == 0       ? paged_chunk_launch(p, sizeof(T) == 2 ? TYPE_BF16 : TYPE_F32, P, plan.splits, st)
             : plan.tile_rows == 8 ? split_of<T, D, 1, P>(p, plan, vec, st)
                                   : split_of<T, D, 2, P>(p, plan, vec, st);
    if (rc == 0 && plan.splits > plan.in_place()) rc = combine<T, D>(p, plan, vec, sm_count, st);
    return rc;
}

}  // namespace

size_t paged_attn_workspace_bytes(const Paged& c, const Seqs& s, int n_head, int sm_count) {
    if (s.n_batch == 0 || s.n == 0) return 0;
    return plan_for(c, s, n_head, c.type == TYPE_BF16, sm_count).ws * sizeof(float);
}

int paged_attn_launch(const PagedAttn& p, int type, int pieces, int sm_count, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    if (type == TYPE_BF16) return p.c.d == 64 ? attn<__nv_bfloat16, 64, 1>(p, sm_count, st) : attn<__nv_bfloat16, 128, 1>(p, sm_count, st);
    if (pieces == 1) return p.c.d == 64 ? attn<float, 64, 1>(p, sm_count, st) : attn<float, 128, 1>(p, sm_count, st);
    return p.c.d == 64 ? attn<float, 64, 2>(p, sm_count, st) : attn<float, 128, 2>(p, sm_count, st);
}

}  // namespace zwg
