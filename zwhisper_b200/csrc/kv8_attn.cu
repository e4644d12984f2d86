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
// A warp takes whole blocks; its softmax state is merged with the other warps' in shared memory and
// the splits' partials (m, l, O) by kv8_combine_kernel.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "seqs.cuh"

namespace zwg {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kUnit = 32768.f;  // P's f16 pieces hold 2^15 p: small probabilities stay normal

ZWG_DEV float up(float x) { return x; }
ZWG_DEV float up(__nv_bfloat16 x) { return __bfloat162float(x); }
ZWG_DEV void down(float x, float& y) { y = x; }
ZWG_DEV void down(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }

ZWG_DEV uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Four int8 of a word -> two f16 pairs, exactly: 0x6400 | (x + 128) is 1024 + 128 + x.
ZWG_DEV void ints_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2(__half_raw{0x6480}, __half_raw{0x6480});
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    lo = h2u(__hsub2(*reinterpret_cast<__half2*>(&a), off));
    hi = h2u(__hsub2(*reinterpret_cast<__half2*>(&b), off));
}

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

// x as f16 pieces: the nearest f16 and, with two, the nearest f16 of what is left.
template <int P>
ZWG_DEV void pieces_of(float x, float y, uint32_t (&w)[P]) {
    const __half2 h = __floats2half2_rn(x, y);
    w[0] = h2u(h);
    if (P == 2) {
        const float2 f = __half22float2(h);
        w[P - 1] = h2u(__floats2half2_rn(x - f.x, y - f.y));
    }
}

// The power of two of |x|'s exponent and its inverse; 1 for zero, tiny, infinite and NaN.
ZWG_DEV void power_of(float x, float& p, float& inv) {
    const uint32_t e = __float_as_uint(x) & 0x7f800000u;
    const bool fine = e > 0x01000000u && e < 0x7e000000u;
    p = fine ? __uint_as_float(e) : 1.f;
    inv = fine ? __uint_as_float(0x7f000000u - e) : 1.f;
}

struct Plan {
    int tiles;   // tiles of query rows of a (sequence, kv head)
    int splits;  // cuts of the keys
};

constexpr int WARPS = 4;

// Rows of a tile: one or two 8-wide N tiles.
int tile_rows(int rows) { return rows <= 8 ? 8 : 16; }

Plan plan_for(const Kv8& c, const Seqs& s, int n_head, int sm_count) {
    const int rows = s.n * (n_head / c.n_head_kv);
    Plan p;
    p.tiles = (rows + tile_rows(rows) - 1) / tile_rows(rows);
    const long long ctas = (long long)s.n_batch * c.n_head_kv * p.tiles;
    const int blocks = (s.n_past + s.n + KV8_BLOCK - 1) / KV8_BLOCK;
    // four CTAs an SM, each with at least a block for every warp
    const long long want = std::max<long long>(1, 4ll * sm_count / ctas);
    p.splits = (int)std::min<long long>(want, std::max(1, blocks / WARPS));
    return p;
}

template <typename T, int D, int NT, int P>
__global__ void __launch_bounds__(32 * WARPS) kv8_split_kernel(Kv8Attn p, int splits, float scale) {
    chain_release();
    const int z = chain_wait();
    constexpr int R = 8 * NT, CH = D / 64, LDO = D + 4;
    extern __shared__ float sm_o[];  // [WARPS][R][LDO], then m and l [WARPS][R]
    float* sm_m = sm_o + WARPS * R * LDO;
    float* sm_l = sm_m + WARPS * R;
    const int split = blockIdx.x % splits, tile = blockIdx.x / splits;
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh % p.c.n_head_kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = p.n_head / p.c.n_head_kv;
    const Place at = place_of(p.s, b, p.c.blocks * KV8_BLOCK, threadIdx.x == 0 && blockIdx.x == 0 && h == 0 ? p.err : nullptr);
    const int rows = at.count * group, row0 = tile * R;
    if (row0 >= rows) return;
    int first = p.s.first ? __ldcg(p.s.first + b + z) : 0;
    if (first < 0) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    const int last_row = min(rows, row0 + R) - 1;
    const int seen = at.past + last_row / group + 1;  // keys the tile's last row sees
    const int blk_lo = first / KV8_BLOCK, blk_hi = (seen + KV8_BLOCK - 1) / KV8_BLOCK;
    const int n_blk = max(0, blk_hi - blk_lo);
    const int from = blk_lo + (int)((long long)n_blk * split / splits);
    const int to = blk_lo + (int)((long long)n_blk * (split + 1) / splits);

    // queries: the B operand, lane (g, t) holds row g's 16 consecutive elements of each 64
    uint32_t qf[NT][CH][4][P][2];
    float unit[NT][2];  // of the columns 2t, 2t + 1: 2^e * log2(e) / sqrt(d)
    int lim[NT][2];     // keys below it are seen
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int row = row0 + nt * 8 + g;
        float x[CH][16];
        float top = 0.f;
        const bool live = row < rows;
        const T* q = static_cast<const T*>(p.q.data) + z + b * p.q.bs +
                     (live ? (row / group) * p.q.ts + (size_t)(h * group + row % group) * D : 0);
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                x[i][e] = live ? up(q[i * 64 + t * 16 + e]) : 0.f;
                top = fmaxf(top, fabsf(x[i][e]));
            }
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
    float ref = 0.f;  // the largest vs so far
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            m[nt][e] = -INFINITY;
            l[nt][e] = 0.f;
        }

    const size_t head = (size_t)bh * p.c.blocks;
    for (int blk = from + warp; blk < to; blk += WARPS) {
        const int8_t* kb = p.c.k + (head + blk) * (KV8_BLOCK * D) + z;
        const int8_t* vb = p.c.v + (head + blk) * (KV8_BLOCK * D) + z;
        float ks = __ldcg(p.c.k_scale + head + blk + z), vs = __ldcg(p.c.v_scale + head + blk + z);
        if (vs != vs) {  // values that read as NaN: through the scores, which a mask covers
            ks = vs;
            vs = 0.f;
        }
        // S^T: rows are tokens, logical row (mt, hf, r) is token (r / 2) * 8 + mt * 4 + hf * 2 + r % 2
        float s[2][NT][4] = {};
        uint4 kw[2][2][CH];
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
#pragma unroll
                for (int i = 0; i < CH; i++)
                    kw[mt][hf][i] = __ldcg(reinterpret_cast<const uint4*>(
                        kb + ((g >> 1) * 8 + mt * 4 + hf * 2 + (g & 1)) * D + i * 64 + t * 16));
        uint2 vw[D / 16][2];
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int hf = 0; hf < 2; hf++)
                vw[j][hf] = __ldcg(reinterpret_cast<const uint2*>(vb + (j * 16 + hf * 8 + g) * KV8_BLOCK + t * 8));
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
                            mma(s[mt][nt], a0, a1, a2, a3, qf[nt][i][st][c][0], qf[nt][i][st][c][1]);
                }
        // softmax over the block, for the columns 2t and 2t + 1
        const float top = fmaxf(ref, vs);
        const float ratio = top > 0.f ? vs / top : 0.f;
        const float shrink = top > 0.f ? ref / top : 1.f;
        ref = top;
        uint32_t pt[2][2][NT][P];
        const int key0 = blk * KV8_BLOCK;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float keep[2];
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
                        x = key < lim[nt][e] && key >= first ? x * f : -INFINITY;
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
                keep[e] = alpha * shrink;
            }
#pragma unroll
            for (int j = 0; j < D / 16; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[j][nt][e] *= keep[e & 1];
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
        for (int j = 0; j < D / 16; j++)
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                uint32_t a0, a1, a2, a3;
                ints_to_f16(mt ? vw[j][0].y : vw[j][0].x, a0, a2);
                ints_to_f16(mt ? vw[j][1].y : vw[j][1].x, a1, a3);
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < P; c++) mma(o[j][nt], a0, a1, a2, a3, pt[mt][0][nt][c], pt[mt][1][nt][c]);
            }
    }

    // the warp's state: sums over the lanes, O in its true units
    const float units = ref * (1.f / kUnit);
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            float sum = l[nt][e];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const int r = nt * 8 + 2 * t + e;
            if (g == 0) {
                sm_m[warp * R + r] = m[nt][e];
                sm_l[warp * R + r] = sum;
            }
            float* row = sm_o + (warp * R + r) * LDO;
#pragma unroll
            for (int j = 0; j < D / 16; j++) {
                row[j * 16 + g] = o[j][nt][e] * units;
                row[j * 16 + 8 + g] = o[j][nt][2 + e] * units;
            }
        }
    __syncthreads();
    for (int idx = threadIdx.x; idx < R * D; idx += 32 * WARPS) {
        const int r = idx / D, c = idx % D, row = row0 + r;
        if (row >= rows) break;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; w++) mx = fmaxf(mx, sm_m[w * R + r]);
        const float base = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float f = exp2_approx(sm_m[w * R + r] - base);
            sum += sm_l[w * R + r] * f;
            acc += sm_o[(w * R + r) * LDO + c] * f;
        }
        if (splits == 1) {
            T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + (row / group) * p.out.ts +
                     (size_t)(h * group + row % group) * D + c;
            down(sum == 0.f ? 0.f : acc / sum, *out);
        } else {
            float* ws = p.ws + z + (((size_t)bh * gridDim.x + blockIdx.x) * R + r) * (D + 2);
            ws[2 + c] = acc;
            if (c == 0) {
                ws[0] = mx;
                ws[1] = sum;
            }
        }
    }
}

// One CTA of D threads per query row: the splits' partials to the output.
template <typename T, int D>
__global__ void __launch_bounds__(D) kv8_combine_kernel(Kv8Attn p, int splits, int R) {
    chain_release();
    const int z = chain_wait();
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh % p.c.n_head_kv, row = blockIdx.x, c = threadIdx.x;
    const int group = p.n_head / p.c.n_head_kv;
    const Place at = place_of(p.s, b, p.c.blocks * KV8_BLOCK, nullptr);
    if (row >= at.count * group || (p.s.first && __ldcg(p.s.first + b + z) < 0)) return;
    const int tiles = (p.s.n * group + R - 1) / R;
    const float* ws = p.ws + z + (((size_t)bh * tiles + row / R) * splits * R + row % R) * (D + 2);
    const size_t step = (size_t)R * (D + 2);
    float mx = -INFINITY;
    for (int s = 0; s < splits; s++) mx = fmaxf(mx, __ldcg(ws + s * step));
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f, acc = 0.f;
    for (int s = 0; s < splits; s++) {
        const float f = exp2_approx(__ldcg(ws + s * step) - base);
        sum += __ldcg(ws + s * step + 1) * f;
        acc += __ldcg(ws + s * step + 2 + c) * f;
    }
    T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + (row / group) * p.out.ts +
             (size_t)(h * group + row % group) * D + c;
    down(sum == 0.f ? 0.f : acc / sum, *out);
}

template <typename T, int D, int NT, int P>
int split_launch(const Kv8Attn& p, const Plan& plan, cudaStream_t st) {
    constexpr size_t smem = WARPS * 8 * NT * (D + 4 + 2) * sizeof(float);
    static_assert(smem <= 48 * 1024, "the merge fits without opting in");
    const float scale = (float)(1.0 / sqrt((double)D)) * kLog2e;
    const int rows = p.s.n * (p.n_head / p.c.n_head_kv);
    const unsigned segs = (unsigned)(p.s.n_batch * p.c.n_head_kv);
    cudaError_t e = launch_chained_smem(kv8_split_kernel<T, D, NT, P>, dim3((unsigned)(plan.tiles * plan.splits), segs),
                                        dim3(32 * WARPS), smem, st, p, plan.splits, scale);
    if (e == cudaSuccess && plan.splits > 1)
        e = launch_chained(kv8_combine_kernel<T, D>, dim3((unsigned)rows, segs), dim3(D), st, p, plan.splits, 8 * NT);
    return e == cudaSuccess ? 0 : -1;
}

template <typename T, int D>
int attn(const Kv8Attn& p, int pieces, int sm_count, cudaStream_t st) {
    const Plan plan = plan_for(p.c, p.s, p.n_head, sm_count);
    const bool small = p.s.n * (p.n_head / p.c.n_head_kv) <= 8;
    if (pieces == 1) return small ? split_launch<T, D, 1, 1>(p, plan, st) : split_launch<T, D, 2, 1>(p, plan, st);
    return small ? split_launch<T, D, 1, 2>(p, plan, st) : split_launch<T, D, 2, 2>(p, plan, st);
}

}  // namespace

size_t kv8_attn_workspace_bytes(const Kv8& c, const Seqs& s, int n_head, int sm_count) {
    if (s.n_batch == 0 || s.n == 0) return 0;
    const Plan p = plan_for(c, s, n_head, sm_count);
    const int rows = s.n * (n_head / c.n_head_kv);
    return p.splits == 1 ? 0
                         : (size_t)s.n_batch * c.n_head_kv * p.tiles * p.splits * tile_rows(rows) * (c.d + 2) * sizeof(float);
}

int kv8_attn_launch(const Kv8Attn& p, int type, int pieces, int sm_count, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    if (type == TYPE_BF16)
        return p.c.d == 64 ? attn<__nv_bfloat16, 64>(p, 1, sm_count, st) : attn<__nv_bfloat16, 128>(p, 1, sm_count, st);
    return p.c.d == 64 ? attn<float, 64>(p, pieces, sm_count, st) : attn<float, 128>(p, pieces, sm_count, st);
}

}  // namespace zwg
