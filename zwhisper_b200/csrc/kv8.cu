// The cache in 8 bits (zwg_kv8): appending to it and reading it back.
//
//   scale = max |x| / 127 over a block's 32 x d values of one head,  q = rint(127 x / max |x|)
//
// kv8_append_kernel: a CTA of 512 threads takes one block that the call touches, keys in its
// first 256 threads and values in the rest. The block's rows (new ones from the caller, rotated
// on the way; older ones from the open rows, or from the int8 values where the block is not the
// open one) meet in shared memory as f32, one pass takes their largest magnitude, the next one
// writes the int8 values. The first and the last block a call touches share the open rows, the
// first reading what the last one replaces, so one CTA takes both, one after the other.
// Bound by memory for a chunk of a prompt (f32 in, a quarter of it out), by the latency of one
// CTA's chain of loads and barriers for a step.
//
// Rounding: the rounded quotient is found from 127 x * (1 / max |x|) in f32 unless that is
// within 1e-3 of the border between two integers; there the f64 quotient of the exact product
// 127 x decides, which is exact at a border (the operands have 31 and 24 bits). So the values
// are the correctly rounded ones, whatever the order of operations elsewhere.
#include <cuda_bf16.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "seqs.cuh"

namespace zwg {
namespace {

constexpr int HALF = 256;  // threads for keys, and as many for values

ZWG_DEV float up(float x) { return x; }
ZWG_DEV float up(__nv_bfloat16 x) { return __bfloat162float(x); }

ZWG_DEV int round127(float x, float inv, float top) {
    const float y = __fmul_rn(x, inv);
    const float r = rintf(y);
    if (fabsf(fabsf(y - r) - 0.5f) < 1e-3f || !(fabsf(y) < 200.f)) {
        // the products and the quotient in f64; a largest magnitude too small for an f32 1 / x comes here too
        return (int)rint(__ddiv_rn(127.0 * (double)x, (double)top));
    }
    return (int)r;
}

ZWG_DEV uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)(d & 255) << 24;
}

template <typename T, int D>
__global__ void __launch_bounds__(2 * HALF) kv8_append_kernel(Kv8Append p) {
    chain_release();
    const int z = chain_wait();
    constexpr int LD = D + 1;  // odd: neither rows nor columns of the staging meet in a bank
    extern __shared__ float stage[];  // [2][32][LD]
    __shared__ uint32_t top_of[2][HALF / 32];
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh % p.c.n_head_kv;
    const int side = threadIdx.x / HALF, tid = threadIdx.x % HALF, lane = tid & 31, warp = tid >> 5;
    Place at = place_of(p.s, b, p.c.blocks * KV8_BLOCK, threadIdx.x == 0 && blockIdx.x == 0 && h == 0 ? p.err : nullptr);
    if (p.rope.cos && at.past + at.count > p.rope.n_ctx) {
        if (threadIdx.x == 0 && blockIdx.x == 0 && h == 0) set_error(p.err, kErrBounds);
        at.count = 0;
    }
    if (at.count == 0) return;
    const int end = at.past + at.count, b0 = at.past / KV8_BLOCK, b1 = (end - 1) / KV8_BLOCK;
    if ((int)blockIdx.x > 0 && b0 + (int)blockIdx.x >= b1) return;  // CTA 0 takes b0 and b1
    const bool is_k = side == 0;
    float* tile = stage + side * (KV8_BLOCK * LD);
    float* open = (is_k ? p.c.k_open : p.c.v_open) + (size_t)bh * KV8_BLOCK * D + z;
    const T* src = static_cast<const T*>(is_k ? p.k.data : p.v.data) + z;
    const size_t bs = is_k ? p.k.bs : p.v.bs, ts = is_k ? p.k.ts : p.v.ts;
    const size_t hs = is_k ? p.k_hs : p.v_hs, es = is_k ? p.k_es : 1;
    src += b * bs + h * hs;
    const int opened = __ldcg(p.c.open_block + bh + z);
    for (int blk = b0 + blockIdx.x;; blk = b1) {
        const int lo = blk * KV8_BLOCK, held = max(0, at.past - lo), live = min(KV8_BLOCK, end - lo);
        const size_t at_blk = (size_t)bh * p.c.blocks + blk;
        int8_t* ints = (is_k ? p.c.k : p.c.v) + at_blk * (KV8_BLOCK * D) + z;
        float* scale = (is_k ? p.c.k_scale : p.c.v_scale) + at_blk + z;
        // rows of the block: [0, held) the cache's, [held, live) new, the others zero
        const float old_scale = held && opened != blk ? __ldcg(scale) : 0.f;
        if (es == 1) {
            for (int e = tid; e < KV8_BLOCK * D; e += HALF) {
                const int r = e / D, c = e % D;
                float x = 0.f;
                if (r < held) {
                    x = opened == blk ? __ldcg(open + e)
                                      : (float)ints[is_k ? e : c * KV8_BLOCK + r] * old_scale;
                } else if (r < live) {
                    x = up(src[(size_t)(lo + r - at.past) * ts + c]);
                }
                tile[r * LD + c] = x;
            }
        } else {  // transposed keys: neighbouring tokens are neighbours in memory
            for (int e = tid; e < KV8_BLOCK * D; e += HALF) {
                const int c = e / KV8_BLOCK, r = e % KV8_BLOCK;
                float x = 0.f;
                if (r < held) {
                    x = opened == blk ? __ldcg(open + r * D + c)
                                      : (float)ints[is_k ? r * D + c : e] * old_scale;
                } else if (r < live) {
                    x = up(src[(size_t)(lo + r - at.past) * ts + c * es]);
                }
                tile[r * LD + c] = x;
            }
        }
        __syncthreads();
        if (is_k && p.rope.cos) {
            const int half = p.rope.rot / 2;
            for (int e = tid; e < (live - held) * half; e += HALF) {
                const int r = held + e / half, i = e % half;
                const size_t row = (size_t)(lo + r) * half + i;
                const float c = p.rope.cos[row], s = p.rope.sin[row];
                float* x = tile + r * LD + (p.rope.interleaved ? 2 * i : i);
                float* y = p.rope.interleaved ? x + 1 : x + half;
                const float a = *x, bb = *y;
                *x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(bb, s));
                *y = __fadd_rn(__fmul_rn(a, s), __fmul_rn(bb, c));
            }
        }
        if (p.rope.cos) __syncthreads();
        // |x|'s bit pattern orders like the value, with infinities and NaN above all others
        uint32_t top = 0;
        for (int e = tid; e < KV8_BLOCK * D; e += HALF) {
            const int r = e / D, c = e % D;
            const float x = tile[r * LD + c];
            top = max(top, __float_as_uint(fabsf(x)));
            if (blk == b1 && (r >= held || opened != blk)) __stcg(open + e, x);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) top_of[side][warp] = top;
        __syncthreads();
        top = top_of[side][0];
#pragma unroll
        for (int w = 1; w < HALF / 32; w++) top = max(top, top_of[side][w]);
        const float big = __uint_as_float(top);
        const bool finite = top < 0x7f800000u;
        const float inv = top && finite ? __fdiv_rn(127.f, big) : 0.f;
        // 16 values a thread: a piece of a key's row, or of a value column's 32 tokens
        constexpr int PIECES = KV8_BLOCK * D / 16;
        for (int e = tid; e < PIECES; e += HALF) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                int q[4];
#pragma unroll
                for (int l = 0; l < 4; l++) {
                    const int o = j * 4 + l;
                    const float x = is_k ? tile[(e * 16 / D) * LD + e * 16 % D + o]
                                         : tile[((e / D) * 16 + o) * LD + e % D];
                    q[l] = top && finite ? round127(x, inv, big) : 0;
                }
                w[j] = pack4(q[0], q[1], q[2], q[3]);
            }
            const int to = is_k ? e * 16 : (e % D) * KV8_BLOCK + (e / D) * 16;
            *reinterpret_cast<uint4*>(ints + to) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if (tid == 0) *scale = finite ? __fdiv_rn(big, 127.f) : __uint_as_float(0x7fffffffu);
        if (blk >= b1 || blockIdx.x > 0) break;
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.c.open_block[bh + z] = b1;
}

// A CTA of 256 threads reads one block's int8 keys or values and writes its rows in f32.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, Seqs s, float* k, float* v, int* err) {
    chain_release();
    const int z = chain_wait();
    __shared__ uint4 raw[KV8_BLOCK * D / 16];
    const int bh = blockIdx.y, b = bh / c.n_head_kv, h = bh % c.n_head_kv;
    const bool is_k = blockIdx.z == 0;
    float* out = is_k ? k : v;
    const Place at = place_of(s, b, c.blocks * KV8_BLOCK, threadIdx.x == 0 && blockIdx.x == 0 ? err : nullptr);
    const int blk = at.past / KV8_BLOCK + blockIdx.x, lo = blk * KV8_BLOCK;
    if (!out || lo >= at.past + at.count) return;
    out += z;
    const size_t at_blk = (size_t)bh * c.blocks + blk;
    const uint4* ints = reinterpret_cast<const uint4*>((is_k ? c.k : c.v) + at_blk * (KV8_BLOCK * D) + z);
    for (int e = threadIdx.x; e < KV8_BLOCK * D / 16; e += 256) raw[e] = ints[e];
    const float scale = (is_k ? c.k_scale : c.v_scale)[at_blk + z];
    __syncthreads();
    const int8_t* q = reinterpret_cast<const int8_t*>(raw);
    const size_t ts = (size_t)c.n_head_kv * D;
    for (int e = threadIdx.x; e < KV8_BLOCK * D / 4; e += 256) {
        const int r = e / (D / 4), col = e % (D / 4) * 4, i = lo + r - at.past;
        if (i < 0 || i >= at.count) continue;
        float4 x;
        if (is_k) {
            const char4 w = *reinterpret_cast<const char4*>(q + r * D + col);
            x = make_float4(w.x, w.y, w.z, w.w);
        } else {
            x = make_float4(q[col * KV8_BLOCK + r], q[(col + 1) * KV8_BLOCK + r], q[(col + 2) * KV8_BLOCK + r],
                            q[(col + 3) * KV8_BLOCK + r]);
        }
        float* to = out + ((size_t)b * s.n + i) * ts + (size_t)h * D + col;
        to[0] = x.x * scale;
        to[1] = x.y * scale;
        to[2] = x.z * scale;
        to[3] = x.w * scale;
    }
}

// The most blocks a call of n tokens can touch, wherever it starts.
int touched(int n) { return (n + 2 * (KV8_BLOCK - 1)) / KV8_BLOCK; }

template <typename T, int D>
int append(const Kv8Append& p, cudaStream_t st) {
    constexpr size_t smem = 2 * KV8_BLOCK * (D + 1) * sizeof(float);
    static_assert(smem <= 48 * 1024, "staging fits without opting in");
    // CTA 0 takes the first and the last block
    const dim3 grid((unsigned)std::max(1, touched(p.s.n) - 1), (unsigned)(p.s.n_batch * p.c.n_head_kv));
    return launch_chained_smem(kv8_append_kernel<T, D>, grid, dim3(2 * HALF), smem, st, p) == cudaSuccess ? 0 : -1;
}

}  // namespace

int kv8_append_launch(const Kv8Append& p, int type, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    if (type == TYPE_BF16) return p.c.d == 64 ? append<__nv_bfloat16, 64>(p, st) : append<__nv_bfloat16, 128>(p, st);
    return p.c.d == 64 ? append<float, 64>(p, st) : append<float, 128>(p, st);
}

int kv8_read_launch(const Kv8& c, const Seqs& s, float* k, float* v, int* err, cudaStream_t st) {
    if (s.n_batch == 0 || s.n == 0 || (!k && !v)) return 0;
    const dim3 grid((unsigned)touched(s.n), (unsigned)(s.n_batch * c.n_head_kv), 2);
    void (*kern)(Kv8, Seqs, float*, float*, int*) = c.d == 64 ? kv8_read_kernel<64> : kv8_read_kernel<128>;
    return launch_chained(kern, grid, dim3(256), st, c, s, k, v, err) == cudaSuccess ? 0 : -1;
}

}  // namespace zwg
