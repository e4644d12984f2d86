// The cache in 8 bits (zwg_kv8): appending to it and reading it back.
//
//   scale = max |x| / 127 over a block's 32 x d values of one head,  q = rint(127 x / max |x|)
//
// kv8_append_kernel: a CTA of 512 threads takes one block that the call touches, keys in its
// first 256 threads and values in the rest. A thread holds 4 (d 64: 2) rows' pieces of 4 elements in
// registers, new ones from the caller and older ones from the open rows, or from the int8 values
// where the block is not the open one; one reduction takes the largest magnitude, and each thread
// quantises what it holds: keys go out as rows, values, 4 tokens to a word, through shared memory
// as columns. Keys that are rotated on the way in, or that lie transposed, meet in shared memory
// first. The first and the last block a call touches share the open rows, the first reading what
// the last one replaces, so one CTA takes both, one after the other.
// Bound by memory and by issue alike for a chunk of a prompt (f32 in, a quarter of it out; the exact
// quotients and byte turns take 62 % of the issue slots): 64 sequences x 256 tokens, 2 heads of d 128, f32,
// 42 MB: 14.5 us, 2.9 TB/s, and reading them back 6.2 us out of L2 (10.8 from memory). Staging every row in
// shared memory and turning values byte by byte there took 92 us for both. Cold, under a profiler: 21.0 us (bf16 rows
// 22.9), 35.5 where the keys lie transposed in the staging of the q/k/v product and 63 where they are rotated here: both
// go through shared memory one element at a time, in 64 registers with 176 to 204 bytes of spills read back in a
// thread at d 128 (the direct forms: 4 at most). Bound by the latency of one CTA's
// chain of loads and barriers for a step: 4.0 us for 64 sequences' token.
//
// Rounding: the rounded quotient is found from 127 x * (1 / max |x|) in f32 unless that is
// within 3e-5 of the border between two integers; there the f64 quotient of the exact product
// 127 x decides, which is exact at a border (the operands have 31 and 24 bits). So the values
// are the correctly rounded ones, whatever the order of operations elsewhere.
#include <cuda_bf16.h>

#include <algorithm>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv8_attn.cuh"
#include "seqs.cuh"

namespace zwg {
namespace {

using namespace kv8;

constexpr int HALF = 256;  // threads for keys, and as many for values

// rint(127 x / top) of four values whose f32 quotients come near a border (or overflow 127 / top).
__device__ __noinline__ uint32_t exact4(float4 x, float top) {
    const auto q = [&](float v) { return (uint32_t)(int)rint(__ddiv_rn(127.0 * (double)v, (double)top)) & 255u; };
    return q(x.x) | q(x.y) << 8 | q(x.z) << 16 | q(x.w) << 24;
}

// The four int8 of a word; inv = 127 / top in f32.
ZWG_DEV uint32_t quantise4(float4 x, float inv, float top) {
    constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer, in the low bits
    const float y[4] = {__fmul_rn(x.x, inv), __fmul_rn(x.y, inv), __fmul_rn(x.z, inv), __fmul_rn(x.w, inv)};
    uint32_t t[4];
    float near = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float r = __fadd_rn(y[i], kRound);
        t[i] = __float_as_uint(r);
        near = fmaxf(near, fabsf(__fsub_rn(y[i], __fsub_rn(r, kRound))));
    }
    // y is off by 127 * 2^-23 = 1.5e-5 at most
    if (near > 0.49997f || !(inv < 3e38f)) return exact4(x, top);
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

// 4 x 4 bytes turned: byte i of word j becomes byte j of word i.
ZWG_DEV void turn4x4(uint32_t (&w)[4]) {
    const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
    const uint32_t c = __byte_perm(w[0], w[1], 0x7362), d = __byte_perm(w[2], w[3], 0x7362);
    w[0] = __byte_perm(a, b, 0x5410);
    w[1] = __byte_perm(a, b, 0x7632);
    w[2] = __byte_perm(c, d, 0x5410);
    w[3] = __byte_perm(c, d, 0x7632);
}

// Word w (tokens 4w .. 4w + 3) of a value column of 8 words in shared memory: the words are shuffled by
// column, so that a warp's columns meet in few banks.
ZWG_DEV int turned(int column, int w) { return column * 8 + (w ^ ((column >> 2) & 7)); }

// STAGED: keys are rotated or lie transposed. WIDE: pieces of four elements are aligned.
template <typename T, int D, bool STAGED, bool WIDE>
__global__ void __launch_bounds__(2 * HALF, 2) kv8_append_kernel(Kv8Append p) {
    chain_release();
    const int z = chain_wait();
    constexpr int LD = D + 1;     // odd: neither rows nor columns of the staging meet in a bank
    constexpr int LANES = D / 4;  // threads to a row
    constexpr int GROUPS = HALF / LANES, ROWS = KV8_BLOCK / GROUPS;  // a thread's rows: GROUPS * i + its group
    static_assert(ROWS == 4 || ROWS == 2, "a thread's rows make whole or half words of a value column");
    extern __shared__ float stage[];  // [32][LD] where STAGED
    __shared__ __align__(16) uint32_t columns[D * 8];
    __shared__ uint32_t top_of[2][HALF / 32];
    const int bh = blockIdx.y, b = bh / p.c.n_head_kv, h = bh - b * p.c.n_head_kv;
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
    float* open = (is_k ? p.c.k_open : p.c.v_open) + (size_t)bh * KV8_BLOCK * D + z;
    const T* src = static_cast<const T*>(is_k ? p.k.data : p.v.data) + z;
    const size_t ts = is_k ? p.k.ts : p.v.ts;
    src += b * (is_k ? p.k.bs : p.v.bs) + h * (is_k ? p.k_hs : p.v_hs);
    const int opened = __ldcg(p.c.open_block + bh + z);
    // rows 4 g .. 4 g + 3 (d 64: 2 g, 2 g + 1) and columns c .. c + 3
    const int g = tid / LANES, c = tid % LANES * 4, row0 = g * ROWS;
    for (int blk = b0 + blockIdx.x;; blk = b1) {
        const int lo = blk * KV8_BLOCK, held = max(0, at.past - lo), live = min(KV8_BLOCK, end - lo);
        const size_t at_blk = (size_t)bh * p.c.blocks + blk;
        int8_t* ints = (is_k ? p.c.k : p.c.v) + at_blk * (KV8_BLOCK * D) + z;
        float* scale = (is_k ? p.c.k_scale : p.c.v_scale) + at_blk + z;
        const bool from_open = opened == blk;
        const float old_scale = held && !from_open ? __ldcg(scale) : 0.f;
        // rows of the block: [0, held) the cache's, [held, live) new, the others zero. Every thread loads
        // rows of the call for all of its own, the nearest ones for those that are not new.
        float4 x[ROWS];
        Four<T> fresh[ROWS];
        if (!(STAGED && is_k)) {
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                fresh[i] = load_four(src + (size_t)min(max(lo + row0 + i - at.past, 0), at.count - 1) * ts + c, WIDE);
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const int r = row0 + i;
            x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < held) {
                if (from_open) {
                    x[i] = __ldcg(reinterpret_cast<const float4*>(open + r * D + c));
                } else {
                    const int8_t* q = ints + (is_k ? r * D + c : c * KV8_BLOCK + r);
                    const int e = is_k ? 1 : KV8_BLOCK;
                    x[i] = make_float4(q[0] * old_scale, q[e] * old_scale, q[2 * e] * old_scale, q[3 * e] * old_scale);
                }
            }
        }
        if (!(STAGED && is_k)) {
#pragma unroll
            for (int i = 0; i < ROWS; i++)
                if (row0 + i >= held && row0 + i < live) x[i] = value_of(fresh[i]);
        }
        if constexpr (STAGED) {  // new keys, to where each thread's are, by way of shared memory
            const int n = live - held;
            if (is_k && p.k_es == 1) {
                for (int e = tid; e < n * D; e += HALF) {
                    const int r = held + e / D, i = e % D;
                    stage[r * LD + i] = up(src[(size_t)(lo + r - at.past) * ts + i]);
                }
            } else if (is_k) {  // transposed: neighbouring tokens are neighbours in memory
#pragma unroll 8
                for (int e = tid; e < KV8_BLOCK * D; e += HALF) {
                    const int i = e / KV8_BLOCK, r = e % KV8_BLOCK;
                    if (r >= held && r < live) stage[r * LD + i] = up(src[(size_t)(lo + r - at.past) * ts + i * p.k_es]);
                }
            }
            __syncthreads();
            if (is_k && p.rope.cos) {
                const int half = p.rope.rot / 2;
                for (int e = tid; e < n * half; e += HALF) {
                    const int r = held + e / half, i = e % half;
                    const size_t row = (size_t)(lo + r) * half + i;
                    const float co = p.rope.cos[row], si = p.rope.sin[row];
                    float* xa = stage + r * LD + (p.rope.interleaved ? 2 * i : i);
                    float* xb = p.rope.interleaved ? xa + 1 : xa + half;
                    const float a = *xa, bb = *xb;
                    *xa = __fsub_rn(__fmul_rn(a, co), __fmul_rn(bb, si));
                    *xb = __fadd_rn(__fmul_rn(a, si), __fmul_rn(bb, co));
                }
            }
            __syncthreads();
            if (is_k) {
#pragma unroll
                for (int i = 0; i < ROWS; i++) {
                    const int r = row0 + i;
                    const float* s = stage + r * LD + c;
                    if (r >= held && r < live) x[i] = make_float4(s[0], s[1], s[2], s[3]);
                }
            }
        }
        // |x|'s bit pattern orders like the value, with infinities and NaN above all others
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            top = max(max(top, __float_as_uint(fabsf(x[i].x))), __float_as_uint(fabsf(x[i].y)));
            top = max(max(top, __float_as_uint(fabsf(x[i].z))), __float_as_uint(fabsf(x[i].w)));
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) top_of[side][warp] = top;
        __syncthreads();  // and every thread has read the int8 values and open rows
#pragma unroll
        for (int w = 0; w < HALF / 32; w++) top = max(top, top_of[side][w]);
        const float big = __uint_as_float(top);
        const bool some = top && top < 0x7f800000u;
        const float inv = some ? __fdiv_rn(127.f, big) : 0.f;
        uint32_t q[4] = {};
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const int r = row0 + i;
            if (blk == b1 && (r >= held || !from_open)) __stcg(reinterpret_cast<float4*>(open + r * D + c), x[i]);
            if (some) q[i] = quantise4(x[i], inv, big);
            if (is_k) *reinterpret_cast<uint32_t*>(ints + r * D + c) = q[i];
        }
        if (!is_k) {
            turn4x4(q);  // word j: column c + j of the thread's rows
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (ROWS == 4) columns[turned(c + j, g)] = q[j];
                else reinterpret_cast<uint16_t*>(columns)[turned(c + j, g / 2) * 2 + g % 2] = (uint16_t)q[j];
            }
        }
        __syncthreads();
        if (!is_k) {
            for (int e = tid; e < D * 2; e += HALF) {
                const int col = e / 2, w = e % 2 * 4;
                *reinterpret_cast<uint4*>(ints + e * 16) = make_uint4(columns[turned(col, w)], columns[turned(col, w + 1)],
                                                                      columns[turned(col, w + 2)], columns[turned(col, w + 3)]);
            }
        }
        if (tid == 0) *scale = top < 0x7f800000u ? __fdiv_rn(big, 127.f) : __uint_as_float(0x7fffffffu);
        if (blk >= b1 || blockIdx.x > 0) break;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) p.c.open_block[bh + z] = b1;
}

// A CTA of 256 threads reads one block's int8 keys or values and writes its rows in f32, four rows'
// pieces of four elements a thread.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(Kv8 c, Seqs s, float* k, float* v, int* err) {
    chain_release();
    const int z = chain_wait();
    constexpr int LANES = D / 4, GROUPS = 256 / LANES, ROWS = KV8_BLOCK / GROUPS;
    __shared__ uint32_t columns[D * 8];
    const int bh = blockIdx.y, b = bh / c.n_head_kv, h = bh - b * c.n_head_kv, tid = threadIdx.x;
    const bool is_k = blockIdx.z == 0;
    float* out = is_k ? k : v;
    const Place at = place_of(s, b, c.blocks * KV8_BLOCK, tid == 0 && blockIdx.x == 0 ? err : nullptr);
    const int blk = at.past / KV8_BLOCK + blockIdx.x, lo = blk * KV8_BLOCK;
    if (!out || lo >= at.past + at.count) return;
    const size_t at_blk = (size_t)bh * c.blocks + blk;
    const int8_t* ints = (is_k ? c.k : c.v) + at_blk * (KV8_BLOCK * D) + z;
    const float scale = (is_k ? c.k_scale : c.v_scale)[at_blk + z];
    const int g = tid / LANES, col = tid % LANES * 4;
    uint32_t q[4] = {};
    if (is_k) {
#pragma unroll
        for (int i = 0; i < ROWS; i++) q[i] = *reinterpret_cast<const uint32_t*>(ints + (g * ROWS + i) * D + col);
    } else {
        for (int e = tid; e < D * 2; e += 256) {
            const uint4 w = *reinterpret_cast<const uint4*>(ints + e * 16);
            const int column = e / 2, at_w = e % 2 * 4;
            columns[turned(column, at_w)] = w.x;
            columns[turned(column, at_w + 1)] = w.y;
            columns[turned(column, at_w + 2)] = w.z;
            columns[turned(column, at_w + 3)] = w.w;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 4; j++)
            q[j] = ROWS == 4 ? columns[turned(col + j, g)]
                             : reinterpret_cast<uint16_t*>(columns)[turned(col + j, g / 2) * 2 + g % 2];
        turn4x4(q);
    }
    const size_t ts = (size_t)c.n_head_kv * D;
    out += z + (size_t)b * s.n * ts + (size_t)h * D + col;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const int t = lo + g * ROWS + i - at.past;
        if (t < 0 || t >= at.count) continue;
        const char4 w = *reinterpret_cast<char4*>(&q[i]);
        *reinterpret_cast<float4*>(out + t * ts) = make_float4(w.x * scale, w.y * scale, w.z * scale, w.w * scale);
    }
}

// The most blocks a call of n tokens can touch, wherever it starts.
int touched(int n) { return (n + 2 * (KV8_BLOCK - 1)) / KV8_BLOCK; }

template <typename T, int D>
int append(const Kv8Append& p, cudaStream_t st) {
    const bool staged = p.rope.cos || p.k_es != 1;
    const size_t smem = staged ? KV8_BLOCK * (D + 1) * sizeof(float) : 0;
    // rows whose pieces of four elements are aligned
    const auto whole = [](const Rows& r, size_t hs) {
        return ((uintptr_t)r.data | (r.bs * sizeof(T)) | (r.ts * sizeof(T)) | (hs * sizeof(T))) % (4 * sizeof(T)) == 0;
    };
    const bool wide = (staged || whole(p.k, p.k_hs)) && whole(p.v, p.v_hs);
    // CTA 0 takes the first and the last block
    const dim3 grid((unsigned)std::max(1, touched(p.s.n) - 1), (unsigned)(p.s.n_batch * p.c.n_head_kv));
    void (*kern)(Kv8Append) = staged ? (wide ? kv8_append_kernel<T, D, true, true> : kv8_append_kernel<T, D, true, false>)
                                     : (wide ? kv8_append_kernel<T, D, false, true> : kv8_append_kernel<T, D, false, false>);
    return launch_chained_smem(kern, grid, dim3(2 * HALF), smem, st, p) == cudaSuccess ? 0 : -1;
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
