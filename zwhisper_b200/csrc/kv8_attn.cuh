// What the kernels of a cache in 8 bits share: int8 values as exact f16, f32 values as f16 pieces, and
// the loads and stores of rows.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "sm100.cuh"

namespace zwg {
namespace kv8 {

constexpr float kLog2e = 1.4426950408889634f;

ZWG_DEV uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Four int8 of a word -> two f16 pairs, exactly: 0x6400 | (x + 128) is 1024 + 128 + x.
ZWG_DEV void ints_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2(__half_raw{0x6480}, __half_raw{0x6480});
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    lo = h2u(__hsub2(*reinterpret_cast<__half2*>(&a), off));
    hi = h2u(__hsub2(*reinterpret_cast<__half2*>(&b), off));
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

// The power of two of |x|'s exponent and its inverse, both normal numbers: 2^-126 for zero and what is smaller,
// 2^126 for what is larger (x / 2^126 is below 4), infinite or NaN.
ZWG_DEV void power_of(float x, float& p, float& inv) {
    const uint32_t e = min(max(__float_as_uint(x) & 0x7f800000u, 0x00800000u), 0x7e800000u);
    p = __uint_as_float(e);
    inv = __uint_as_float(0x7f000000u - e);
}

ZWG_DEV float up(float x) { return x; }
ZWG_DEV float up(__nv_bfloat16 x) { return __bfloat162float(x); }

// Four elements of a row as they lie in memory, and as f32: loads are kept apart from their conversion,
// so that several of them are on their way at once.
template <typename T>
struct Four;
template <>
struct Four<float> {
    float4 w;
};
template <>
struct Four<__nv_bfloat16> {
    uint2 w;
};
ZWG_DEV Four<float> load_four(const float* p, bool wide) {
    return {wide ? *reinterpret_cast<const float4*>(p) : make_float4(p[0], p[1], p[2], p[3])};
}
ZWG_DEV Four<__nv_bfloat16> load_four(const __nv_bfloat16* p, bool wide) {
    if (wide) return {*reinterpret_cast<const uint2*>(p)};
    const uint16_t* u = reinterpret_cast<const uint16_t*>(p);
    return {make_uint2(u[0] | (uint32_t)u[1] << 16, u[2] | (uint32_t)u[3] << 16)};
}
ZWG_DEV float4 value_of(Four<float> x) { return x.w; }
ZWG_DEV float4 value_of(Four<__nv_bfloat16> x) {
    return make_float4(__uint_as_float(x.w.x << 16), __uint_as_float(x.w.x & 0xffff0000u), __uint_as_float(x.w.y << 16),
                       __uint_as_float(x.w.y & 0xffff0000u));
}

// Four output elements of a row whose weights sum to l (0: no key was seen).
ZWG_DEV void store4(float* out, float4 o, float inv, bool vec) {
    const float4 y = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (vec) {
        *reinterpret_cast<float4*>(out) = y;
    } else {
        out[0] = y.x;
        out[1] = y.y;
        out[2] = y.z;
        out[3] = y.w;
    }
}
ZWG_DEV void store4(__nv_bfloat16* out, float4 o, float inv, bool vec) {
    __nv_bfloat162 y[2] = {__floats2bfloat162_rn(o.x * inv, o.y * inv), __floats2bfloat162_rn(o.z * inv, o.w * inv)};
    if (vec) {
        *reinterpret_cast<uint2*>(out) = *reinterpret_cast<uint2*>(y);
    } else {
        out[0] = y[0].x;
        out[1] = y[0].y;
        out[2] = y[1].x;
        out[3] = y[1].y;
    }
}

// 16 consecutive elements as f32.
ZWG_DEV void load16(const float* q, float (&x)[16], bool vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 v = reinterpret_cast<const float4*>(q)[i];
            x[i * 4] = v.x, x[i * 4 + 1] = v.y, x[i * 4 + 2] = v.z, x[i * 4 + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = q[i];
    }
}
ZWG_DEV void load16(const __nv_bfloat16* q, float (&x)[16], bool vec) {
    if (vec) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint4 v = reinterpret_cast<const uint4*>(q)[i];
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[i * 8 + j * 2] = __uint_as_float(w[j] << 16);
                x[i * 8 + j * 2 + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) x[i] = __bfloat162float(q[i]);
    }
}

// Rows whose elements can be read or written 16 bytes (of f32; 8 of bf16) at a time.
inline bool wide(const Rows& r, size_t elem, size_t bytes) {
    return ((uintptr_t)r.data | (r.bs * elem) | (r.ts * elem)) % bytes == 0;
}

}  // namespace kv8
}  // namespace zwg
