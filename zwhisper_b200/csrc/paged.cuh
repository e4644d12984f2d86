// What the kernels of a cache in pages share: where a slot's rows are, the trees of drafted tokens,
// and 16-bit elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "seqs.cuh"

namespace zwg {
namespace paged {

// The cache's type beside rows of T: f16 holds 11 bits of an f32 row, and two f16 pieces of a query
// against it have f32's accuracy; bf16 rows are held as they are.
template <typename T>
struct Held;
template <>
struct Held<float> {
    using type = __half;
    static constexpr uint32_t exponent = 0x7c00u;  // all ones: infinite or NaN
};
template <>
struct Held<__nv_bfloat16> {
    using type = __nv_bfloat16;
    static constexpr uint32_t exponent = 0x7f80u;
};

ZWG_DEV __half held(float x, __half) { return __float2half_rn(x); }
ZWG_DEV __nv_bfloat16 held(float x, __nv_bfloat16) { return __float2bfloat16_rn(x); }
ZWG_DEV float up(float x) { return x; }
ZWG_DEV float up(__half x) { return __half2float(x); }
ZWG_DEV float up(__nv_bfloat16 x) { return __bfloat162float(x); }

ZWG_DEV void add(float& x, float y) { x += y; }
ZWG_DEV void add(__nv_bfloat16& x, float y) { x = __float2bfloat16_rn(__bfloat162float(x) + y); }

// A word's two 16-bit elements, those that are infinite or NaN as zero.
ZWG_DEV uint32_t finite(uint32_t w, uint32_t exponent) {
    if ((w & exponent) == exponent) w &= 0xffff0000u;
    if ((w & exponent << 16) == exponent << 16) w &= 0xffffu;
    return w;
}

// The page of sequence b's slot (below c.room), or -1: the table's entry is not one of the pool's.
ZWG_DEV int page_of(const Paged& c, int b, int slot) {
    const int id = __ldcg(c.table + b * c.ts + (slot >> c.log_page));
    return (unsigned)id < (unsigned)c.n_pages ? id : -1;
}

// Element of a page's row: head h, slot's place in the page.
ZWG_DEV size_t row_at(const Paged& c, int page, int h, int slot) {
    return page * c.ps + ((((size_t)h << c.log_page) + (slot & ((1 << c.log_page) - 1))) * c.d);
}

// The whole CTA: the parents of a sequence's `count` tokens (at most MOST_TREE) into shared memory, and whether
// each is below its own index. One that is not leaves the sequence out.
template <typename I>
ZWG_DEV bool read_tree(const Tree& t, int b, int count, int z, I* parent) {
    int bad = 0;
    const int n = blockDim.x * blockDim.y * blockDim.z;
    for (int i = threadIdx.x + blockDim.x * (threadIdx.y + blockDim.y * threadIdx.z); i < count; i += n) {
        const int a = __ldcg(t.parent + b * t.bs + i + z);
        parent[i] = (I)a;  // (where it is not bad, below MOST_TREE)
        bad |= a < -1 || a >= i;
    }
    return __syncthreads_or(bad) == 0;
}

}  // namespace paged
}  // namespace zwg
