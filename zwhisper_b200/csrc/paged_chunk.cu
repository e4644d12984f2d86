// Attention over a cache in pages for many query rows of a kv head (prompt chunks, trees of drafted tokens), on the
// tcgen05 tensor cores: the formulas of paged_attn.cu with 128 keys and 2 x 128 query rows at a time.
//
// paged_chunk_kernel. A CTA of 20 warps takes 256 rows (row = query * group + head) of one (sequence, kv head), or
// a cut of their keys, in two slots of 128 rows; where it has 128 rows or less, both slots take them and every
// other tile of keys, so that one's softmax still runs during the other's products, and their sums meet in shared
// memory at the end. Warps 0-7 and 8-15 are the slots' softmax, two threads a row that take half of a tile's keys
// (and later half of O's columns) each, so that these stay in its registers, and tell each other their maxima.
// Warps 16 and 17 issue the products of one slot each, S = Q K^T (from shared memory) into TMEM and O += P V; warp
// 18 brings keys and values by TMA, a box to each page, in the 128-byte swizzle (keys K-major, values MN-major:
// neither is transposed); warp 19 sees to it that values of slots that no row sees are zero, and takes out
// infinities and NaN that only some rows see (noted in `flagged`; the rows that do see them take them in at the
// end, by themselves).
// One piece: P goes beside S (d 64) or into shared memory (d 128), so that the next S is computed during this
// one's softmax; O stays in TMEM and is rescaled there only where a row's maximum grows by more than 2^8 (bf16
// rows) or 2^4.
// Two f16 pieces (f32 rows; P's hold 2^11 p with p below 2^4): P goes over S, and as the tensor cores truncate
// their sums, each tile's O starts from zero and is added in f32 to the row's in the threads' registers.
// Bound by the softmax beside the products: 32 sequences of 256 tokens after 1744, 12 / 2 heads of d 128, bf16, in
// a graph, 130.6 us (57 us of products at the rate of a large bf16 product). Of the cycles in which an SM has a CTA the
// tensor cores are busy 42 %, the exponentials' unit 41 %, issue 52 %; of all cycles the tensor cores 32 %, as 384
// CTAs fill 148 SMs 2.6 times. DRAM reads 93 MB. f32 in two pieces 262 to 276 us, by the scores, for twice the
// products; 16 sequences of up to 1750 tokens with 250 new ones, 14 / 2 heads of d 64, f32, 61 to 63 us, of which about
// 16 are a CTA's start and end. A softmax thread's 104 registers are too few in every form: bytes spilled and read back
// bf16 132 / 328 (d 128), 108 / 316 (d 64); f32 in two pieces 304 / 492, 188 / 240; in one 140 / 336, 108 / 316.
#include <algorithm>
#include <climits>
#include <cmath>

#include "chain.cuh"
#include "common.cuh"
#include "kernels.h"
#include "kv8_attn.cuh"
#include "paged.cuh"
#include "seqs.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace zwg {
namespace {

using namespace sm100;
using kv8::Four;
using kv8::kLog2e;
using kv8::load_four;
using kv8::pieces_of;
using kv8::power_of;
using kv8::store4;
using kv8::value_of;
using kv8::wide;
using paged::finite;
using paged::Held;
using paged::page_of;
using paged::read_tree;
using paged::row_at;

constexpr int BM = 128, BN = 128;  // rows of a slot, keys of a tile
constexpr int SOFTMAX = 512, THREADS = SOFTMAX + 128;
// launched with 96 registers a thread (65536 / 640, a multiple of 8): 512 * 104 + 128 * 64 = 640 * 96
constexpr uint32_t REGS_SOFTMAX = 104, REGS_CONTROL = 64;
static_assert(SOFTMAX * REGS_SOFTMAX + 128 * REGS_CONTROL <= THREADS * 96, "register split exceeds the launch");
constexpr uint32_t TMEM_COLS = 512;
constexpr int EDGES = 4;  // tiles that not all of a CTA's rows see whole: its rows are of 256 tokens at the most

// Where P goes: beside S where TMEM has room for it, into shared memory where that has (one piece of d 128, beside one
// buffer of values); else over S, so that the next S waits until the values' product has read it.
template <int D, int P>
constexpr bool BESIDE = D == 64 && P == 1;
template <int D, int P>
constexpr bool SHARED = D == 128 && P == 1;
template <int D, int P>
constexpr bool EARLY = P == 1;  // the next S is computed as soon as this one has been read
// The slots' exponentials take turns, so that one's run while the other loads scores, finds maxima and waits: left
// alone they fall into step, and all wait for the same unit. 32 x 256 tokens after 1744, d 128 bf16 137 -> 130 us, f32
// 271 -> 261, d 64 (14 / 2 heads) bf16 145 -> 134; d 64 in two pieces, whose slots wait for products in between, 200 -> 205: not there.
template <int D, int P>
constexpr bool TURNS = P == 1 || D == 128;
__host__ __device__ constexpr uint32_t s_col(int t) { return t * 128u; }
template <int D, int P>
__host__ __device__ constexpr uint32_t p_col(int t) { return BESIDE<D, P> ? 384u + t * 64u : t * 128u; }
template <int D>
__host__ __device__ constexpr uint32_t o_col(int t) { return 256u + t * D; }

template <int D, int P>
struct Smem {
    // buffers of keys and values; where both slots take the same rows, q[1]'s last piece is another one of what has one
    static constexpr int KS = SHARED<D, P> ? 1 : 2, VS = D * P > 128 ? 1 : 2;
    uint8_t q[2][P][D / 64][BM * 128];  // query slots: [row][64], swizzled
    uint8_t v[VS][D / 64][BN * 128];    // values: [key][64]
    uint8_t k[KS][D / 64][BN * 128];    // keys: [key][64]
    uint8_t p[SHARED<D, P> ? 2 : 1][SHARED<D, P> ? 2 : 1][SHARED<D, P> ? BM * 128 : 16];  // P of a slot: [row][64 keys]
    float part[2][2][BM];               // what a row's two threads tell each other: [slot][half]; the queries' scales first
    int16_t parent[MOST_TREE];
    uint32_t valid[4];                  // of a tile: a bit for each 16 keys that lie in a page
    uint32_t flagged[EDGES][BN / 32];   // keys whose infinities and NaN were taken out
    uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_ready[2], v_empty[2], s_full[2], s_free[2], p_full[2], pv_done[2], drained[2];
    uint64_t started, turn[2];  // slot 0's first P is there; a slot may begin its exponentials
    uint32_t tmem_base;
};

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

// One thread of a warp whose threads are all here.
ZWG_DEV bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(one));
    return one != 0;
}

// The lowest n bits (n of any value).
ZWG_DEV uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }

// Whether one of a piece's eight 16-bit elements is infinite or NaN: its magnitude carries into the sign's place.
ZWG_DEV bool not_finite(uint4 w, uint32_t exponent) {
    const uint32_t k = (0x8000u - exponent) * 0x10001u, m = 0x7fff7fffu;
    return (((w.x & m) + k | (w.y & m) + k | (w.z & m) + k | (w.w & m) + k) & 0x80008000u) != 0;
}

// The whole CTA: the sequence that comes n-th by its length, longest first, so that the last CTAs to start are the
// shortest ones (16 sequences of up to 1750 tokens, 250 new ones, 14 / 2 heads of d 64, f32: 75 -> 61 us; 64 of up to
// 1000, 128 new ones, d 128, bf16: 85 -> 72). All CTAs see the same lengths; the lower index goes first where they are
// equal. Up to MOST_SORTED sequences: a CTA compares each with all, and SMs have several CTAs of more of them in turn, so
// that one long one holds up less. scratch: MOST_SORTED + 4 ints, free behind the call.
constexpr int MOST_SORTED = 256;
ZWG_DEV int by_length(const Seqs& s, int n, int z, int4* scratch) {
    int* lengths = reinterpret_cast<int*>(scratch);
    const int i = threadIdx.x, padded = (s.n_batch + 3) & ~3, mine = i < s.n_batch ? __ldcg(s.past + i + z) : INT_MIN;
    if (i < padded) lengths[i] = mine;  // (behind the last sequence: shorter than any, or as short and after it)
    __syncthreads();
    if (i < s.n_batch) {
        int before = 0;
        for (int j = 0; j < padded; j += 4) {
            const int4 w = scratch[j / 4];
            before += (w.x > mine || (w.x == mine && j < i)) + (w.y > mine || (w.y == mine && j + 1 < i)) +
                      (w.z > mine || (w.z == mine && j + 2 < i)) + (w.w > mine || (w.w == mine && j + 3 < i));
        }
        if (before == n) lengths[MOST_SORTED] = i;
    }
    __syncthreads();
    const int b = lengths[MOST_SORTED];
    __syncthreads();
    return b;
}

// vec: bit 0 queries can be read 4 elements at a time, bit 1 outputs written 16 bytes at a time.
template <typename T, int D, int P>
__global__ void __launch_bounds__(THREADS, 1)
    paged_chunk_kernel(PagedAttn p, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                       int splits, int vec, float scale) {
    chain_release();
    const int z = chain_wait();
    extern __shared__ __align__(1024) uint8_t smem_raw[];  // the swizzle goes by address: checked below
    Smem<D, P>& sm = *reinterpret_cast<Smem<D, P>*>(smem_raw);
    if (smem_u32(smem_raw) & 1023) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    using S = Smem<D, P>;
    using H = typename Held<T>::type;
    constexpr bool RAW = sizeof(T) == 2;
    constexpr float SHIFT = RAW ? 0.f : 11.f, STALE = RAW ? 8.f : 4.f;
    constexpr uint32_t EXP = Held<T>::exponent;
    const int tile = blockIdx.x / splits, split = blockIdx.x - tile * splits;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = p.n_head / p.c.n_head_kv;
    const bool tree = p.tree.parent != nullptr;
    int b = blockIdx.y / p.c.n_head_kv;
    const int h = blockIdx.y - b * p.c.n_head_kv;
    if (p.s.past && p.s.n_batch > 1 && p.s.n_batch <= MOST_SORTED) b = by_length(p.s, b, z, reinterpret_cast<int4*>(&sm));
    const int bh = b * p.c.n_head_kv + h;
    const Place at = place_of(p.s, b, p.c.room, threadIdx.x == 0 && blockIdx.x == 0 && h == 0 ? p.err : nullptr);
    const int rows = at.count * group, row0 = tile * 2 * BM;
    if (row0 >= rows) return;
    const int first = p.s.first ? __ldcg(p.s.first + b + z) : 0;
    if (first < 0) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    if (tree && !read_tree(p.tree, b, at.count, z, sm.parent)) {
        if (threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    const bool two = row0 + BM < rows;                                     // a slot to each 128 rows
    const int end = at.past + (min(rows, row0 + 2 * BM) - 1) / group + 1;  // slots from it on: seen by no row
    const int by_all = tree ? at.past : at.past + row0 / group + 1;        // slots below it: by all
    const int lo = first / BN, all = first < end ? (end + BN - 1) / BN - lo : 0;
    const int from = (int)((long long)all * split / splits), n_tiles = (int)((long long)all * (split + 1) / splits) - from;
    const int key_lo = (lo + from) * BN;
    const int edge0 = max(0, by_all / BN - lo - from);  // the first tile (of this CTA) that not all rows see whole
    int* err = p.err;
    // buffers of keys and of values, less one: tile j's is j & that, filled for the (j >> that)th time
    const int more_k = S::KS == 2 || !two ? 1 : 0, more_v = S::VS == 2 || !two ? 1 : 0;
    const auto k_at = [&](int j) { return !(j & more_k) ? sm.k[0][0] : S::KS == 2 ? sm.k[S::KS - 1][0] : sm.q[1][P - 1][0]; };
    const auto v_at = [&](int j) { return !(j & more_v) ? sm.v[0][0] : S::VS == 2 ? sm.v[S::VS - 1][0] : sm.q[1][P - 1][0]; };
    constexpr int ISSUER = SOFTMAX / 32;             // the first of the four other warps
    constexpr int EVERYONE = SOFTMAX + 32;           // the softmax warps and the last one

    if (threadIdx.x < EDGES * (BN / 32)) sm.flagged[threadIdx.x / (BN / 32)][threadIdx.x % (BN / 32)] = 0;
    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; t++) {
            mbar_init(&sm.q_full[t], two ? 8 : 16);
            mbar_init(&sm.s_full[t], 2);  // the products' completion, and the issuer's own: it has seen the tile's pages
            mbar_init(&sm.s_free[t], 8);
            mbar_init(&sm.p_full[t], 8);
            mbar_init(&sm.pv_done[t], 1);
            mbar_init(&sm.drained[t], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.k_full[i], 1);
            mbar_init(&sm.k_empty[i], two ? 2 : 1);
            mbar_init(&sm.v_full[i], 1);
            mbar_init(&sm.v_ready[i], 1);
            mbar_init(&sm.v_empty[i], two ? 2 : 1);
        }
        mbar_init(&sm.started, 1);
        mbar_init(&sm.turn[0], 8);
        mbar_init(&sm.turn[1], 8);
        fence_mbar_init();
    }
    __syncwarp();
    if (warp == ISSUER) {
        tmem_alloc(&sm.tmem_base, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    if (warp >= ISSUER) {
        regs_dec<REGS_CONTROL>();
        if (warp < ISSUER + 2) {
            // ------------------------------------------------ the products of slot t
            const int t = warp - ISSUER, mine = two ? n_tiles : (n_tiles - t + 1) / 2;
            if (mine > 0 && elect_one()) {
                constexpr uint32_t idesc_s = idesc_f16(BM, BN, RAW, false, false);
                constexpr uint32_t idesc_o = idesc_f16(BM, D, RAW, false, true);
                const int qt = two ? t : 0;
                // descriptors: their bases, to which addresses in units of 16 bytes are added
                const uint64_t q_desc = smem_desc_sw128(smem_u32(sm.q[qt][0][0]), 16, 1024);
                const uint64_t k_desc = smem_desc_sw128(smem_u32(k_at(0)), 16, 1024), v_desc = smem_desc_sw128(smem_u32(v_at(0)), BN * 128, 1024);
                const int k_step = (int)(k_at(1) - k_at(0)) / 16, v_step = (int)(v_at(1) - v_at(0)) / 16;  // to the other buffer
                const uint64_t p_desc = smem_desc_sw128(smem_u32(sm.p[SHARED<D, P> ? t : 0][0]), 16, 1024);
                constexpr int HALF = BM * 128 / 16, SIDE = D / 64 * HALF;  // 64 columns of a tile, a tile
                bool ok = mbar_wait(&sm.q_full[qt], 0, err);
                const auto tile_of = [&](int it) { return two ? it : 2 * it + t; };
                const auto keys = [&](int it) { return mbar_wait(&sm.k_full[tile_of(it) & more_k], tile_of(it) >> more_k & 1, err); };
                const auto scores = [&](int it) {
                    const int j = tile_of(it);
                    const uint64_t kb = k_desc + (int64_t)(j & more_k ? k_step : 0);
                    // S goes where the last S was read from, or its P, which the PV reads
                    if (it > 0 && !mbar_wait(EARLY<D, P> ? &sm.s_free[t] : &sm.pv_done[t], (it - 1) & 1, err)) return false;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < P; c++)  // (the small pieces first)
#pragma unroll
                        for (int kk = 0; kk < D / 16; kk++) {
                            const int at_k = kk / 4 * HALF + kk % 4 * 2;
                            mma_f16_ss(tmem + s_col(t), q_desc + (P - 1 - c) * SIDE + at_k, kb + at_k, idesc_s, c > 0 || kk > 0);
                        }
                    mma_commit(&sm.s_full[t]);
                    mma_commit(&sm.k_empty[j & more_k]);
                    mbar_arrive(&sm.s_full[t]);
                    return true;
                };
                ok = ok && keys(0) && scores(0);
                for (int it = 0; ok && it < mine; it++) {
                    const int j = tile_of(it), vs = j & more_v, turn = j >> more_v & 1;
                    const bool more = it + 1 < mine;
                    // waits that end during the softmax come before the one for its end: the next keys' too, but where each
                    // slot has one buffer of them, and they arrive while the values' product runs
                    if (more && two && !(ok = keys(it + 1))) break;
                    if (EARLY<D, P> && more && two && !(ok = scores(it + 1))) break;
                    if (!(ok = mbar_wait(&sm.v_full[vs], turn, err) && mbar_wait(&sm.v_ready[vs], turn, err))) break;
                    const uint64_t vb = v_desc + (int64_t)(vs ? v_step : 0);
                    if (!(ok = mbar_wait(&sm.p_full[t], it & 1, err))) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < P; c++)
#pragma unroll
                        for (int kk = 0; kk < BN / 16; kk++) {
                            const uint32_t pa = p_col<D, P>(t) + kk * 8 * P + (P - 1 - c) * 8, sum = (P == 1 && it > 0) || c > 0 || kk > 0;
                            if (SHARED<D, P>) mma_f16_ss(tmem + o_col<D>(t), p_desc + kk / 4 * HALF + kk % 4 * 2, vb + kk * 128, idesc_o, sum);
                            else mma_f16_ts(tmem + o_col<D>(t), tmem + pa, vb + kk * 128, idesc_o, sum);
                        }
                    mma_commit(&sm.pv_done[t]);
                    mma_commit(&sm.v_empty[vs]);
                    if (t == 0 && it == 0) mbar_arrive(&sm.started);
                    if (more && !two) ok = keys(it + 1);
                    if (more && !(EARLY<D, P> && two)) ok = ok && scores(it + 1);
                }
                if (!ok) {  // gave up: the products on their way end before TMEM is given back
                    mma_commit(&sm.drained[t]);
                    mbar_wait_drain(&sm.drained[t], 0);
                }
            }
        } else if (warp == ISSUER + 2) {
            // ------------------------------------------------ keys and values, a box of each page
            const int log_box = min(p.c.log_page, 7), box = 1 << log_box, n_box = BN >> log_box;  // a box's rows, a tile's boxes
            const auto look = [&](int j) {  // the page of the lane's box; -1: none of the pool's, -2: not needed
                const int slot = key_lo + j * BN + lane * box;
                if (j >= n_tiles || lane >= n_box || slot >= end || slot + box <= first) return -2;
                return page_of(p.c, b, slot + z);
            };
            int issued = 0, next = look(0);
            for (int j = 0; j < n_tiles; j++) {
                const int page = next, ks = j & more_k, vs = j & more_v;
                next = look(j + 1);
                if (page == -1) set_error(err, kErrBounds);
                const uint32_t there = __ballot_sync(0xffffffffu, page >= 0), none = __ballot_sync(0xffffffffu, page == -1);
                const uint32_t bytes = __popc(there) * box * 128 * (D / 64);
                const int row = (h << p.c.log_page) + ((key_lo + j * BN + lane * box) & ((1 << p.c.log_page) - 1));
                if (j > more_k && !mbar_wait_warp(&sm.k_empty[ks], ((j >> more_k) - 1) & 1, err)) break;
                if (lane == 0) {
                    uint32_t valid = 0;
                    for (int g = 0; g < BN / 16; g++) valid |= (none >> (g * 16 >> log_box) & 1 ? 0u : 1u) << g;
                    sm.valid[j & 3] = valid;
                    mbar_arrive_expect_tx(&sm.k_full[ks], bytes);
                }
                __syncwarp();
                if (page >= 0)
#pragma unroll
                    for (int c = 0; c < D / 64; c++) tma_load_3d(&tm_k, &sm.k_full[ks], k_at(j) + c * (BN * 128) + lane * box * 128, c * 64, row, page);
                issued = 2 * j + 1;
                if (j > more_v && !mbar_wait_warp(&sm.v_empty[vs], ((j >> more_v) - 1) & 1, err)) break;
                if (lane == 0) mbar_arrive_expect_tx(&sm.v_full[vs], bytes);
                __syncwarp();
                if (page >= 0)
#pragma unroll
                    for (int c = 0; c < D / 64; c++) tma_load_3d(&tm_v, &sm.v_full[vs], v_at(j) + c * (BN * 128) + lane * box * 128, c * 64, row, page);
                issued = 2 * j + 2;
            }
            // the copies on their way end before the CTA does (they have, unless a wait gave up)
            for (int i = 0; i <= more_k; i++) {
                const int j = (issued + 1) / 2 - 1 - i;
                if (j >= 0) mbar_wait_drain(&sm.k_full[j & more_k], j >> more_k & 1);
            }
            for (int i = 0; i <= more_v; i++) {
                const int j = issued / 2 - 1 - i;
                if (j >= 0) mbar_wait_drain(&sm.v_full[j & more_v], j >> more_v & 1);
            }
        } else {
            // ------------------------------------------------ values that some rows do not see
            for (int j = 0; j < n_tiles; j++) {
                const int vs = j & more_v, key0 = key_lo + j * BN;
                if (!mbar_wait_warp(&sm.v_full[vs], j >> more_v & 1, err)) break;
                const uint32_t valid = sm.valid[j & 3];
                if (key0 < first || key0 + BN > by_all || valid != 0xffu) {
                    // a lane has the same 16 bytes of every so many rows, whose places in the swizzle repeat every 4 of them
                    constexpr int UNITS = D / 8, AT_ONCE = 32 / UNITS;
                    const int u = lane % UNITS, r0 = lane / UNITS;
                    uint8_t* column = v_at(j) + u / 8 * (BN * 128);
                    const auto at_row = [&](int r) { return reinterpret_cast<uint4*>(column + r * 128 + ((u % 8 ^ (r & 7)) << 4)); };
                    const int begin = first > key0 || valid != 0xffu ? 0 : max(0, by_all - key0) & ~(4 * AT_ONCE - 1);
                    bool bad = false;
#pragma unroll 1
                    for (int r = begin + r0; r < BN; r += 4 * AT_ONCE) {
                        uint4 w[4];
#pragma unroll
                        for (int n = 0; n < 4; n++) w[n] = *at_row(r + n * AT_ONCE);
#pragma unroll
                        for (int n = 0; n < 4; n++) {
                            const int rr = r + n * AT_ONCE, slot = key0 + rr;
                            if (slot < first || slot >= end || !(valid >> (rr >> 4) & 1)) *at_row(rr) = make_uint4(0, 0, 0, 0);
                            else bad |= not_finite(w[n], EXP);
                        }
                    }
                    if (__any_sync(0xffffffffu, bad)) {  // (rarely)
#pragma unroll 1
                        for (int r = max(0, max(by_all, first) - key0) + r0; r < min(BN, end - key0); r += AT_ONCE) {
                            const uint4 w = *at_row(r);
                            if (!not_finite(w, EXP) || !(valid >> (r >> 4) & 1)) continue;
                            *at_row(r) = make_uint4(finite(w.x, EXP), finite(w.y, EXP), finite(w.z, EXP), finite(w.w, EXP));
                            atomicOr(&sm.flagged[(j - edge0) & (EDGES - 1)][r >> 5], 1u << (r & 31));
                        }
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.v_ready[vs]);
            }
            all_of(9, EVERYONE, true);
        }
    } else {
        regs_inc<REGS_SOFTMAX>();
        // ---------------------------------------------------- softmax of slot t, half of each tile's keys and of O's columns
        const int t = warp >> 3, half = warp >> 2 & 1, quarter = warp & 3, r = quarter * 32 + lane, qt = two ? t : 0;
        const int row = row0 + qt * BM + r, mine = two ? n_tiles : (n_tiles - t + 1) / 2;
        const int pair = 1 + t * 4 + quarter;  // the barrier of a row's two threads
        const bool live = row < rows;
        const int i = live ? row / group : 0;
        const size_t in_token = (size_t)(h * group + (live ? row - i * group : 0)) * D;
        const uint32_t live_rows = __ballot_sync(0xffffffffu, live);
        {
            // queries: whole rows, a lane four elements; the warps that have a quarter's rows share them out
            constexpr int LANES = D / 4, AT_ONCE = 32 / LANES, BATCH = (RAW ? 16 : 8) / AT_ONCE;  // loads on their way
            const T* q = static_cast<const T*>(p.q.data) + z + b * p.q.bs + lane % LANES * 4;
            const size_t q_off = i * p.q.ts + in_token;
            const int n_lo = two ? half * 16 : (t * 2 + half) * 8, n_hi = n_lo + (two ? 16 : 8);
#pragma unroll 1
            for (int n0 = n_lo; n0 < n_hi; n0 += BATCH * AT_ONCE) {
                Four<T> xs[BATCH];
                size_t off[BATCH];
#pragma unroll
                for (int c = 0; c < BATCH; c++) off[c] = __shfl_sync(0xffffffffu, q_off, min(n0 + c * AT_ONCE, n_hi - AT_ONCE) + lane / LANES);
                if (vec & 1) {  // (a row behind the last one: the first token's)
#pragma unroll
                    for (int c = 0; c < BATCH; c++) xs[c] = load_four(q + off[c], true);
                } else {
#pragma unroll
                    for (int c = 0; c < BATCH; c++) xs[c] = load_four(q + off[c], false);
                }
#pragma unroll
                for (int c = 0; c < BATCH; c++) {
                    if (n0 + c * AT_ONCE >= n_hi) break;
                    const int rr = n0 + c * AT_ONCE + lane / LANES, qr = quarter * 32 + rr, e = lane % LANES * 4;
                    const bool is_live = live_rows >> rr & 1;
                    uint2 w[P];
                    if constexpr (RAW) {
                        w[0] = is_live ? xs[c].w : make_uint2(0, 0);
                        if (e == 0) sm.part[qt][0][qr] = scale;
                    } else {
                        float4 x = value_of(xs[c]);
                        if (!is_live) x = make_float4(0.f, 0.f, 0.f, 0.f);
                        uint32_t top = max(max(__float_as_uint(fabsf(x.x)), __float_as_uint(fabsf(x.y))),
                                           max(__float_as_uint(fabsf(x.z)), __float_as_uint(fabsf(x.w))));
                        top = __reduce_max_sync(LANES == 32 ? 0xffffffffu : lane < 16 ? 0xffffu : 0xffff0000u, top);
                        float p2, inv;
                        power_of(__uint_as_float(top), p2, inv);
                        if (e == 0) sm.part[qt][0][qr] = p2 * scale;
                        uint32_t a[P], d[P];
                        pieces_of<P>(x.x * inv, x.y * inv, a);
                        pieces_of<P>(x.z * inv, x.w * inv, d);
#pragma unroll
                        for (int k = 0; k < P; k++) w[k] = make_uint2(a[k], d[k]);
                    }
#pragma unroll
                    for (int k = 0; k < P; k++)
                        *reinterpret_cast<uint2*>(sm.q[qt][k][e / 64] + qr * 128 + (((e % 64 / 8) ^ (qr & 7)) << 4) + e / 4 % 2 * 8) = w[k];
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.q_full[qt]);
            __syncwarp();
        }
        const auto meet = [&] { return two ? all_of(pair, 64, true) : all_of(10, SOFTMAX, true); };
        meet();
        const float unit = sm.part[qt][0][r];  // of the row's scores
        bool ok = meet();

        constexpr int KEYS = BN / 2, COLS = D / 2;                                    // the thread's
        const int lim = live ? at.past + i + 1 : 0;                                   // slots below it may be seen
        const int by_slot = tree ? at.past : at.past + (row0 + qt * BM) / group + 1;  // by all of the slot's rows
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const uint32_t s_addr = tmem + lanes + s_col(t) + half * KEYS, o_addr = tmem + lanes + o_col<D>(t) + half * COLS;
        const uint32_t p_addr = tmem + lanes + p_col<D, P>(t) + half * (KEYS / 2 * P);
        // which of 64 slots from key0 on the row sees, where pages are (a bit for each 16)
        const auto mask_of = [&](int key0, uint32_t valid, uint32_t (&m)[2]) {
            const int upto = tree ? min(lim, at.past) : lim;
            m[0] = below(upto - key0);
            m[1] = below(upto - key0 - 32);
            if (tree && live)
                for (int a = i; a >= 0; a = sm.parent[a]) {
                    const int off = at.past + a - key0;
                    if (off >> 5 == 0) m[0] |= 1u << off;
                    if (off >> 5 == 1) m[1] |= 1u << (off & 31);
                }
            m[0] &= ~below(first - key0) & ((valid & 1 ? 0xffffu : 0u) | (valid & 2 ? 0xffff0000u : 0u));
            m[1] &= ~below(first - key0 - 32) & ((valid & 4 ? 0xffffu : 0u) | (valid & 8 ? 0xffff0000u : 0u));
        };
        float m = -INFINITY, l = 0.f;
        float acc[P == 2 ? COLS : 1];  // two pieces: the row's O
#pragma unroll
        for (int e = 0; e < (P == 2 ? COLS : 1); e++) acc[e] = 0.f;
        const auto add_tile = [&] {
            if constexpr (P == 2) {
#pragma unroll
                for (int c = 0; c < COLS; c += 16) {
                    uint32_t o[16];
                    tmem_ld16(o_addr + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[c + e] += __uint_as_float(o[e]);
                }
            }
        };
        for (int it = 0; ok && it < mine; it++) {
            const int j = two ? it : 2 * it + t, key0 = key_lo + j * BN;
            // slot 1 starts a softmax behind slot 0, so that the one's exponentials run during the other's products
            if (!TURNS<D, P> && t == 1 && it == 0) ok = mbar_wait_warp(&sm.started, 0, err);
            ok = ok && mbar_wait_warp(&sm.s_full[t], it & 1, err);
            tc_fence_after();
            const uint32_t valid = sm.valid[j & 3];
            const bool masked = key0 + BN > by_slot || key0 < first || valid != 0xffu;
            uint32_t seen[2];
            if (masked) mask_of(key0 + half * KEYS, valid >> half * 4, seen);
            __syncwarp();  // (rows have different numbers of ancestors)
            float top = -INFINITY;
            uint32_t s[P == 1 ? KEYS : 16];
            if constexpr (P == 1) {
                tmem_ld64(s_addr, s);
                tmem_ld_wait();
                if (masked) {
#pragma unroll
                    for (int e = 0; e < KEYS; e++)
                        if (!(seen[e / 32] >> (e % 32) & 1)) s[e] = __float_as_uint(-INFINITY);
                }
                float mx[4];
#pragma unroll
                for (int k = 0; k < 4; k++) mx[k] = fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 4]));
#pragma unroll
                for (int e = 8; e < KEYS; e += 8)
#pragma unroll
                    for (int k = 0; k < 4; k++) mx[k] = fmax3(mx[k], __uint_as_float(s[e + k]), __uint_as_float(s[e + 4 + k]));
                top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            } else {
                if (it > 0) add_tile();
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < KEYS; c += 16) {
                    tmem_ld16(s_addr + c, s);
                    tmem_ld_wait();
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (!(seen[c / 32] >> (c % 32 + e) & 1)) s[e] = __float_as_uint(-INFINITY);
                    }
#pragma unroll
                    for (int e = 0; e < 16; e += 8)
#pragma unroll
                        for (int k = 0; k < 4; k++) mx[k] = fmax3(mx[k], __uint_as_float(s[e + k]), __uint_as_float(s[e + 4 + k]));
                }
                top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            }
            sm.part[t][half][r] = top;
            ok = all_of(pair, 64, ok);
            if (!ok) break;  // both threads know
            top = fmaxf(top, sm.part[t][half ^ 1][r]) * unit;
            if (EARLY<D, P>) {  // S has been read (and the other thread's maximum)
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.s_free[t]);
                __syncwarp();  // what follows is for whole warps (.aligned)
            }
            const bool grow = top > m + STALE;  // from nothing, too
            const float was = m;
            if (grow) m = top;
            const float base = m == -INFINITY ? 0.f : m, alpha = grow ? exp2_approx(was - base) : 1.f;
            l *= alpha;
            // the last PV is through before O is rescaled or P overwritten (without room beside S, S waited for it)
            if (EARLY<D, P> && it > 0) {
                ok = mbar_wait_warp(&sm.pv_done[t], (it - 1) & 1, err);
                tc_fence_after();
            }
            if (it > 0 && __any_sync(0xffffffffu, grow)) {
                if constexpr (P == 2) {
#pragma unroll
                    for (int e = 0; e < COLS; e++) acc[e] *= alpha;
                } else {
#pragma unroll
                    for (int c = 0; c < COLS; c += 32) {
                        uint32_t o[32];
                        tmem_ld32(o_addr + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                        tmem_st32(o_addr + c, o);
                    }
                }
            }
            // (a slot's last turn may be one that the other, with a tile less, does not wait for)
            if (TURNS<D, P> && (t == 1 || it > 0)) ok = mbar_wait_warp(&sm.turn[t], (t == 0 ? it - 1 : it) & 1, err) && ok;
            const float2 u2 = make_float2(unit, unit), nb = make_float2(SHIFT - base, SHIFT - base);
            float2 sum[2] = {};
            if constexpr (P == 1) {
                uint32_t w[KEYS / 2];
#pragma unroll
                for (int e = 0; e < KEYS / 2; e++) {
                    float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), u2, nb);
                    x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                    if constexpr (RAW) {
                        const __nv_bfloat162 y = __floats2bfloat162_rn(x.x, x.y);
                        w[e] = *reinterpret_cast<const uint32_t*>(&y);
                        x = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
                    } else {
                        uint32_t one[1];
                        pieces_of<1>(x.x, x.y, one);
                        w[e] = one[0];
                    }
                    sum[e & 1] = __fadd2_rn(sum[e & 1], x);
                }
                if constexpr (SHARED<D, P>) {
                    uint8_t* to = sm.p[t][half] + r * 128;
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        *reinterpret_cast<uint4*>(to + ((u ^ (r & 7)) << 4)) = make_uint4(w[u * 4], w[u * 4 + 1], w[u * 4 + 2], w[u * 4 + 3]);
                    fence_proxy_async_smem();
                } else {
                    tmem_st32(p_addr, w);
                }
            } else {
#pragma unroll
                for (int c = 0; c < KEYS; c += 16) {
                    uint32_t w[8][P];
                    tmem_ld16(s_addr + c, s);
                    tmem_ld_wait();
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 16; e++)
                            if (!(seen[c / 32] >> (c % 32 + e) & 1)) s[e] = __float_as_uint(-INFINITY);
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        float2 x = __ffma2_rn(make_float2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), u2, nb);
                        x = make_float2(exp2_approx(x.x), exp2_approx(x.y));
                        sum[e & 1] = __fadd2_rn(sum[e & 1], x);
                        pieces_of<P>(x.x, x.y, w[e]);
                    }
                    // over the same 16 keys' scores
#pragma unroll
                    for (int k = 0; k < P; k++) {
                        uint32_t o[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) o[e] = w[e][k];
                        tmem_st8(p_addr + c + k * 8, o);
                    }
                }
            }
            if (TURNS<D, P>) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.turn[t ^ 1]);
                __syncwarp();
            }
            const float2 s2 = __fadd2_rn(sum[0], sum[1]);
            l += s2.x + s2.y;
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.p_full[t]);
            __syncwarp();
        }
        if (ok && mine > 0) ok = mbar_wait_warp(&sm.pv_done[t], (mine - 1) & 1, err);
        tc_fence_after();
        if (P == 2 && mine > 0) add_tile();
        // both slots and the last warp are through: the rings are free, and every flag is set
        ok = all_of(9, EVERYONE, ok);
        sm.part[t][half][r] = l;
        ok = all_of(pair, 64, ok);
        l += sm.part[t][half ^ 1][r];
        float w_self = 1.f, w_other = 0.f;
        float* swap = reinterpret_cast<float*>(S::KS == 2 ? sm.k[0][0] : sm.v[0][0]);  // two buffers: [slot][half][piece of 4 columns][row][4]
        // columns that the thread ends: its own half, or a half of that, the other slot's thread the other one
        const int c_lo = two ? 0 : t * (COLS / 2), c_hi = two ? COLS : c_lo + COLS / 2;
        const auto columns = [&](int c, float (&o)[16]) {  // 16 of the thread's own O
            if constexpr (P == 2) {
#pragma unroll
                for (int k = 0; k < COLS; k += 16) {
                    if (k == c) {
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = acc[k + e];
                    }
                }
            } else {
                uint32_t x[16] = {};
                if (mine > 0) {
                    tmem_ld16(o_addr + c, x);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 16; e++) o[e] = __uint_as_float(x[e]);
            }
        };
        if (!two) {
            float2* ml = reinterpret_cast<float2*>(S::KS == 2 ? sm.v[0][0] : sm.k[0][0]);
            if (half == 0) ml[t * BM + r] = make_float2(m, l);
#pragma unroll 1
            for (int c = 0; c < COLS / 2; c += 16) {
                float o[16];
                columns((t ^ 1) * (COLS / 2) + c, o);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    *reinterpret_cast<float4*>(swap + (((t * 2 + half) * (D / 16) + c / 4 + u) * BM + r) * 4) =
                        make_float4(o[u * 4], o[u * 4 + 1], o[u * 4 + 2], o[u * 4 + 3]);
            }
            ok = all_of(10, SOFTMAX, ok);
            const float2 x = ml[(t ^ 1) * BM + r];
            const float most = fmaxf(m, x.x), base = most == -INFINITY ? 0.f : most;
            w_self = exp2_approx(m - base);
            w_other = exp2_approx(x.x - base);
            l = l * w_self + x.y * w_other;
            m = most;
        }
        const float f = splits > 1 ? 1.f : l == 0.f ? 0.f : 1.f / l;
        T* out = static_cast<T*>(const_cast<void*>(p.out.data)) + z + b * p.out.bs + half * COLS;
        const size_t out_off = i * p.out.ts + in_token;
        float* ws = p.ws + z + (((size_t)bh * gridDim.x + blockIdx.x) * 2 * BM + qt * BM + quarter * 32) * (D + 4) + 4 + half * COLS;
        // 16 of the thread's columns, ended
        const auto ended = [&](int k, float (&o)[16]) {
            columns(k, o);
            if (!two) {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const float4 x = *reinterpret_cast<const float4*>(swap + ((((t ^ 1) * 2 + half) * (D / 16) + (k - c_lo) / 4 + u) * BM + r) * 4);
                    o[u * 4] = o[u * 4] * w_self + x.x * w_other;
                    o[u * 4 + 1] = o[u * 4 + 1] * w_self + x.y * w_other;
                    o[u * 4 + 2] = o[u * 4 + 2] * w_self + x.z * w_other;
                    o[u * 4 + 3] = o[u * 4 + 3] * w_self + x.w * w_other;
                }
            }
#pragma unroll
            for (int e = 0; e < 16; e++) o[e] *= f;
        };
        if (splits > 1) {
            // the row's part of the keys' cuts, 16 columns at a time: 4 lanes write 64 consecutive bytes of a row
            uint8_t* stage = &sm.q[0][0][0][0] + warp * 2048;
#pragma unroll 1
            for (int k = c_lo; k < c_hi; k += 16) {
                float o[16];
                ended(k, o);
#pragma unroll
                for (int u = 0; u < 4; u++)
                    *reinterpret_cast<float4*>(stage + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) = make_float4(o[u * 4], o[u * 4 + 1], o[u * 4 + 2], o[u * 4 + 3]);
                __syncwarp();
#pragma unroll
                for (int n = 0; n < 32; n += 8) {
                    const int rr = n + lane / 4, u = lane & 3;
                    const float4 y = *reinterpret_cast<const float4*>(stage + rr * 64 + ((u ^ (rr >> 1 & 3)) << 4));
                    if (ok && (live_rows >> rr & 1)) *reinterpret_cast<float4*>(ws + rr * (D + 4) + k + u * 4) = y;
                }
                __syncwarp();
            }
        } else {
            // the row's outputs, all of the thread's columns through the warp's part of the queries' shared memory, so that
            // neighbouring lanes write a row's consecutive bytes
            // (f32 rows in one piece reach into the values' buffers, but not where those pass sums on)
            const int n_u = (c_hi - c_lo) * (int)sizeof(T) / 16;  // 16-byte pieces of a row, a power of two
            uint8_t* stage = &sm.q[0][0][0][0] + warp * (32 * 16 * n_u);
            const auto piece = [&](int rr, int u) { return reinterpret_cast<uint4*>(stage + (rr * n_u + (u ^ (rr & (n_u - 1) & 7))) * 16); };
#pragma unroll 1
            for (int k = c_lo; k < c_hi; k += 16) {
                float o[16];
                ended(k, o);
#pragma unroll
                for (int u = 0; u < (int)sizeof(T); u++) {  // 16 columns are that many pieces
                    uint4 y;
                    if constexpr (RAW) {
                        __nv_bfloat162 h2[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) h2[e] = __floats2bfloat162_rn(o[(u % 2) * 8 + 2 * e], o[(u % 2) * 8 + 2 * e + 1]);
                        y = *reinterpret_cast<const uint4*>(h2);
                    } else {
                        y = make_uint4(__float_as_uint(o[u * 4]), __float_as_uint(o[u * 4 + 1]), __float_as_uint(o[u * 4 + 2]), __float_as_uint(o[u * 4 + 3]));
                    }
                    *piece(lane, (k - c_lo) * (int)sizeof(T) / 16 + u) = y;
                }
            }
            __syncwarp();
            for (int e = lane; e < 32 * n_u; e += 32) {
                const int rr = e / n_u, u = e & (n_u - 1);
                const uint4 y = *piece(rr, u);
                T* to = out + __shfl_sync(0xffffffffu, out_off, rr) + c_lo + u * (16 / (int)sizeof(T));
                if (!ok || !(live_rows >> rr & 1)) continue;
                if (vec & 2) {
                    *reinterpret_cast<uint4*>(to) = y;
                } else {
                    const T* x = reinterpret_cast<const T*>(&y);
#pragma unroll
                    for (int c = 0; c < 16 / (int)sizeof(T); c++) to[c] = x[c];
                }
            }
            __syncwarp();
        }
        if (splits > 1 && live && ok && half == 0 && (two || t == 0)) *reinterpret_cast<float2*>(ws + lane * (D + 4) - 4) = make_float2(m, l);
        // what was taken out of the values comes in where a row sees it
        bool flagged = false;
#pragma unroll
        for (int e = 0; e < EDGES * (BN / 32); e++) flagged |= sm.flagged[e / (BN / 32)][e % (BN / 32)] != 0;
        if (flagged && live && ok) {
#pragma unroll 1
            for (int n = 0; n < EDGES * 2; n++) {
                const int key0 = key_lo + edge0 * BN + n * KEYS;
                uint32_t seen[2];
                mask_of(key0, 0xfu, seen);
#pragma unroll 1
                for (int e = 0; e < KEYS; e++) {
                    if (!(sm.flagged[n / 2][n % 2 * 2 + e / 32] & (e < 32 ? seen[0] : seen[1]) & 1u << (e & 31))) continue;
                    const H* v = static_cast<const H*>(p.c.v) + row_at(p.c, max(0, page_of(p.c, b, key0 + e)), h, key0 + e) + half * COLS + z;
#pragma unroll 1
                    for (int c = c_lo; c < c_hi; c++) {
                        const float y = paged::up(v[c]);
                        if (fabsf(y) < INFINITY) continue;
                        if (splits > 1) ws[lane * (D + 4) + c] += y;
                        else paged::add(out[out_off + c], y);
                    }
                }
            }
        }
        tc_fence_before();
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == ISSUER) {
        tc_fence_after();
        tmem_dealloc(tmem, TMEM_COLS);
    }
}

// A pool side as [page][head * page + row][d], in boxes of up to 128 rows of 64 elements.
bool map_of(CUtensorMap* map, const void* data, const Paged& c, bool bf16) {
    const EncodeTiledFn encode = encode_tiled_fn();
    if (!encode) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)c.d, (cuuint64_t)c.n_head_kv << c.log_page, (cuuint64_t)c.n_pages};
    const cuuint64_t strides[2] = {(cuuint64_t)c.d * 2, (cuuint64_t)c.ps * 2};
    const cuuint32_t box[3] = {64, 1u << std::min(c.log_page, 7), 1}, step[3] = {1, 1, 1};
    return encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(data), dims, strides,
                  box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D, int P>
int launch(const PagedAttn& p, int splits, cudaStream_t st) {
    const auto kern = paged_chunk_kernel<T, D, P>;
    constexpr int smem = sizeof(Smem<D, P>);
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    static std::atomic<uint64_t> done{0};
    if (allow_smem(done, (const void*)kern, smem) != cudaSuccess) return -1;
    CUtensorMap k, v;
    if (!map_of(&k, p.c.k, p.c, sizeof(T) == 2) || !map_of(&v, p.c.v, p.c, sizeof(T) == 2)) return -1;
    const int rows = p.s.n * (p.n_head / p.c.n_head_kv), tiles = (rows + PAGED_CHUNK_ROWS - 1) / PAGED_CHUNK_ROWS;
    const float scale = (float)(1.0 / sqrt((double)D)) * kLog2e;
    const int vec = (wide(p.q, sizeof(T), 4 * sizeof(T)) ? 1 : 0) | (wide(p.out, sizeof(T), 16) ? 2 : 0);
    return launch_chained_smem(kern, dim3((unsigned)(tiles * splits), (unsigned)(p.s.n_batch * p.c.n_head_kv)), dim3(THREADS),
                               smem, st, p, k, v, splits, vec, scale) == cudaSuccess
               ? 0
               : -1;
}

}  // namespace

int paged_chunk_launch(const PagedAttn& p, int type, int pieces, int splits, cudaStream_t st) {
    static_assert(PAGED_CHUNK_ROWS == 2 * BM && PAGED_CHUNK_KEYS == BN, "the plan's tiles are the kernel's");
    if (type == TYPE_BF16) return p.c.d == 64 ? launch<__nv_bfloat16, 64, 1>(p, splits, st) : launch<__nv_bfloat16, 128, 1>(p, splits, st);
    if (pieces == 1) return p.c.d == 64 ? launch<float, 64, 1>(p, splits, st) : launch<float, 128, 1>(p, splits, st);
    return p.c.d == 64 ? launch<float, 64, 2>(p, splits, st) : launch<float, 128, 2>(p, splits, st);
}

}  // namespace zwg
