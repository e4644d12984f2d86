// A key/value cache in pages (zwg_paged): the append that rotates keys and queries on the way
// (zwg_paged_append), and what follows a tree of drafted tokens: which of them the model agrees with
// (zwg_tree_accept), and their rows moved to where the sequence goes on (zwg_paged_keep).
#include <algorithm>

#include "chain.cuh"
#include "paged.cuh"

namespace zwg {
namespace {

using namespace paged;

template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec {
    T e[N];
};

// f32 values rounded to elements of a type, two at a time where it has 16 bits.
ZWG_DEV uint32_t pair_of(float a, float b, __half) {
    const __half2 x = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
}
ZWG_DEV uint32_t pair_of(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&x);
}
template <typename H, int N>
ZWG_DEV void rounded(const float (&a)[N], Vec<H, N>& o) {
    if constexpr (sizeof(H) == 4) {
#pragma unroll
        for (int j = 0; j < N; j++) o.e[j] = a[j];
    } else if constexpr (N == 1) {
        o.e[0] = held(a[0], H());
    } else {
#pragma unroll
        for (int j = 0; j < N; j += 2) reinterpret_cast<uint32_t*>(&o)[j / 2] = pair_of(a[j], a[j + 1], H());
    }
}

// ---- append ------------------------------------------------------------------------------
//
//   a' = a cos - b sin,  b' = a sin + b cos,  (a, b) = (x[i], x[i + rot/2]) or (x[2i], x[2i + 1])
//
// of q and k at position past + i, or past + (token i's ancestors in the call) in a tree; the f32 operations
// one by one, as rope_kernel, so that both give the same bits. k' and v are rounded once to the cache's type.
// Bound by memory: every row in once, out once. A thread takes a piece of 8 elements (or, where pairs are
// halves, both sides' pieces) of up to eight (four) of a token's q, k and v heads: they share its table entries, and all
// its loads are on their way before the first is used. Rows that are not aligned for that, and rotated parts
// that do not divide into it, go four elements or one at a time. In a graph: 64 x 256 tokens, 12 + 2 heads of d 128, bf16,
// interleaved, 24.9 us (134 MB in and out: 5.4 TB/s; issue slots 62 % busy); 64 steps of a token, f32, 2.8 us.
constexpr int heads_of(bool one) { return one ? 8 : 4; }  // of a thread: eight pieces on their way

// N: elements a thread moves at a time (8, 4, or 1). Threads: (piece, group of heads, token).
template <typename T, int N, bool INTER>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppend p) {
    chain_release();
    const int z = chain_wait();
    using H = typename Held<T>::type;
    using V = Vec<T, N>;
    using W = Vec<H, N>;
    constexpr bool ONE = INTER && N > 1;  // a piece holds both sides of its pairs
    constexpr int C = ONE ? N / 2 : N;    // pairs of a piece
    constexpr int HEADS = heads_of(ONE);
    using F = Vec<float, C>;
    __shared__ int parent[MOST_TREE];
    const bool lead = threadIdx.x == 0 && threadIdx.y == 0 && threadIdx.z == 0 && blockIdx.x == 0 && blockIdx.z == 0;
    const int b = blockIdx.y, i = blockIdx.x * blockDim.z + threadIdx.z, piece = threadIdx.x;
    const Place at = place_of(p.s, b, min(p.c.room, p.rope.cos ? p.rope.n_ctx : p.c.room), lead ? p.err : nullptr);
    if (p.tree.parent && !read_tree(p.tree, b, at.count, z, parent)) {
        if (lead) set_error(p.err, kErrBounds);
        return;
    }
    if (i >= at.count) return;
    const int slot = at.past + i;
    int pos = slot;
    if (p.tree.parent) {
        pos = at.past;
        for (int a = parent[i]; a >= 0; a = parent[a]) pos++;
    }
    const int rot = p.rope.cos ? p.rope.rot : 0, half = rot / 2;
    const int turned = ONE ? rot / N : half / N;  // pieces of a head that are rotated; the others stay
    const bool turn = piece < turned;
    int ea, eb;  // where the two sides of a pair are (a piece that holds both: one place)
    if (!turn) ea = eb = rot + (piece - turned) * N;
    else if (ONE) ea = eb = piece * N;
    else if (INTER) ea = 2 * piece, eb = ea + 1;
    else ea = piece * N, eb = ea + half;
    const int kv = p.c.n_head_kv, h0 = (blockIdx.z * blockDim.y + threadIdx.y) * HEADS, heads = min(HEADS, p.n_head + 2 * kv - h0), d = p.c.d;
    const T* q = static_cast<const T*>(p.q.data) + (b * p.q.bs + i * p.q.ts + z);
    const T* k = static_cast<const T*>(p.k.data) + (b * p.k.bs + i * p.k.ts + z);
    const T* v = static_cast<const T*>(p.v.data) + (b * p.v.bs + i * p.v.ts + z);
    V va[HEADS], vb[HEADS];
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        if (u >= heads) break;
        const int h = h0 + u - p.n_head;
        const T* x = h < 0 ? q + (h + p.n_head) * d : h < kv ? k + h * d : v + (h - kv) * d;
        va[u] = *reinterpret_cast<const V*>(x + ea);
        if (!ONE && turn) vb[u] = *reinterpret_cast<const V*>(x + eb);
    }
    F co, si;
    if (turn) {
        const size_t t = (size_t)pos * half + piece * C;
        co = *reinterpret_cast<const F*>(p.rope.cos + t + z);
        si = *reinterpret_cast<const F*>(p.rope.sin + t + z);
    }
    const int page = page_of(p.c, b, slot + z);
    if (page < 0 && piece == 0 && threadIdx.y == 0) set_error(p.err, kErrBounds);
    T* qo = static_cast<T*>(const_cast<void*>(p.q_out.data)) + (b * p.q_out.bs + i * p.q_out.ts + z);
    const size_t in_k = row_at(p.c, max(page, 0), 0, slot) + z;
    H* const ko = static_cast<H*>(p.c.k) + in_k;
    H* const vo = static_cast<H*>(p.c.v) + in_k;
    const size_t hs = (size_t)d << p.c.log_page;  // from head to head in a page
#pragma unroll
    for (int u = 0; u < HEADS; u++) {
        if (u >= heads) break;
        const int h = h0 + u - p.n_head;
        const bool turns = turn && h < kv;
        float a[N], c[N];
        if (turns || sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < N; j++) {
                a[j] = up(va[u].e[j]);
                c[j] = ONE ? 0.f : up(vb[u].e[j]);
            }
        }
        if (turns) {
#pragma unroll
            for (int j = 0; j < C; j++) {
                float& x = ONE ? a[(2 * j) % N] : a[j];
                float& y = ONE ? a[(2 * j + 1) % N] : c[j];
                const float x0 = x, y0 = y;
                x = __fsub_rn(__fmul_rn(x0, co.e[j]), __fmul_rn(y0, si.e[j]));
                y = __fadd_rn(__fmul_rn(x0, si.e[j]), __fmul_rn(y0, co.e[j]));
            }
            rounded(a, va[u]);
            if (!ONE) rounded(c, vb[u]);
        }
        if (h < 0) {
            T* y = qo + (h + p.n_head) * d;
            *reinterpret_cast<V*>(y + ea) = va[u];
            if (!ONE && turn) *reinterpret_cast<V*>(y + eb) = vb[u];
        } else if (page >= 0) {
            H* y = h < kv ? ko + h * hs : vo + (h - kv) * hs;
            W wa, wb;
            if constexpr (sizeof(T) == 4) {
                rounded(a, wa);
                if (!ONE) rounded(c, wb);
            } else {  // as it is, or as it was rounded
                wa = *reinterpret_cast<const W*>(&va[u]);
                if (!ONE) wb = *reinterpret_cast<const W*>(&vb[u]);
            }
            *reinterpret_cast<W*>(y + ea) = wa;
            if (!ONE && turn) *reinterpret_cast<W*>(y + eb) = wb;
        }
    }
}

bool aligned(const Rows& r, size_t elem, size_t bytes) { return ((uintptr_t)r.data | (r.bs * elem) | (r.ts * elem)) % bytes == 0; }

template <typename T, int N>
int append(const PagedAppend& p, cudaStream_t st) {
    const bool inter = p.rope.cos && p.rope.interleaved;
    const int rot = p.rope.cos ? p.rope.rot : 0;
    // a head's pieces: a pair of pieces, or a piece that holds its pairs, counts once
    const int pieces = (inter && N > 1 ? rot / N : rot / 2 / N) + (p.c.d - rot) / N;
    const int heads = heads_of(inter && N > 1), groups = (p.n_head + 2 * p.c.n_head_kv + heads - 1) / heads;
    const int y = std::min(groups, std::max(1, 256 / pieces)), tokens = std::min({std::max(1, 256 / (pieces * y)), p.s.n, 64});
    const dim3 grid((p.s.n + tokens - 1) / tokens, p.s.n_batch, (groups + y - 1) / y);
    return launch_chained(inter ? paged_append_kernel<T, N, true> : paged_append_kernel<T, N, false>, grid,
                          dim3(pieces, y, tokens), st, p) == cudaSuccess
               ? 0
               : -1;
}

// Whether rows and rotated parts divide into pieces of n elements that are aligned to their 16 bytes, or to all of them.
template <typename T>
bool divides(const PagedAppend& p, int n) {
    const size_t bytes = std::min<size_t>(16, n * sizeof(T));
    const int half = p.rope.cos ? p.rope.rot / 2 : 0, pairs = p.rope.interleaved ? n / 2 : n;  // of a piece, and of its table entries
    return aligned(p.q, sizeof(T), bytes) && aligned(p.q_out, sizeof(T), bytes) && aligned(p.k, sizeof(T), bytes) &&
           aligned(p.v, sizeof(T), bytes) && half % pairs == 0 && (((uintptr_t)p.rope.cos | (uintptr_t)p.rope.sin) % std::min(16, pairs * 4)) == 0;
}

template <typename T>
int append_type(const PagedAppend& p, cudaStream_t st) {
    return divides<T>(p, 8) ? append<T, 8>(p, st) : divides<T>(p, 4) ? append<T, 4>(p, st) : append<T, 1>(p, st);
}

// ---- acceptance --------------------------------------------------------------------------
//
// From node 0, whose token is already chosen: the child with the lowest index whose token is what the model
// says after its parent, as long as there is one. A warp takes a sequence: a lane holds every 32nd token and
// its parent, a step is a lane's scan of its own and a minimum over the lanes. Bound by latency: the loads,
// then about 40 cycles and n / 32 compares a step. With the kept rows behind it, in a graph: 4.7 us for one tree of 25
// tokens and 28 caches, 7.1 for 64 trees of 61 and 24 caches.
constexpr int PER_LANE = MOST_TREE / 32;
__global__ void __launch_bounds__(32) tree_accept_kernel(TreeAccept p) {
    chain_release();
    const int z = chain_wait();
    __shared__ int ids[MOST_TREE];
    const int b = blockIdx.x, lane = threadIdx.x, n = p.s.n;
    int count = p.s.count ? __ldcg(p.s.count + b + z) : n;
    bool bad = count < 0 || count > n;
    if (bad) count = 0;
    int parent[PER_LANE], token[PER_LANE];
#pragma unroll
    for (int u = 0; u < PER_LANE; u++) {
        const int i = u * 32 + lane;
        parent[u] = -1;
        token[u] = 0;
        if (i < count) {
            parent[u] = __ldcg(p.tree.parent + b * p.tree.bs + i + z);
            token[u] = __ldcg(p.tokens + (size_t)b * n + i + z);
            ids[i] = __ldcg(p.ids + (size_t)b * n + i + z);
            bad |= parent[u] < -1 || parent[u] >= i;
        }
    }
    if (__any_sync(0xffffffffu, bad)) {
        if (lane == 0) set_error(p.err, kErrBounds);
        count = 0;
    }
    __syncwarp();
    int at = count ? 0 : -1, kept = 0, last = -1;
    int32_t* path = p.path + (size_t)b * n + z;
    while (at >= 0) {
        if (lane == 0) path[kept] = at;
        kept++;
        last = at;
        const int want = ids[at];
        unsigned best = 0xffffffffu;
#pragma unroll
        for (int u = PER_LANE - 1; u >= 0; u--)
            if (u * 32 + lane < count && parent[u] == at && token[u] == want) best = u * 32 + lane;
        at = (int)__reduce_min_sync(0xffffffffu, best);  // none: -1
    }
    for (int i = kept + lane; i < n; i += 32) path[i] = -1;
    if (lane == 0) {
        p.n_path[b + z] = kept;
        p.next[b + z] = last < 0 ? -1 : ids[last];
    }
}

// ---- kept rows ---------------------------------------------------------------------------
//
// Row path[j] of the call to slot past + j, in every cache's K and V. path rises, so path[j] >= j: a thread that
// has the same 16 bytes of every row moves them in the order of j, in batches of loads before their stores, and
// never writes what it reads later. Bound by latency (a path of 8 tokens, 24 caches of 2 heads of d 64: 2 x 2 KB a
// sequence and cache).
constexpr int BATCH = 8;
__global__ void __launch_bounds__(128) paged_keep_kernel(const __grid_constant__ PagedKeep p) {
    chain_release();
    const int z = chain_wait();
    __shared__ long long from[MOST_TREE], to[MOST_TREE];  // rows of head 0, -1: nothing to move
    const int b = blockIdx.y, n = p.s.n;
    const bool lead = blockIdx.x == 0 && blockIdx.z == 0;
    Seqs s = p.s;
    s.count = p.n_path;
    const Place at = place_of(s, b, p.c.room, lead && threadIdx.x == 0 ? p.err : nullptr);
    int bad = 0;
    for (int j = threadIdx.x; j < at.count; j += blockDim.x) {
        const int i = __ldcg(p.path + (size_t)b * n + j + z), before = j ? __ldcg(p.path + (size_t)b * n + j - 1 + z) : -1;
        const bool fits = i > before && i < n && i < p.c.room - at.past;
        bad |= !fits;
        from[j] = to[j] = -1;
        if (fits && i != j) {
            const int a = page_of(p.c, b, at.past + i), c = page_of(p.c, b, at.past + j);
            if (a >= 0 && c >= 0) {
                from[j] = (long long)row_at(p.c, a, 0, at.past + i);
                to[j] = (long long)row_at(p.c, c, 0, at.past + j);
            } else if (lead) {
                set_error(p.err, kErrBounds);
            }
        }
    }
    if (__syncthreads_or(bad)) {
        if (lead && threadIdx.x == 0) set_error(p.err, kErrBounds);
        return;
    }
    const int pieces = p.c.d / 8, e = blockIdx.x * blockDim.x + threadIdx.x;  // (side, head, 16-byte piece)
    if (e >= 2 * p.c.n_head_kv * pieces) return;
    const int side = e / (p.c.n_head_kv * pieces), h = e / pieces % p.c.n_head_kv, piece = e % pieces;
    uint16_t* data = static_cast<uint16_t*>(side ? p.v[blockIdx.z] : p.k[blockIdx.z]) + ((size_t)h << p.c.log_page) * p.c.d + piece * 8 + z;
    for (int j0 = 0; j0 < at.count; j0 += BATCH) {
        uint4 w[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; u++)
            if (j0 + u < at.count && from[j0 + u] >= 0) w[u] = *reinterpret_cast<const uint4*>(data + from[j0 + u]);
#pragma unroll
        for (int u = 0; u < BATCH; u++)
            if (j0 + u < at.count && from[j0 + u] >= 0) *reinterpret_cast<uint4*>(data + to[j0 + u]) = w[u];
    }
}

}  // namespace

int paged_append_launch(const PagedAppend& p, int type, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0) return 0;
    return type == TYPE_BF16 ? append_type<__nv_bfloat16>(p, st) : append_type<float>(p, st);
}

int tree_accept_launch(const TreeAccept& p, cudaStream_t st) {
    if (p.s.n_batch == 0) return 0;
    return launch_chained(tree_accept_kernel, dim3(p.s.n_batch), dim3(32), st, p) == cudaSuccess ? 0 : -1;
}

int paged_keep_launch(const PagedKeep& p, cudaStream_t st) {
    if (p.s.n_batch == 0 || p.s.n == 0 || p.n == 0) return 0;
    const int pieces = 2 * p.c.n_head_kv * p.c.d / 8;
    return launch_chained(paged_keep_kernel, dim3((pieces + 127) / 128, p.s.n_batch, p.n), dim3(128), st, p) == cudaSuccess ? 0 : -1;
}

}  // namespace zwg
