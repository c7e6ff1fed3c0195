// Shared by the paged-cache kernels: 8-element row chunks, the sequence that a
// token or tile belongs to, and the arguments of the attention kernels.
#pragma once

#include <atomic>
#include <initializer_list>

#include "common.cuh"

namespace qv {

// Eight consecutive elements as loaded (16 bytes of a 16-bit type, 32 of fp32).
template <int DT> struct Chunk8 { uint4 u[DT == QV_F32 ? 2 : 1]; };

template <int DT> __device__ __forceinline__ Chunk8<DT> load8(const void* base, size_t elt) {
    Chunk8<DT> c;
    const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const typename Elt<DT>::T*>(base) + elt);
    c.u[0] = p[0];
    if constexpr (DT == QV_F32) c.u[1] = p[1];
    return c;
}

template <int DT> __device__ __forceinline__ void widen8(const Chunk8<DT>& c, float* x) {
    const typename Elt<DT>::T* e = reinterpret_cast<const typename Elt<DT>::T*>(c.u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = Elt<DT>::f(e[i]);
}

template <int DT> __device__ __forceinline__ void store8(void* base, size_t elt, const float* x) {
    Chunk8<DT> c;
    typename Elt<DT>::T* e = reinterpret_cast<typename Elt<DT>::T*>(c.u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = Elt<DT>::t(x[i]);
    uint4* p = reinterpret_cast<uint4*>(reinterpret_cast<typename Elt<DT>::T*>(base) + elt);
    p[0] = c.u[0];
    if constexpr (DT == QV_F32) p[1] = c.u[1];
}

// Eight INT8 codes times their row's scale.
__device__ __forceinline__ void widen8_codes(uint2 u, float scale, float* x) {
    const int8_t* e = reinterpret_cast<const int8_t*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)e[i] * scale;
}

struct PagedArgs {
    const void* k;               // [pages][H][page][D], dtype or int8
    const void* v;
    const float* k_scale;        // [pages][H][page] (int8 pages)
    const float* v_scale;
    int32_t* err;                // may be null
    const int32_t* block_table;  // [B][max_pages]
    const int32_t* kv_lens;      // [B]
    const int32_t* cu_q;         // [B + 1]
    const void* q;               // [total_q][G*H][D], token stride q_stride elements
    void* out;                   // [total_q][G*H][D]
    float* part_o;               // [splits][total_q*G*H][D]
    float* part_ml;              // [splits][total_q*G*H][2]: row maximum (base-2 logits), sum
    int64_t q_stride;
    int pages, H, G, page_shift, max_pages, B, total_q, max_q, max_kv, causal, splits, chunk;
    float scale_log2;            // softmax scale * log2(e)
};

// One sequence of the batch, clamped so that no address leaves its buffer
// whatever the device-side lengths hold.
struct PagedSeq {
    int q0, n, kv;   // first row of the chunk, its tokens, cached tokens (the chunk's own included)
    int live;        // tokens of the chunk that are computed: min(n, max_q)
};
__device__ __forceinline__ PagedSeq paged_seq(const PagedArgs& a, int b) {
    PagedSeq s;
    const int lo = min(max(a.cu_q[b], 0), a.total_q), hi = min(max(a.cu_q[b + 1], 0), a.total_q);
    s.q0 = lo;
    s.n = max(hi - lo, 0);
    const int kv = a.kv_lens[b];
    s.kv = min(max(kv, 0), a.max_kv);
    s.live = min(s.n, a.max_q);
    if ((kv != s.kv || s.live != s.n) && a.err) set_err(a.err, QV_DERR_CAPACITY);
    return s;
}

// Raises the error word where a sequence's rows descend or leave the queries.  Once per launch, by 32 threads t of
// its first block, beside the warp that looks for the tile.
__device__ __forceinline__ void paged_check_rows(const PagedArgs& a, int t) {
    if (!a.err) return;
    for (int b = t; b < a.B; b += 32) {
        const int at = a.cu_q[b], to = a.cu_q[b + 1];
        if (at < 0 || to < at || to > a.total_q) set_err(a.err, QV_DERR_CAPACITY);
    }
}

// Keys that token i of the chunk sees.
__device__ __forceinline__ int paged_limit(const PagedArgs& a, const PagedSeq& s, int i) {
    return a.causal ? min(s.kv, s.kv - s.n + i + 1) : s.kv;
}

// Page that holds a key; an id outside the pool raises the error word and reads page 0.
__device__ __forceinline__ int paged_page(const PagedArgs& a, int b, int key) {
    int p = a.block_table[(size_t)b * a.max_pages + (key >> a.page_shift)];
    if ((unsigned)p >= (unsigned)a.pages) {
        if (a.err) set_err(a.err, QV_DERR_TABLE);
        p = 0;
    }
    return p;
}

// The sequence that holds a block's tile, and the tile within it (-1 past the
// last).  Every chunk of n tokens (up to max_q) is cut into ceil(n *
// rows_per_token / tile_rows) tiles; they are dealt out longest first, so that no
// long one starts last: sequences over half of max_kv, over a quarter, over an
// eighth, the rest, and in each sequence the last tile first (the longest where
// causal).  Called by one full warp: each lane counts a run of sequences.
__device__ __forceinline__ int2 paged_find_tile(const PagedArgs& a, int tile, int rows_per_token, int tile_rows) {
    auto tiles_of = [&](int b) {
        const int lo = min(max(a.cu_q[b], 0), a.total_q), hi = min(max(a.cu_q[b + 1], 0), a.total_q);
        return (int)(((long long)min(max(hi - lo, 0), a.max_q) * rows_per_token + tile_rows - 1) / tile_rows);
    };
    if (a.B == 1) {
        const int n = tiles_of(0);
        return tile < n ? make_int2(0, n - 1 - tile) : make_int2(-1, 0);
    }
    auto class_of = [&](int b) {
        const int kv = a.kv_lens[b];
        return kv > a.max_kv >> 1 ? 0 : kv > a.max_kv >> 2 ? 1 : kv > a.max_kv >> 3 ? 2 : 3;
    };
    const int lane = threadIdx.x & 31;
    const int per = (a.B + 31) / 32, b0 = min(lane * per, a.B), b1 = min(b0 + per, a.B);
    int cnt[4] = {0, 0, 0, 0};
    for (int b = b0; b < b1; ++b) {
        const int n = tiles_of(b), c = class_of(b);
#pragma unroll
        for (int i = 0; i < 4; ++i) cnt[i] += c == i ? n : 0;
    }
    int before = 0;
    int2 hit = make_int2(-1, 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int incl = cnt[i];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        int mine = before + incl - cnt[i];
        if (tile >= mine && tile < mine + cnt[i]) {
            for (int b = b0; b < b1; ++b) {
                if (class_of(b) != i) continue;
                const int n = tiles_of(b);
                if (tile < mine + n) { hit = make_int2(b, mine + n - 1 - tile); break; }
                mine += n;
            }
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
    }
    const int src = __ffs(__ballot_sync(0xffffffffu, hit.x >= 0)) - 1;
    if (src < 0) return make_int2(-1, 0);
    return make_int2(__shfl_sync(0xffffffffu, hit.x, src), __shfl_sync(0xffffffffu, hit.y, src));
}

// A buffer of a call (none: 0 bytes), for the host's check of what may not overlap.
struct Span { uintptr_t at; size_t bytes; };
inline Span span(const void* p, size_t bytes) { return {reinterpret_cast<uintptr_t>(p), p ? bytes : 0}; }
inline bool meets(Span a, std::initializer_list<Span> others) {
    for (const Span& b : others)
        if (a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes) return true;
    return false;
}
// The pool's rows, and its row scales (none without INT8).
inline size_t pool_bytes(const qv_paged_cache* c) {
    return (size_t)c->pages * c->kv_heads * c->page_size * c->head_dim * (c->bits == 8 ? 1 : elt_size(c->dtype));
}
inline size_t pool_scale_bytes(const qv_paged_cache* c) {
    return c->bits == 8 ? (size_t)c->pages * c->kv_heads * c->page_size * sizeof(float) : 0;
}

// Raise a kernel's dynamic shared-memory limit once per device (`seen`: a bit per
// device, one word per kernel), so that later launches make no attribute call.
template <typename K> inline cudaError_t paged_smem(K kernel, size_t bytes, std::atomic<uint64_t>* seen) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (seen->load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && dev < 64) seen->fetch_or(bit, std::memory_order_relaxed);
    return e;
}

// Index of the last entry of the ascending cu[0..B] that is <= t, below B.
__device__ __forceinline__ int paged_find_token(const int32_t* cu, int B, int t) {
    int lo = 0, hi = B;   // cu[lo] <= t, and hi is past it
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid] <= t) lo = mid; else hi = mid;
    }
    return lo;
}

}  // namespace qv
