// Attention of a ragged batch of chunks of new tokens over a paged KV cache:
// how the work is cut, the launches, and the merge of key splits.
//
// Token i of a chunk of n, in a sequence of L cached tokens (the chunk's own
// included), sees the keys j < L - n + i + 1 (causal) or j < L:
//   o = sum_j softmax_j(scale q.k_j) v_j,  and 0 where it sees none.
// Where the tiles of query rows alone would not fill the GPU, the key axis is
// cut into splits of equal length; each split leaves its unnormalised output,
// row maximum and sum in fp32, and paged_combine_kernel merges them in split
// order (the same bits for the same call, whatever finished first).
#include <math.h>

#include "paged.cuh"
#include "paged_simt.cuh"

namespace qv {

int paged_cache_check(const qv_paged_cache* c);
int paged_shift(int page);

int paged_tc_launch(const PagedArgs& a, int dt, int D, bool q8, int64_t tiles, cudaStream_t s);
int paged_few_launch(const PagedArgs& a, int dt, int D, bool q8, bool wide, cudaStream_t s);

constexpr int PC_THREADS = 256;

// W warps per (token, query head) row, 8 / W rows per block: one where there are
// rows enough to fill the GPU, otherwise eight, which take a row's splits in
// turn and join in shared memory.  Lane i holds D / 32 columns of the row.
template <int DT, int D, int W>
__global__ void __launch_bounds__(PC_THREADS) paged_combine_kernel(const PagedArgs a) {
    constexpr int E = D / 32;
    __shared__ float s_o[W > 1 ? W : 1][W > 1 ? D : 1], s_l[8], s_m[8];
    asm volatile("griddepcontrol.wait;" ::: "memory");   // launched while the splits still run
    const int Hq = a.H * a.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (8 / W) + (W == 1 ? warp : 0);
    if (row >= (int64_t)a.total_q * Hq) return;
    const int t = (int)(row / Hq);
    const int b = paged_find_token(a.cu_q, a.B, t);
    const PagedSeq s = paged_seq(a, b);
    const int i = t - s.q0;
    if (i < 0 || i >= s.live || s.kv <= a.chunk) return;   // behind the last sequence, or written by its only split
    const int limit = paged_limit(a, s, i);
    const int n = limit > 0 ? (limit + a.chunk - 1) / a.chunk : 0;
    const size_t step = (size_t)a.total_q * Hq;
    float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    for (int s0 = W == 1 ? 0 : warp; s0 < n; s0 += 4 * W) {
        // four splits' loads at once
        float ms[4], ls[4], v[4][E];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int sp = s0 + u * W;
            ms[u] = -INFINITY;
            ls[u] = 0.f;
            if (sp < n) {
                const size_t p = sp * step + row;
                ms[u] = a.part_ml[2 * p];
                ls[u] = a.part_ml[2 * p + 1];
            }
#pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = sp < n ? a.part_o[(sp * step + row) * D + E * lane + e] : 0.f;
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < 4; ++u) mn = fmaxf(mn, ms[u]);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float f = exp2f(m - base);
        m = mn;
        l *= f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] *= f;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float g = exp2f(ms[u] - base);
            l = fmaf(ls[u], g, l);
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(v[u][e], g, o[e]);
        }
    }
    if constexpr (W == 1) {
        const float inv = l > 0.f ? 1.f / l : l;
#pragma unroll
        for (int e = 0; e < E; ++e) st<DT>(a.out, row * D + E * lane + e, o[e] * inv);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) s_o[warp][E * lane + e] = o[e];
        if (lane == 0) { s_l[warp] = l; s_m[warp] = m; }
        __syncthreads();
        if (threadIdx.x >= D) return;
        float mm = s_m[0];
#pragma unroll
        for (int w = 1; w < W; ++w) mm = fmaxf(mm, s_m[w]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f, x = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = exp2f(s_m[w] - base);
            sum = fmaf(s_l[w], f, sum);
            x = fmaf(s_o[w][threadIdx.x], f, x);
        }
        st<DT>(a.out, row * D + threadIdx.x, sum > 0.f ? x / sum : sum);
    }
}

// ---------------------------------------------------------------- plan
enum PagedKernel { PK_SIMT, PK_TC, PK_FEW };

struct PagedPlan {
    PagedKernel kernel;
    int rows;      // query rows per tile (PK_SIMT)
    bool wide;     // eight warps per block (PK_FEW)
    int64_t tiles; // upper bound of the query tiles of a KV head
    int splits, chunk;
};

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Splits of the key axis that a simple model of the time finds best: a block
// costs `start` us and `key_us` per 128 keys; the lengths are equal (one
// sequence, hardly changed by causality: whole rounds of blocks count) or
// uneven (half of the longest on average, dealt out longest first: the sum over
// the slots, or the longest block); the merge writes and reads every split's
// fp32 rows once.  Measured for the tcgen05 kernel: four 512-token chunks over
// up to 16384 INT8 keys 314 / 330 / 241 / 272 / 237 us with 1 .. 5 splits (3 taken),
// 17 sequences of up to 4000 keys 102 / 158 us with 1 / 2, a 2048-token prompt
// 43 / 85 us with 1 / 2.
static int choose_splits(int64_t blocks, int slots, int max_kv, bool equal, double start, double key_us, double merge_bytes,
                         int least_keys) {
    const int64_t steps = ceil_div(max_kv, 128), most = ceil_div(max_kv, least_keys);
    int best = 1;
    double best_t = 1e30;
    for (int64_t each = steps; each > 0; each = each > 64 ? each * 7 / 8 : each - 1) {   // steps per split
        const int n = (int)ceil_div(steps, each);
        if (n > most || n > 1024) break;
        const double one = start + key_us * each;
        double t = equal ? (double)ceil_div(blocks * n, slots) * one
                         : fmax(one, (double)blocks * (start * n + key_us * steps / 2) / slots);
        if (n > 1) t += 3.0 + 2.0 * n * merge_bytes / 4e6;
        if (t < best_t * 0.98) { best_t = t; best = n; }   // more splits only for a clear gain
    }
    return best;
}

static PagedPlan paged_plan(int dt, int B, int H, int G, int D, int total_q, int max_q, int max_kv) {
    PagedPlan p = {};
    const bool few = (int64_t)max_q * G <= 16;
    p.kernel = dt == QV_F32 ? PK_SIMT : few ? PK_FEW : PK_TC;
    p.rows = few ? 16 : (int64_t)max_q * G <= 64 ? 64 : 128;
    // tokens (times G: rows) per tile; every sequence ends in at most one partial
    // tile, and none is longer than max_q
    const int64_t unit = p.kernel == PK_TC ? 1 : G, per = p.kernel == PK_TC ? 2 * (128 / G) : p.rows;
    p.tiles = total_q * unit / per + (B < total_q ? B : total_q);
    const int64_t by_len = (int64_t)B * ceil_div(max_q * unit, per);
    if (p.tiles > by_len) p.tiles = by_len;
    const bool equal = B == 1 && max_kv >= 2 * max_q;
    const double merge = 4.0 * total_q * G * H * D;
    int n;
    if (p.kernel == PK_FEW) {
        // blocks that fit at once: three per SM (two with more than eight rows).  Few
        // sequences: one round of blocks (two per SM for a single one; a quarter more
        // where lengths differ), of at least 128 keys; many: rounds enough to even out, of at least 1024
        const int64_t per_round = ((int64_t)max_q * G <= 8 ? 3 : 2) * 148, blocks = (int64_t)B * H;
        int64_t most;
        // Short and few: one block of eight warps reads a sequence's head alone, no
        // splits and no merge (measured in paged_few.cu)
        p.wide = blocks <= 148 && max_kv <= (B > 1 ? 1024 : 512);
        if (p.wide) { n = 1; most = 1; }
        else if (2 * blocks <= per_round) { n = (int)((B > 1 ? per_round * 5 / 4 : 2 * 148) / blocks); most = ceil_div(max_kv, 128); }
        else { n = (int)ceil_div(6 * per_round, blocks); most = ceil_div(max_kv, 1024); }
        if (n > most) n = (int)most;
    } else if (p.kernel == PK_TC) {
        n = choose_splits(p.tiles * H, 148, max_kv, equal, 5.0, 2.0 * D / 128, merge, 512);
    } else {
        n = choose_splits(p.tiles * H, p.rows == 128 ? 148 : 2 * 148, max_kv, equal, 5.0, (p.rows == 16 ? 4.0 : p.rows == 64 ? 20.0 : 26.0) * D / 128,
                          merge, 256);
    }
    if (n < 1) n = 1;
    // a multiple of every kernel's tile times its warps
    p.chunk = (int)(ceil_div(ceil_div(max_kv, n), 128) * 128);
    if (p.chunk < 128) p.chunk = 128;
    p.splits = (int)ceil_div(max_kv, p.chunk);
    if (p.splits < 1) p.splits = 1;
    return p;
}

static size_t paged_ws_bytes(const PagedPlan& p, int total_q, int Hq, int D) {
    return p.splits > 1 ? (size_t)p.splits * total_q * Hq * (D + 2) * sizeof(float) : 0;
}

// ---------------------------------------------------------------- launch
template <int D, bool Q8, int BM>
static int simt_launch(const PagedArgs& a, const PagedPlan& p, cudaStream_t s) {
    constexpr size_t bytes = paged_simt_smem<D, BM>();
    static std::atomic<uint64_t> seen{0};
    const cudaError_t e = paged_smem(paged_simt_kernel<D, Q8, BM>, bytes, &seen);
    if (e != cudaSuccess) return set_cuda_error(e);
    paged_simt_kernel<D, Q8, BM><<<dim3((unsigned)p.tiles, a.H, p.splits), PS_THREADS, bytes, s>>>(a);
    return check_launch();
}

template <int D, bool Q8> static int simt_dispatch(const PagedArgs& a, const PagedPlan& p, cudaStream_t s) {
    if (p.rows == 16) return simt_launch<D, Q8, 16>(a, p, s);
    return p.rows == 64 ? simt_launch<D, Q8, 64>(a, p, s) : simt_launch<D, Q8, 128>(a, p, s);
}

template <int DT, int D> static int paged_launch(const PagedArgs& a, const PagedPlan& p, bool q8, cudaStream_t s) {
    int rc;
    if constexpr (DT == QV_F32) rc = q8 ? simt_dispatch<D, true>(a, p, s) : simt_dispatch<D, false>(a, p, s);
    else if (p.kernel == PK_FEW) rc = paged_few_launch(a, DT, D, q8, p.wide, s);
    else rc = paged_tc_launch(a, DT, D, q8, p.tiles, s);
    if (rc != QV_OK || p.splits == 1) return rc;
    const int64_t rows = (int64_t)a.total_q * a.H * a.G;
    const bool many = rows >= 16 * 148;
    const cudaError_t e = launch_pdl(many ? paged_combine_kernel<DT, D, 1> : paged_combine_kernel<DT, D, 8>,
                                     dim3((unsigned)(many ? ceil_div(rows, 8) : rows)), dim3(PC_THREADS), 0, s, a);
    return e == cudaSuccess ? check_launch() : set_cuda_error(e);
}

}  // namespace qv

using namespace qv;

static bool attn_dims_ok(const qv_paged_cache* c, int32_t batch, int32_t q_heads, int32_t total_q, int32_t max_q,
                         int32_t max_kv) {
    if (batch < 0 || total_q < 0 || max_q < 0 || max_kv < 0 || max_kv > 1 << 30 || q_heads <= 0) return false;
    if (c->head_dim != 64 && c->head_dim != 128) return false;
    if (q_heads % c->kv_heads || q_heads / c->kv_heads > 16 || c->kv_heads > 65535) return false;
    return (int64_t)total_q * q_heads <= 0x7fffffff;
}

extern "C" size_t qv_paged_attention_workspace_bytes(const qv_paged_cache* c, int32_t batch, int32_t q_heads,
                                                     int32_t total_q, int32_t max_q, int32_t max_kv) {
    if (paged_cache_check(c) != QV_OK || !attn_dims_ok(c, batch, q_heads, total_q, max_q, max_kv)) return 0;
    if (batch == 0 || total_q == 0 || max_q == 0) return 0;
    return paged_ws_bytes(paged_plan(c->dtype, batch, c->kv_heads, q_heads / c->kv_heads, c->head_dim, total_q, max_q, max_kv), total_q,
                          q_heads, c->head_dim);
}

extern "C" int qv_paged_attention(const qv_paged_cache* c, int32_t batch, int32_t q_heads, const int32_t* block_table,
                                  int32_t max_pages, const int32_t* kv_lens, const int32_t* cu_q, int32_t total_q,
                                  int32_t max_q, int32_t max_kv, const void* q, int64_t q_stride, float scale,
                                  int32_t causal, void* out, void* workspace, size_t workspace_bytes,
                                  qv_stream_t stream) {
    const int rc = paged_cache_check(c);
    if (rc != QV_OK) return rc;
    if (!attn_dims_ok(c, batch, q_heads, total_q, max_q, max_kv)) return QV_EINVAL;
    if (batch == 0 || total_q == 0 || max_q == 0) return QV_OK;
    if (!block_table || max_pages <= 0 || !kv_lens || !cu_q || !q || !out) return QV_EINVAL;
    if ((int64_t)max_kv > (int64_t)max_pages * c->page_size) return QV_EINVAL;
    if (!(scale > 0.f && scale < INFINITY)) return QV_EINVAL;
    const int64_t per16 = 16 / (int64_t)elt_size(c->dtype);
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) || q_stride % per16 ||
        q_stride < (int64_t)q_heads * c->head_dim)
        return QV_EINVAL;
    const int G = q_heads / c->kv_heads;
    const PagedPlan p = paged_plan(c->dtype, batch, c->kv_heads, G, c->head_dim, total_q, max_q, max_kv);
    if (p.tiles * c->kv_heads > 0x7fffffff || (int64_t)batch * c->kv_heads > 0x7fffffff) return QV_EINVAL;
    const size_t need = paged_ws_bytes(p, total_q, q_heads, c->head_dim);
    if (need > workspace_bytes) return QV_ESPACE;
    if (need && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15))) return QV_EINVAL;
    // out may be q where that is contiguous (a block reads the rows that it writes, and no others' heads); nothing else
    // that is written may be read
    const size_t e = elt_size(c->dtype), row = (size_t)q_heads * c->head_dim, sb = pool_scale_bytes(c);
    const Span qs = span(q, ((size_t)(total_q - 1) * q_stride + row) * e), o = span(out, (size_t)total_q * row * e);
    const Span ws = span(workspace, need);
    for (const Span& x : {o, ws})
        if (meets(x, {span(c->k, pool_bytes(c)), span(c->v, pool_bytes(c)), span(c->k_scale, sb), span(c->v_scale, sb),
                      span(block_table, (size_t)batch * max_pages * 4), span(kv_lens, (size_t)batch * 4),
                      span(cu_q, ((size_t)batch + 1) * 4), span(c->err, 4)}))
            return QV_EINVAL;
    if (meets(ws, {qs, o}) || (meets(o, {qs}) && !(o.at == qs.at && o.bytes == qs.bytes))) return QV_EINVAL;
    PagedArgs a = {};
    a.k = c->k; a.v = c->v; a.k_scale = c->k_scale; a.v_scale = c->v_scale; a.err = c->err;
    a.block_table = block_table; a.kv_lens = kv_lens; a.cu_q = cu_q; a.q = q; a.out = out;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + (size_t)p.splits * total_q * q_heads * c->head_dim;
    a.q_stride = q_stride; a.pages = c->pages; a.H = c->kv_heads; a.G = G; a.page_shift = paged_shift(c->page_size);
    a.max_pages = max_pages; a.B = batch; a.total_q = total_q; a.max_q = max_q; a.max_kv = max_kv; a.causal = causal != 0;
    a.splits = p.splits; a.chunk = p.chunk;
    a.scale_log2 = (float)((double)scale * 1.4426950408889634);
    const bool q8 = c->bits == 8;
    cudaStream_t s = (cudaStream_t)stream;
    if (c->head_dim == 128) {
        if (c->dtype == QV_F32) return paged_launch<QV_F32, 128>(a, p, q8, s);
        if (c->dtype == QV_BF16) return paged_launch<QV_BF16, 128>(a, p, q8, s);
        return paged_launch<QV_F16, 128>(a, p, q8, s);
    }
    if (c->dtype == QV_F32) return paged_launch<QV_F32, 64>(a, p, q8, s);
    if (c->dtype == QV_BF16) return paged_launch<QV_BF16, 64>(a, p, q8, s);
    return paged_launch<QV_F16, 64>(a, p, q8, s);
}
