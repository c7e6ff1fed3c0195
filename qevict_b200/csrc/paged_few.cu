// Paged attention of few query rows (a decode step; a few tokens times the
// heads of a group, up to 16 rows per KV head), bf16 and fp16, pages in the same
// type or INT8.
//
// Bound by HBM: every cached row is read once for at most 16 query rows, two
// orders of magnitude below the tensor cores' balance, so the work is keeping
// loads in flight.  A block takes one KV head of one sequence and a range of its
// keys; each of its warps walks its own tiles of 16 or 32 keys through a
// ring of its own in shared memory (TMA, one elected lane, one mbarrier per
// stage), so that no barrier couples the warps until their states join at the
// end.  Blocks of four warps with 64 KB of rings: three share an SM (two with more
// than eight rows), and one's start and end hide behind the others' loads.  64
// sequences over up to 8192 INT8 tokens: 109 us, 122 us with two blocks and rings of
// three stages instead of two.  Short sequences that a block reads alone take eight
// warps with 192 KB (512 keys 6.1 us, as four splits and their merge take with a
// launch more; 8 uneven sequences of up to 1000 keys 9.2 against 9.5).
//
// Per tile, with warp-level MMA (m16n8k16) and the cached rows as the M side, so
// that up to 8 query rows cost one n-tile and no padding of the conversions:
//   S^T = K Q^T,  P = exp2(S c - m),  l += P,  O^T += V^T P^T
// P^T's operand registers are the accumulators' 8x8 blocks transposed
// (movmatrix).  The reference m is set 2^7 below a maximum and moves only when a
// logit exceeds it by 2^15, so that a tile needs no row maximum across lanes and
// P spans fp16 down to 2^-31 of the largest.  With bf16 pages P is split into two
// bf16 parts (P V is then exact to 2^-17; the tensor pipe is idle anyway).  fp16's P is one
// fp16 number, as precise as the output: outputs are 1.3-1.4 times as far from 64 bits as
// fp32 arithmetic rounded once (bf16: as far).
//
// INT8 rows: the codes become exact fp16 integers in registers and the scales
// stay in fp32,
//   u = S c ks + log2(vs),  P = exp2(u - m),  O += P code,  l += P / vs,
// with P in fp16 whatever the type; bf16 queries become fp16 scaled by a power
// of two of their row's own (off by at most 2^-25 of the row's largest element).
// The contraction over the head's elements may run in any order, and so may the
// rows of O^T: each lane takes 16-byte chunks of codes as the elements of its
// own fragments.
#include <cudaTypedefs.h>
#include <math.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace qv {

constexpr float PF_BELOW = 7.f, PF_LAZY = 15.f;
// 2^-60: a smaller value scale counts as this, a zero row's 0 too.  P carries the
// scale and the sum divides by it, so a zero row of weight 2^-24 still counts (P is
// a normal number) beside value scales up to 2^49 = 2^(126 + 7 - 60 - 24).  fp16's
// own scales are 2^-31 .. 2^9.
constexpr float PF_MIN_SCALE = 8.6736173798840355e-19f;

// W warps: 4, several blocks per SM; 8, one block per SM, for short sequences
// that a block then reads alone, without a merge after it.
template <int D, bool Q8, int W> struct PfCfg {
    static constexpr int KT = D == 128 && !Q8 ? 16 : 32;            // keys per tile
    static constexpr int ROWB = Q8 ? D : 2 * D;                     // bytes of a cached row
    static constexpr int HALF = KT * ROWB, STAGE = 2 * HALF;        // K, V
    static constexpr int STAGES = (W == 4 ? 16 : 24) * 1024 / STAGE;   // 64 or 192 KB per block in all
    static constexpr int STATE = 16 * (D + 4) * 4;                  // a warp's output at the end, in its ring's place
    static constexpr size_t SMEM = 1024 + (size_t)W * STAGES * (STAGE + (Q8 ? 2 * KT * 4 : 0));
    static_assert(STATE <= STAGES * STAGE, "state");
};

__device__ __forceinline__ float pf_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int DT> __device__ __forceinline__ uint32_t pf_cvt2(float lo, float hi) {
    uint32_t p;
    if (DT == QV_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    return p;
}
template <int DT> __device__ __forceinline__ void pf_mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    const uint32_t b[2] = {b0, b1};
    if (DT == QV_BF16) mma_bf16(c, a, b); else mma_f16(c, a, b);
}
// Two biased codes (bytes of u and v chosen by sel; the other bytes become 0x64)
// as exact fp16 integers: 0x6400 | b is 1024 + b, b = code + 128.
__device__ __forceinline__ uint32_t pf_codes(uint32_t u, uint32_t v, uint32_t sel) {
    const uint32_t p = __byte_perm(u, v, sel);
    uint32_t r;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(0x64806480u));
    return r;
}

// NQ: n-tiles of 8 query rows.
template <int DT, int D, bool Q8, int NQ, int W>
__global__ void __launch_bounds__(32 * W, W == 8 ? 1 : NQ == 1 ? 3 : 2)
paged_few_kernel(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV, const PagedArgs a) {
    using C = PfCfg<D, Q8, W>;
    constexpr int PF_WARPS = W, PF_THREADS = 32 * W;
    using T = typename Elt<DT>::T;
    constexpr int MT = Q8 ? QV_F16 : DT;                 // type of the products
    constexpr bool HILO = MT == QV_BF16;
    constexpr int KT = C::KT, NM = KT / 16, KS = D / 16, ND = D / 16;
    extern __shared__ unsigned char pf_raw[];
    unsigned char* sm = pf_raw + ((1024u - (smem_u32(pf_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[PF_WARPS][C::STAGES];
    __shared__ float s_m[PF_WARPS][16], s_l[PF_WARPS][16];
    __shared__ int s_bad;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PF_WARPS * C::STAGES; ++i) mbar_init(&full[0][0] + i, 1);
        s_bad = 0;
        fence_barrier_init();
        prefetch_tensormap(&mK);
        prefetch_tensormap(&mV);
    }
    // launched while the kernel before still ran; what is launched on this one starts only when that has ended
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, sp = blockIdx.y;
    const PagedSeq s = paged_seq(a, b);
    const int rows = s.live * a.G;
    const bool split = a.splits > 1 && s.kv > a.chunk;
    // as paged_check_rows, in one block of the sequence
    const bool check = h == 0 && sp == 0 && a.err && threadIdx.x == 32 * W - 1;
    auto rows_ok = [&]() { return a.cu_q[b] == s.q0 && a.cu_q[b + 1] == s.q0 + s.n; };
    if (rows == 0 || (!split && sp > 0)) {
        if (check && !rows_ok()) set_err(a.err, QV_DERR_CAPACITY);
        return;
    }
    const int last = paged_limit(a, s, s.live - 1);
    const int k_begin = split ? sp * a.chunk : 0;
    const int k_end = split ? min(last, k_begin + a.chunk) : last;
    if (split && k_begin >= last) return;
    const int tiles = k_end > k_begin ? (k_end - k_begin + KT - 1) / KT : 0;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = sm + warp * C::STAGES * C::STAGE;
    float* ring_sc = reinterpret_cast<float*>(sm + PF_WARPS * C::STAGES * C::STAGE) + warp * C::STAGES * 2 * KT;
    __syncthreads();

    // lane 0 loads: tile i of this warp holds the keys from k_begin + (warp + W i) KT on
    // (a TMA box is a whole tile, or at 16-token pages 16 of its keys)
    const int mine = tiles > warp ? (tiles - warp + PF_WARPS - 1) / PF_WARPS : 0;
    const int first = k_begin + warp * KT, past = first + mine * PF_WARPS * KT;
    const int piece = min(KT, 1 << a.page_shift), page_mask = (1 << a.page_shift) - 1;
    const int32_t* table = a.block_table + (size_t)b * a.max_pages;
    int ids[NM], next_key = first;       // the tile to load next, its stage, and its pages
    int next_st = 0;
    auto find_pages = [&]() {
#pragma unroll
        for (int p = 0; p < NM; ++p) {
            const int key = next_key + p * piece;
            ids[p] = -1;
            if (next_key < past && p * piece < KT && key < s.kv) {
                ids[p] = table[key >> a.page_shift];
                if ((unsigned)ids[p] >= (unsigned)a.pages) {     // as paged_page
                    if (a.err) set_err(a.err, QV_DERR_TABLE);
                    ids[p] = 0;
                }
            }
        }
    };
    auto issue = [&]() {
        uint64_t* bar = &full[warp][next_st];
        unsigned char* dst = ring + next_st * C::STAGE;
        const int n = NM == 2 && ids[1] >= 0 ? 2 : 1;
        mbar_arrive_expect_tx(bar, n * piece * (2 * C::ROWB + (Q8 ? 8 : 0)));
#pragma unroll
        for (int p = 0; p < NM; ++p) {
            if (p >= n) continue;
            const int off = (next_key + p * piece) & page_mask;
            if (Q8) {
                tma_load_4d(dst + p * piece * D, &mK, 0, off, h, ids[p], bar);
                tma_load_4d(dst + C::HALF + p * piece * D, &mV, 0, off, h, ids[p], bar);
                const size_t row = ((size_t)(ids[p] * (int64_t)a.H + h) << a.page_shift) + off;
                float* sc = ring_sc + next_st * 2 * KT + p * piece;
                bulk_load(sc, a.k_scale + row, piece * 4, bar);
                bulk_load(sc + KT, a.v_scale + row, piece * 4, bar);
            } else {
#pragma unroll
                for (int w = 0; w < D / 64; ++w) {
                    tma_load_4d(dst + w * KT * 128 + p * piece * 128, &mK, 64 * w, off, h, ids[p], bar);
                    tma_load_4d(dst + C::HALF + w * KT * 128 + p * piece * 128, &mV, 64 * w, off, h, ids[p], bar);
                }
            }
        }
        next_key += PF_WARPS * KT;
        next_st = next_st + 1 == C::STAGES ? 0 : next_st + 1;
    };
    if (lane == 0) {
        for (int i = 0; i < C::STAGES && i < mine; ++i) { find_pages(); issue(); }
        find_pages();
    }
    if (check && !rows_ok()) set_err(a.err, QV_DERR_CAPACITY);   // (behind the first loads)

    // query fragments: lane (g, t) holds row 8 q + g; its four slots of a k-step are elements 2t, 2t + 1,
    // 2t + 8, 2t + 9, or with INT8 the four consecutive codes of the chunk it reads
    uint32_t qb[NQ][KS][2];
    float cq[NQ][2];                     // c of the rows 8 q + 2t, 8 q + 2t + 1
    int lim[NQ][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        const int r = 8 * q + g;
        const T* src = r < rows ? reinterpret_cast<const T*>(a.q) + (size_t)(s.q0 + r / a.G) * a.q_stride + (size_t)(h * a.G + r % a.G) * D : nullptr;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int d0 = Q8 ? 64 * (k >> 2) + 16 * t + 4 * (k & 3) : 16 * k + 2 * t;
            qb[q][k][0] = src ? *reinterpret_cast<const uint32_t*>(src + d0) : 0u;
            qb[q][k][1] = src ? *reinterpret_cast<const uint32_t*>(src + d0 + (Q8 ? 2 : 8)) : 0u;
        }
        float back = 1.f;
        if constexpr (Q8 && DT == QV_BF16) {
            float mx = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    mx = fmaxf(mx, fabsf(__uint_as_float(qb[q][k][e] << 16)));
                    mx = fmaxf(mx, fabsf(__uint_as_float(qb[q][k][e] & 0xFFFF0000u)));
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // 2^-e with 2^e <= mx < 2^(e+1), from the exponent's bits (kept where both powers are normal)
            const int e = min(max((int)(__float_as_uint(mx) >> 23), 2), 252);
            const float down = __uint_as_float((uint32_t)(254 - e) << 23);
            back = __uint_as_float((uint32_t)e << 23);
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int w = 0; w < 2; ++w)
                    qb[q][k][w] = pf_cvt2<QV_F16>(__uint_as_float(qb[q][k][w] << 16) * down,
                                                  __uint_as_float(qb[q][k][w] & 0xFFFF0000u) * down);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int rr = 8 * q + 2 * t + e;
            cq[q][e] = a.scale_log2 * __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
            lim[q][e] = min(rr < rows ? paged_limit(a, s, rr / a.G) : s.kv, k_end);
        }
    }
    const int lim_min = min(paged_limit(a, s, 0), k_end);
    float o[NQ][ND][4], m[NQ][2], l[NQ][2];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
        m[q][0] = m[q][1] = -INFINITY;
        l[q][0] = l[q][1] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[q][d][0] = o[q][d][1] = o[q][d][2] = o[q][d][3] = 0.f;
    }

    int stage = 0, phase = 0;
    for (int k0 = first; k0 < past; k0 += PF_WARPS * KT) {
        bool ok = mbar_wait_bounded(&full[warp][stage], phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
            if (lane == 0) { s_bad = 1; if (a.err) set_err(a.err, QV_DERR_TIMEOUT); }
            break;
        }
        unsigned char* kt = ring + stage * C::STAGE;
        unsigned char* vt = kt + C::HALF;
        const uint32_t ka = smem_u32(kt), va = smem_u32(vt);
        float x[NM][NQ][4];              // keys 16 i + g (, + 8) x rows 2t, 2t + 1
#pragma unroll
        for (int i2 = 0; i2 < NM; ++i2)
#pragma unroll
            for (int q = 0; q < NQ; ++q) x[i2][q][0] = x[i2][q][1] = x[i2][q][2] = x[i2][q][3] = 0.f;
        if constexpr (!Q8) {
            const int r = lane & 15, hi = lane >> 4;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint32_t ch = (((2 * k) & 7) + hi) ^ (r & 7);
#pragma unroll
                for (int i2 = 0; i2 < NM; ++i2) {
                    uint32_t w[4];
                    ldsm_x4(ka + (k >> 2) * KT * 128 + (16 * i2 + r) * 128 + (ch << 4), w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) pf_mma<MT>(x[i2][q], w, qb[q][k][0], qb[q][k][1]);
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
#pragma unroll
                for (int i2 = 0; i2 < NM; ++i2) {
                    const int key = 16 * i2 + g;                 // and key + 8: the same place in the swizzle
                    const int ch = (t + 4 * c) ^ (D == 128 ? key & 7 : (key >> 1) & 3);
                    uint4 u = *reinterpret_cast<const uint4*>(kt + key * D + (ch << 4));
                    uint4 v = *reinterpret_cast<const uint4*>(kt + (key + 8) * D + (ch << 4));
                    const uint32_t* wu = reinterpret_cast<const uint32_t*>(&u);
                    const uint32_t* wv = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t cu = wu[k] ^ 0x80808080u, cv = wv[k] ^ 0x80808080u;
                        const uint32_t w[4] = {pf_codes(cu, 0x64646464u, 0x4140), pf_codes(cv, 0x64646464u, 0x4140),
                                               pf_codes(cu, 0x64646464u, 0x4342), pf_codes(cv, 0x64646464u, 0x4342)};
#pragma unroll
                        for (int q = 0; q < NQ; ++q) pf_mma<MT>(x[i2][q], w, qb[q][4 * c + k][0], qb[q][4 * c + k][1]);
                    }
                }
        }
        // base-2 logits; keys behind a row's limit leave
        const bool edge = k0 + KT > lim_min;
        float iv[NM][2];
        float top[NQ][2];
#pragma unroll
        for (int q = 0; q < NQ; ++q) top[q][0] = top[q][1] = -INFINITY;
#pragma unroll
        for (int i2 = 0; i2 < NM; ++i2)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = k0 + 16 * i2 + g + 8 * e;
                float ks = 1.f, lv = 0.f;
                if constexpr (Q8) {
                    const float* sc = ring_sc + stage * 2 * KT + 16 * i2 + g + 8 * e;
                    ks = sc[0];
                    float vs = sc[KT];
                    vs = fabsf(vs) < PF_MIN_SCALE ? PF_MIN_SCALE : vs;   // also a zero row, whose codes are 0; below: NaN
                    if (edge && key >= s.kv) { ks = 0.f; vs = 1.f; }     // what lies there is not a row
                    lv = __log2f(vs);
                    iv[i2][e] = pf_ex2(-lv);
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float& y = x[i2][q][2 * e + j];
                        y = Q8 ? fmaf(y * cq[q][j], ks, lv) : y * cq[q][j];
                        if (edge && key >= lim[q][j]) y = -INFINITY;
                        top[q][j] = fmaxf(top[q][j], y);
                    }
            }
        bool move = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) move = move || top[q][0] > m[q][0] + PF_LAZY || top[q][1] > m[q][1] + PF_LAZY;
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    float mx = top[q][j];
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
                    const bool mv = mx > m[q][j] + PF_LAZY;
                    const float mn = mv ? mx - PF_BELOW : m[q][j];
                    const float f = mv && m[q][j] != -INFINITY ? pf_ex2(m[q][j] - mn) : 1.f;
                    m[q][j] = mn;
                    l[q][j] *= f;
#pragma unroll
                    for (int d = 0; d < ND; ++d) { o[q][d][j] *= f; o[q][d][2 + j] *= f; }
                }
        }
        uint32_t p[NM][NQ][2], plo[NM][NQ][2];       // P^T as operand; the low parts
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const float b0 = m[q][0] == -INFINITY ? 0.f : m[q][0], b1 = m[q][1] == -INFINITY ? 0.f : m[q][1];
#pragma unroll
            for (int i2 = 0; i2 < NM; ++i2)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float p0 = pf_ex2(x[i2][q][2 * e] - b0), p1 = pf_ex2(x[i2][q][2 * e + 1] - b1);
                    l[q][0] = Q8 ? fmaf(p0, iv[i2][e], l[q][0]) : l[q][0] + p0;
                    l[q][1] = Q8 ? fmaf(p1, iv[i2][e], l[q][1]) : l[q][1] + p1;
                    const uint32_t w = pf_cvt2<MT>(p0, p1);
                    p[i2][q][e] = movm_t(w);
                    if constexpr (HILO)
                        plo[i2][q][e] = movm_t(pf_cvt2<MT>(p0 - __uint_as_float(w << 16), p1 - __uint_as_float(w & 0xFFFF0000u)));
                }
        }
        if (!Q8 && k0 + KT > s.kv) {
            // rows behind the sequence may hold anything: 0 times that must be 0
            for (int c = lane; c < KT * (D / 64) * 8; c += 32)
                if (k0 + ((c >> 3) % KT) >= s.kv) *reinterpret_cast<uint4*>(vt + c * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
#pragma unroll
        for (int i2 = 0; i2 < NM; ++i2) {
            if constexpr (!Q8) {
                const int r = 16 * i2 + (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    uint32_t w[4];
                    ldsm_x4_t(va + (d >> 2) * KT * 128 + r * 128 + (((((2 * d) & 7) + hi) ^ (r & 7)) << 4), w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        pf_mma<MT>(o[q][d], w, p[i2][q][0], p[i2][q][1]);
                        if constexpr (HILO) pf_mma<MT>(o[q][d], w, plo[i2][q][0], plo[i2][q][1]);
                    }
                }
            } else {
                // lane (g, t): chunk g (D / 8 codes) of key rows 2t, 2t + 1, 2t + 8, 2t + 9; rows g and g + 8 of tile d
                // are its elements 2d and 2d + 1
                uint32_t w[4][D / 32];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = 16 * i2 + 2 * t + (e & 1) + 8 * (e >> 1);
                    if constexpr (D == 128) {
                        const uint4 u = *reinterpret_cast<const uint4*>(vt + key * D + ((g ^ (key & 7)) << 4));
                        w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2*>(vt + key * D + (((g >> 1) ^ ((key >> 1) & 3)) << 4) + 8 * (g & 1));
                        w[e][0] = u.x; w[e][1] = u.y;
                    }
                }
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    // byte i of both keys of a pair, then 0x64 above each code
                    const uint32_t a0 = __byte_perm(w[0][c], w[1][c], 0x5140) ^ 0x80808080u, a1 = __byte_perm(w[0][c], w[1][c], 0x7362) ^ 0x80808080u;
                    const uint32_t b0 = __byte_perm(w[2][c], w[3][c], 0x5140) ^ 0x80808080u, b1 = __byte_perm(w[2][c], w[3][c], 0x7362) ^ 0x80808080u;
                    const uint32_t f[2][4] = {{pf_codes(a0, 0x64646464u, 0x4140), pf_codes(a0, 0x64646464u, 0x4342),
                                               pf_codes(b0, 0x64646464u, 0x4140), pf_codes(b0, 0x64646464u, 0x4342)},
                                              {pf_codes(a1, 0x64646464u, 0x4140), pf_codes(a1, 0x64646464u, 0x4342),
                                               pf_codes(b1, 0x64646464u, 0x4140), pf_codes(b1, 0x64646464u, 0x4342)}};
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int q = 0; q < NQ; ++q) pf_mma<MT>(o[q][2 * c + d], f[d], p[i2][q][0], p[i2][q][1]);
                }
            }
        }
        __syncwarp();
        if (lane == 0 && next_key < past) {
            issue();
            find_pages();
        }
        if (++stage == C::STAGES) { stage = 0; phase ^= 1; }
    }
    // the warps' states join
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[q][j] += __shfl_xor_sync(0xffffffffu, l[q][j], w);
    __syncthreads();
    if (s_bad) {
        // a load never arrived: wait (bounded) for those in flight before the block's memory goes
        if (lane == 0)
            for (int st = 0; st < C::STAGES; ++st) { mbar_wait_bounded(&full[warp][st], 0); mbar_wait_bounded(&full[warp][st], 1); }
        return;
    }
    float* so = reinterpret_cast<float*>(ring);          // [16][D + 4]
    constexpr int LD = D + 4;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
#pragma unroll
        for (int d = 0; d < ND; ++d) {
            const int c0 = Q8 ? D / 8 * g + 2 * d : 16 * d + g, c1 = Q8 ? c0 + 1 : c0 + 8;
            so[(8 * q + 2 * t) * LD + c0] = o[q][d][0];
            so[(8 * q + 2 * t + 1) * LD + c0] = o[q][d][1];
            so[(8 * q + 2 * t) * LD + c1] = o[q][d][2];
            so[(8 * q + 2 * t + 1) * LD + c1] = o[q][d][3];
        }
        if (g == 0)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s_m[warp][8 * q + 2 * t + j] = m[q][j];
                s_l[warp][8 * q + 2 * t + j] = l[q][j];
            }
    }
    __syncthreads();
    const int Hq = a.H * a.G;
    const float* all = reinterpret_cast<const float*>(sm);
    constexpr int NEXT = C::STAGES * C::STAGE / 4;
    for (int e = threadIdx.x; e < rows * D; e += PF_THREADS) {
        const int r = e / D, d = e % D;
        float mm = s_m[0][r];
#pragma unroll
        for (int w = 1; w < PF_WARPS; ++w) mm = fmaxf(mm, s_m[w][r]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < PF_WARPS; ++w) {
            const float f = pf_ex2(s_m[w][r] - base);
            sum = fmaf(s_l[w][r], f, sum);
            v = fmaf(all[w * NEXT + r * LD + d], f, v);
        }
        const size_t orow = (size_t)(s.q0 + r / a.G) * Hq + h * a.G + r % a.G;
        if (split) {
            const size_t prow = (size_t)sp * a.total_q * Hq + orow;
            a.part_o[prow * D + d] = v;
            if (d == 0) { a.part_ml[2 * prow] = mm; a.part_ml[2 * prow + 1] = sum; }
        } else {
            st<DT>(a.out, orow * D + d, sum > 0.f ? v / sum : sum);   // no key seen: 0 (a NaN sum stays NaN)
        }
    }
}

// ---------------------------------------------------------------- host
bool paged_map_pages(CUtensorMap* m, const void* base, int dt, bool q8, int D, int page, int H, int pages, int box_rows,
                     CUtensorMapSwizzle codes);

template <int DT, int D, bool Q8, int W> static int pf_launch(const PagedArgs& a, cudaStream_t s) {
    using C = PfCfg<D, Q8, W>;
    CUtensorMap mK, mV;
    const int page = 1 << a.page_shift, piece = page < C::KT ? page : C::KT;
    const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if (!paged_map_pages(&mK, a.k, DT, Q8, D, page, a.H, a.pages, piece, sw) ||
        !paged_map_pages(&mV, a.v, DT, Q8, D, page, a.H, a.pages, piece, sw))
        return QV_EINVAL;
    const bool few8 = a.max_q * a.G <= 8;
    auto kernel = few8 ? paged_few_kernel<DT, D, Q8, 1, W> : paged_few_kernel<DT, D, Q8, 2, W>;
    static std::atomic<uint64_t> seen[2] = {{0}, {0}};
    const cudaError_t e = paged_smem(kernel, C::SMEM, &seen[few8]);
    if (e != cudaSuccess) return set_cuda_error(e);
    const cudaError_t f = launch_pdl(kernel, dim3((unsigned)(a.B * a.H), a.splits), dim3(32 * W), C::SMEM, s, mK, mV, a);
    return f == cudaSuccess ? check_launch() : set_cuda_error(f);
}

template <int DT, int D, bool Q8> static int pf_width(const PagedArgs& a, bool wide, cudaStream_t s) {
    return wide ? pf_launch<DT, D, Q8, 8>(a, s) : pf_launch<DT, D, Q8, 4>(a, s);
}
template <int DT> static int pf_dispatch(const PagedArgs& a, int D, bool q8, bool wide, cudaStream_t s) {
    if (D == 128) return q8 ? pf_width<DT, 128, true>(a, wide, s) : pf_width<DT, 128, false>(a, wide, s);
    return q8 ? pf_width<DT, 64, true>(a, wide, s) : pf_width<DT, 64, false>(a, wide, s);
}

int paged_few_launch(const PagedArgs& a, int dt, int D, bool q8, bool wide, cudaStream_t s) {
    return dt == QV_BF16 ? pf_dispatch<QV_BF16>(a, D, q8, wide, s) : pf_dispatch<QV_F16>(a, D, q8, wide, s);
}

}  // namespace qv
