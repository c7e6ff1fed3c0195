// Paged attention of many query rows on the 5th-generation tensor cores
// (tcgen05 + TMEM), bf16 and fp16, pages in the same type or INT8.
//
// A block takes two tiles of up to 128 query rows of one KV head (row r is token
// r / G of the tile, head r % G of the group) and a range of keys, 128 at a
// time.  Per key tile j and row tile x:  S_x = Q_x K_j^T (fp32, TMEM);  P_x =
// exp2(S_x c - m_x) rounded to 16 bits, written over S_x in TMEM;  O_x += P_x V_j
// with P_x as the TMEM operand.  The two row tiles alternate: while one's 128
// softmax threads work (one row each), the tensor cores run the other's two
// products, so a key tile costs the larger of 2 x 2 products and the
// exponentials (16 per clock and SM) instead of their sum.  The (x, j) pairs take
// two or three S buffers in turn (what O leaves of TMEM's 512 columns), so that at
// D = 64, or once only one row tile has keys left, S of a later tile is ready when a
// tile's softmax ends: 17 chunks and single tokens at D = 64 103 us (114 with one
// buffer per row tile), four 512-token chunks over INT8 pages 241 (272).
//
// m_x is a reference, not the running maximum: softmax is the same for any m, and
// P only has to stay in its type's range.  The first tile sets m to its maximum
// (fp16: 2^7 below, so that P spans 2^-31 .. 2^8 relative to it); later tiles use
// it and move it only where P would pass 2^24 (fp16: 2^15), rescaling O_x and l_x.
// So almost no tile touches O in TMEM.
//
// (Measured and left out, 8192-token prompt at D = 128, 437-443 us in a short run, 513-523
// back to back at the clock that the power cap leaves: a quarter of
// the exponentials as a polynomial on the FMA pipe, 462 us; the two tiles' softmax
// warps taking turns at the exponentials, 456 us; two threads to a row, 494 us; no
// row maximum, the reference moving where a tile's sum of P is too large, 455-468.
// Without any exponentials it takes as long, and the tensor pipe is active in 61 % of the
// cycles: the hand-over between a tile's softmax and its products bounds it.  At D = 64
// (347 us, 346 without exponentials) the bound is the softmax warps' dependent
// instructions: two warps per scheduler issue in 34-39 % of its cycles.)
//
// P is one 16-bit number: outputs are 1.2-1.4 times as far from 64 bits as fp32 arithmetic
// rounded once.
//
// INT8 pages: codes become exact 16-bit integers in shared memory (six extra
// warps); the row scales ks, vs of a key stay in fp32: the logit is S c ks, and the
// value scale goes into P before its one rounding.  bf16 has the range for that:
//   p = exp2(S c ks - m),  l += p,  P = p vs,  O += P code.
// In fp16 it goes into the exponent, so that the row's reference keeps P in range
// whatever the scales are:
//   P = exp2(S c ks + log2(vs) - m),  l += P / vs,  O += P code.
//
// Warps 0-3 and 4-7: the softmax of the two tiles; 8: TMA; 9: MMA (one elected
// thread each); with INT8 10-15 convert.  Every wait is bounded.
#include <cudaTypedefs.h>
#include <math.h>

#include "paged.cuh"
#include "ptx.cuh"
#include "tcgen05.cuh"

namespace qv {

constexpr int PT_KEYS = 128;
constexpr int PT_SLAB = 16384;            // 128 rows x 64 16-bit elements, 128-byte swizzle
constexpr float PT_MIN_SCALE = 8.6736173798840355e-19f;   // 2^-60: a smaller value scale counts as this (fp16's own start at 2^-31)

template <int DT, int D, bool Q8> struct PtCfg {
    static constexpr int NS = D / 64;                       // slabs per operand tile
    static constexpr int SLOT = NS * PT_SLAB;
    static constexpr int SLOTS = Q8 ? (D == 128 ? 3 : 6) : (D == 128 ? 5 : 8);   // K and V tiles in turn
    static constexpr int RAW = PT_KEYS * D;                 // one tile of codes
    static constexpr int RAWS = Q8 ? 2 : 0;
    static constexpr int NB = D == 64 ? 3 : 2;              // S buffers: what of TMEM's 512 columns O leaves
    // Tiles of row scales held (INT8).  Entry j is rewritten for tile j + SC, once the slot of that tile's K is free:
    // at D = 128 after P.V of tile j + 2, at D = 64 after S of tile j + 5, which follows P of tile j + 2 at least.
    static constexpr int SC = D == 64 ? 8 : 4;
    // a row's reference is set this far (base 2) below a maximum, and moves when a logit exceeds it by FAR
    static constexpr float BELOW = DT == QV_F16 ? 7.f : 0.f, FAR = DT == QV_F16 ? 15.f : 24.f;
    static constexpr int THREADS = Q8 ? 512 : 384;
    // registers per thread after the split (the launch holds 128 x 512 or 168 x 384 of them)
    static constexpr int REGS_SOFTMAX = Q8 ? 192 : 208, REGS_OTHER = Q8 ? 64 : 88;
    // Q, slots, codes, and the row scales as loaded (2) and prepared (SC x 3)
    static constexpr size_t SMEM = 1024 + 2 * SLOT + SLOTS * SLOT + RAWS * RAW +
                                   (Q8 ? (2 + SC * 3) * PT_KEYS * 4 : 0);
    static_assert(SMEM <= 232448 - 512, "shared memory");
};

__device__ __forceinline__ float pt_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint64_t pt_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void pt_unpack(uint64_t r, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(r));
}
__device__ __forceinline__ uint64_t pt_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pt_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pt_mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t pt_both(float x) { return pt_pack(x, x); }
__device__ __forceinline__ float pt_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
template <int DT> __device__ __forceinline__ uint32_t pt_cvt2(float lo, float hi) {
    uint32_t p;
    if (DT == QV_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p) : "f"(hi), "f"(lo));
    return p;
}

// Two signed codes (bytes b0, b1 of w, chosen by sel) as exact 16-bit floats.
// fp16: 0x6400 | u is 1024 + u for a byte u; with u = code + 128, minus 1152.
// bf16 has 7 fraction bits: 0x4300 | (code & 127) is 128 + the low seven bits,
// 0x4300 | (code & 128) is 128 or, by the exponent's last bit, 256: their
// difference is the code.
template <int DT> __device__ __forceinline__ uint32_t pt_codes2(uint32_t w, uint32_t sel) {
    uint32_t r;
    if (DT == QV_F16) {
        const uint32_t p = __byte_perm(w ^ 0x80808080u, 0x64646464u, sel);
        asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(0x64806480u));
    } else {
        const uint32_t p = __byte_perm(w, 0, sel);
        const uint32_t lo = (p & 0x007F007Fu) | 0x43004300u, hi = (p & 0x00800080u) | 0x43004300u;
        asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(lo), "r"(hi));
    }
    return r;
}

// Bounded wait: false after about a second (raising the error word), or at once
// when another warp of the block has given up.
__device__ __forceinline__ bool pt_wait_slow(uint64_t* bar, uint32_t parity, volatile int* quit, int32_t* err) {
    const uint64_t t0 = global_ns();
    while (true) {
        if (mbar_try_wait(bar, parity)) return true;
        if (*quit) return false;
        if (global_ns() - t0 > 1000000000ull) {
            *quit = 1;
            if (err) set_err(err, QV_DERR_TIMEOUT);
            return false;
        }
    }
}
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, volatile int* quit, int32_t* err) {
    if (mbar_try_wait(bar, parity)) return true;
    return pt_wait_slow(bar, parity, quit, err);
}

template <int DT, int D, bool Q8>
__global__ void __launch_bounds__(PtCfg<DT, D, Q8>::THREADS, 1)
paged_tc_kernel(const __grid_constant__ CUtensorMap mQ, const __grid_constant__ CUtensorMap mK,
                const __grid_constant__ CUtensorMap mV, const PagedArgs a) {
    using C = PtCfg<DT, D, Q8>;
    constexpr int NS = C::NS, SLOT = C::SLOT, SLOTS = C::SLOTS, NB = C::NB, PT_SC = C::SC;
    extern __shared__ unsigned char pt_raw[];
    unsigned char* sm = pt_raw + ((1024u - (smem_u32(pt_raw) & 1023u)) & 1023u);
    unsigned char* sQ = sm;                              // [2][NS] slabs
    unsigned char* sKV = sQ + 2 * SLOT;                  // [SLOTS]: K0, V0, K1, V1, ...
    unsigned char* sRaw = sKV + SLOTS * SLOT;            // [RAWS] tiles of codes
    float* sRawSc = reinterpret_cast<float*>(sRaw + C::RAWS * C::RAW);   // [2][128] as loaded: ks, vs
    float* sSc = sRawSc + 2 * PT_KEYS;                   // [SC][3][128]: c ks and vs, or (fp16) c ks, log2 vs, 1 / vs
    __shared__ __align__(8) uint64_t q_full, kv_full[SLOTS], kv_empty[SLOTS], raw_full[2], raw_empty[2], sc_full[PT_SC];
    __shared__ __align__(8) uint64_t s_full[NB], p_full[NB][2], o_full[NB], o_last[2], tail, done;
    __shared__ uint32_t s_taddr;
    __shared__ int2 s_tile;
    __shared__ int s_quit;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // uniform
    const int h = blockIdx.x % a.H, sp = blockIdx.y;
    const int QT = PT_KEYS / a.G;                        // tokens per row tile

    if (warp == 0) {
        const int2 t = paged_find_tile(a, blockIdx.x / a.H, 1, 2 * QT);
        if (lane == 0) s_tile = t;
    }
    if (warp == 9 && blockIdx.x == 0 && blockIdx.y == 0) paged_check_rows(a, lane);
    __syncthreads();
    const int b = s_tile.x;
    if (b < 0) return;
    const PagedSeq s = paged_seq(a, b);
    const int Hq = a.H * a.G;
    const bool split = a.splits > 1 && s.kv > a.chunk;
    if (!split && sp > 0) return;
    const int k_begin = split ? sp * a.chunk : 0;
    // per row tile: first token, tokens, key tiles of this block's range
    int tok[2], cnt[2], nt[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        tok[x] = (2 * s_tile.y + x) * QT;
        cnt[x] = min(max(s.live - tok[x], 0), QT);
        int end = cnt[x] > 0 ? paged_limit(a, s, tok[x] + cnt[x] - 1) : 0;
        if (split) end = min(end, k_begin + a.chunk);
        nt[x] = end > k_begin ? (end - k_begin + PT_KEYS - 1) / PT_KEYS : 0;
    }
    const int n = max(nt[0], nt[1]);
    if (split && n == 0) return;
    // keys of the last tile that exist: what lies behind them is never multiplied
    const int live_last = n > 0 ? s.kv - k_begin - (n - 1) * PT_KEYS : PT_KEYS;
    const bool cut = live_last < PT_KEYS;

    if (warp == 9) { tmem_alloc(&s_taddr, 512); tmem_relinquish(); }
    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1);
        for (int i = 0; i < SLOTS; ++i) { mbar_init(&kv_full[i], Q8 ? 6 : 1); mbar_init(&kv_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 6); mbar_init(&o_last[i], 1); }
        for (int i = 0; i < NB; ++i) {
            mbar_init(&s_full[i], 1); mbar_init(&o_full[i], 1);
            mbar_init(&p_full[i][0], 4); mbar_init(&p_full[i][1], 4);
        }
        for (int i = 0; i < PT_SC; ++i) mbar_init(&sc_full[i], 4);
        mbar_init(&tail, 1);
        mbar_init(&done, 1);
        s_quit = 0;
        fence_barrier_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t taddr = s_taddr;      // NB x 128 columns of S (P over it), then O of the two row tiles
    constexpr int O_AT = 128 * NB;
    static_assert(O_AT + 2 * D <= 512, "TMEM columns");
    // The (row tile, key tile) pairs in the order of their products, the two row tiles in turn while both have keys
    // left (the second has at least as many as the first, or none); pair `step` uses buffer step % NB.  S of pair
    // step + NB is issued behind P.V of pair step, so a buffer's barriers (s_full, p_full, o_full) are never more than
    // a phase ahead of a warp that waits on them by parity; the last P.V of a row tile has a barrier of its own
    // (o_last), since the other row tile goes on using the buffers.
    const int both = nt[1] > 0 ? nt[0] : 0, steps = nt[0] + nt[1];
    volatile int* quit = &s_quit;

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::REGS_SOFTMAX));
        // ------------------------------------------------------------ softmax of row tile x
        const int x = warp >> 2, r = threadIdx.x & 127;
        const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t to = taddr + lane_off + O_AT + D * x;
        const int i = r / a.G;
        const int tok_x = x ? tok[1] : tok[0], tn = x ? nt[1] : nt[0];
        const bool live = i < (x ? cnt[1] : cnt[0]);
        int lim = live ? paged_limit(a, s, tok_x + i) - k_begin : 0x7fffffff;   // relative to the block's range
        const bool idle = 32 * (warp & 3) >= (x ? cnt[1] : cnt[0]) * a.G;
        int lim_min = lim;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lim_min = min(lim_min, __shfl_xor_sync(0xffffffffu, lim_min, o));
        float m = -INFINITY;
        uint64_t l2 = pt_pack(0.f, 0.f);
        const float cl = a.scale_log2;
        const uint64_t c2 = pt_pack(cl, cl);
        bool ok = true;
        int step = 0, before = 0;            // this tile's pair, the one before
        for (int j = 0; j < tn; ++j) {
            before = step;
            step = j < both ? 2 * j + x : both + j;
            const int buf = step % NB;
            const uint32_t ts = taddr + lane_off + 128 * buf;
            ok = pt_wait(&s_full[buf], (step / NB) & 1, quit, a.err);
            if (Q8 && ok) ok = pt_wait(&sc_full[j % PT_SC], (j / PT_SC) & 1, quit, a.err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            if (idle) {                      // no live row in this warp: P may hold anything there
                tc_fence_before();
                __syncwarp();
                if (lane == 0) { mbar_arrive(&p_full[buf][0]); mbar_arrive(&p_full[buf][1]); }
                continue;
            }
            float v[128];
#pragma unroll
            for (int w = 0; w < 4; ++w) tmem_ld32(ts + 32 * w, v + 32 * w);
            tmem_wait_ld();
            const float* sc = sSc + (j % PT_SC) * 3 * PT_KEYS;
            if constexpr (Q8) {
                // base-2 logits (fp16: with the value scale in them)
#pragma unroll
                for (int e = 0; e < 128; e += 4) {
                    const float4 k4 = *reinterpret_cast<const float4*>(sc + e);
                    uint64_t u0, u1;
                    if constexpr (DT == QV_F16) {
                        const float4 l4 = *reinterpret_cast<const float4*>(sc + PT_KEYS + e);
                        u0 = pt_fma2(pt_pack(v[e], v[e + 1]), pt_pack(k4.x, k4.y), pt_pack(l4.x, l4.y));
                        u1 = pt_fma2(pt_pack(v[e + 2], v[e + 3]), pt_pack(k4.z, k4.w), pt_pack(l4.z, l4.w));
                    } else {
                        u0 = pt_mul2(pt_pack(v[e], v[e + 1]), pt_pack(k4.x, k4.y));
                        u1 = pt_mul2(pt_pack(v[e + 2], v[e + 3]), pt_pack(k4.z, k4.w));
                    }
                    pt_unpack(u0, v[e], v[e + 1]);
                    pt_unpack(u1, v[e + 2], v[e + 3]);
                }
            }
            const int seen = lim - j * PT_KEYS;
            if (lim_min < (j + 1) * PT_KEYS) {
#pragma unroll
                for (int e = 0; e < 128; ++e) v[e] = e < seen ? v[e] : -INFINITY;
            }
            float hi[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
            for (int e = 4; e < 124; e += 8)
#pragma unroll
                for (int w = 0; w < 4; ++w) hi[w] = pt_max3(hi[w], v[e + 2 * w], v[e + 2 * w + 1]);
            float mx = pt_max3(pt_max3(hi[0], hi[1], hi[2]), pt_max3(hi[3], v[124], v[125]), fmaxf(v[126], v[127]));
            if (!Q8) mx *= cl;
            if (__any_sync(0xffffffffu, mx > m + C::FAR)) {
                // the reference moves, and what was summed before follows
                const bool move = mx > m + C::FAR;
                const float mn = move ? mx - C::BELOW : m;
                const float f = move && m != -INFINITY ? pt_ex2(m - mn) : 1.f;
                m = mn;
                l2 = pt_mul2(l2, pt_both(f));
                if (j > 0) {
                    ok = __all_sync(0xffffffffu, pt_wait(&o_full[before % NB], (before / NB) & 1, quit, a.err));   // P.V of the tile before
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int w = 0; w < D / 16; ++w) {
                        float o[16];
                        uint32_t u[16];
                        tmem_ld16(to + 16 * w, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * f);
                        tmem_st16(to + 16 * w, u);
                    }
                }
            }
            const uint64_t nm2 = pt_both(m == -INFINITY ? 0.f : -m);     // nothing seen yet: every term is 0
            uint64_t acc[2] = {l2, pt_both(0.f)};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                uint32_t p[16];
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const int k = 32 * w + 2 * e;
                    float d[4];
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        const uint64_t v2 = pt_pack(v[k + 2 * h2], v[k + 2 * h2 + 1]);
                        pt_unpack(Q8 ? pt_add2(v2, nm2) : pt_fma2(v2, c2, nm2), d[2 * h2], d[2 * h2 + 1]);
                    }
#pragma unroll
                    for (int i4 = 0; i4 < 4; ++i4) d[i4] = pt_ex2(d[i4]);
                    if constexpr (Q8) {
                        // 1 / vs (fp16), or vs
                        const float4 f4 = *reinterpret_cast<const float4*>(sc + (DT == QV_F16 ? 2 : 1) * PT_KEYS + k);
                        const uint64_t f0 = pt_pack(f4.x, f4.y), f1 = pt_pack(f4.z, f4.w);
                        if constexpr (DT == QV_F16) {
                            acc[0] = pt_fma2(pt_pack(d[0], d[1]), f0, acc[0]);
                            acc[1] = pt_fma2(pt_pack(d[2], d[3]), f1, acc[1]);
                        } else {
                            acc[0] = pt_add2(acc[0], pt_pack(d[0], d[1]));
                            acc[1] = pt_add2(acc[1], pt_pack(d[2], d[3]));
                            pt_unpack(pt_mul2(pt_pack(d[0], d[1]), f0), d[0], d[1]);
                            pt_unpack(pt_mul2(pt_pack(d[2], d[3]), f1), d[2], d[3]);
                        }
                    } else {
                        acc[0] = pt_add2(acc[0], pt_pack(d[0], d[1]));
                        acc[1] = pt_add2(acc[1], pt_pack(d[2], d[3]));
                    }
                    p[e] = pt_cvt2<DT>(d[0], d[1]);
                    p[e + 1] = pt_cvt2<DT>(d[2], d[3]);
                }
                tmem_st16(ts + 16 * w, p);
                if (w & 1) {                 // 64 keys of P: the product may start on them
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[buf][w >> 1]);
                }
            }
            l2 = pt_add2(acc[0], acc[1]);
        }
        float l0, l1;
        pt_unpack(l2, l0, l1);
        const float l = l0 + l1;
        if (tn > 0) ok = ok && pt_wait(&o_last[x], 0, quit, a.err);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
            const size_t orow = (size_t)(s.q0 + tok_x + i) * Hq + h * a.G + (r - i * a.G);
            const size_t prow = (size_t)sp * a.total_q * Hq + orow;
            const float inv = split ? 1.f : l > 0.f ? 1.f / l : l;   // no key seen: 0 (a NaN sum stays NaN)
            if (split && live && tn > 0) {
                a.part_ml[2 * prow] = m;
                a.part_ml[2 * prow + 1] = l;
            }
#pragma unroll
            for (int w = 0; w < D / 32; ++w) {
                float o[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = 0.f;
                if (tn > 0) {
                    tmem_ld32(to + 32 * w, o);
                    tmem_wait_ld();
                }
                if (!live) continue;
                if (split) {
                    if (tn > 0)
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(a.part_o + prow * D + 32 * w + e) =
                                make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                } else {
                    uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.out) + orow * D + 32 * w);
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        dst[e / 8] = make_uint4(pt_cvt2<DT>(o[e] * inv, o[e + 1] * inv),
                                                pt_cvt2<DT>(o[e + 2] * inv, o[e + 3] * inv),
                                                pt_cvt2<DT>(o[e + 4] * inv, o[e + 5] * inv),
                                                pt_cvt2<DT>(o[e + 6] * inv, o[e + 7] * inv));
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::REGS_OTHER));
        if (warp == 8) {
            // -------------------------------------------------------- loads
            if (n > 0 && lane == 0) {
                prefetch_tensormap(&mQ);
                prefetch_tensormap(&mK);
                prefetch_tensormap(&mV);
                int bytes = 0;
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    if (nt[x] > 0) bytes += NS * QT * a.G * 128;
                mbar_arrive_expect_tx(&q_full, bytes);
#pragma unroll
                for (int x = 0; x < 2; ++x)
                    for (int w = 0; nt[x] > 0 && w < NS; ++w)
                        tma_load_3d(sQ + x * SLOT + w * PT_SLAB, &mQ, 64 * w, h * a.G, s.q0 + tok[x], &q_full);
            }
            const int page = 1 << a.page_shift, per_tile = PT_KEYS >> a.page_shift;
            // lane i keeps the id of the tile's page i
            int id = 0, next = 0;
            bool ok = true;
            if (n > 0 && lane < per_tile && lane * page < s.kv - k_begin) next = paged_page(a, b, k_begin + lane * page);
            int issued = 0;
            for (int j = 0; j < n && ok; ++j) {
                id = next;
                const int k0 = k_begin + j * PT_KEYS, left = s.kv - k0;
                const int np = min(per_tile, (left + page - 1) >> a.page_shift);   // pages of the tile that hold keys
                if (j + 1 < n && lane < per_tile && lane * page < left - PT_KEYS)
                    next = paged_page(a, b, k0 + PT_KEYS + lane * page);
                for (int kv = 0; kv < 2 && ok; ++kv) {
                    const int it = 2 * j + kv;
                    const CUtensorMap* map = kv ? &mV : &mK;
                    if constexpr (Q8) {
                        const int st = it & 1;
                        if (it >= 2) ok = pt_wait(&raw_empty[st], ((it >> 1) - 1) & 1, quit, a.err);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&raw_full[st], np * page * (D + (kv ? 0 : 8)));
                        __syncwarp();
                        if (lane < np) {
                            tma_load_4d(sRaw + st * C::RAW + lane * page * D, map, 0, 0, h, id, &raw_full[st]);
                            if (kv == 0) {
                                const size_t row = ((size_t)id * a.H + h) << a.page_shift;
                                float* dst = sRawSc + lane * page;
                                bulk_load(dst, a.k_scale + row, page * 4, &raw_full[st]);
                                bulk_load(dst + PT_KEYS, a.v_scale + row, page * 4, &raw_full[st]);
                            }
                        }
                    } else {
                        const int st = it % SLOTS;
                        if (it >= SLOTS) ok = pt_wait(&kv_empty[st], (it / SLOTS - 1) & 1, quit, a.err);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&kv_full[st], np * page * D * 2);
                        __syncwarp();
                        if (lane < np)
                            for (int w = 0; w < NS; ++w)
                                tma_load_4d(sKV + st * SLOT + w * PT_SLAB + lane * page * 128, map, 64 * w, 0, h, id,
                                            &kv_full[st]);
                    }
                    issued = it + 1;
                }
            }
            if (!Q8 && cut && ok && n > 0) {
                // the last V tile's rows behind the sequence: zero, whatever the pages hold there
                const int it = 2 * n - 1, st = it % SLOTS;
                ok = pt_wait(&kv_full[st], (it / SLOTS) & 1, quit, a.err);
                if (__all_sync(0xffffffffu, ok)) {
                    for (int w = 0; w < NS; ++w)
                        for (int c = live_last * 8 + lane; c < PT_KEYS * 8; c += 32)
                            *reinterpret_cast<uint4*>(sKV + st * SLOT + w * PT_SLAB + c * 16) = make_uint4(0, 0, 0, 0);
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&tail);
                }
            }
            // the copies this warp issued have landed before the block exits
            if (n > 0) mbar_wait_bounded(&q_full, 0);
            constexpr int RING = Q8 ? 2 : SLOTS;
            uint64_t* full = Q8 ? raw_full : kv_full;
            for (int it = max(issued - RING, 0); it < issued; ++it) mbar_wait_bounded(&full[it % RING], (it / RING) & 1);
        } else if (warp == 9) {
            // -------------------------------------------------------- products
            // the whole warp walks the loop (operands in uniform registers), one elected lane issues
            if (n > 0) {
                const uint32_t id_s = umma_idesc_f16(DT == QV_BF16, 128, 128, 0, 0);
                const uint32_t id_o = umma_idesc_f16(DT == QV_BF16, 128, D, 0, 1);
                const uint64_t dq = umma_desc_sw128(smem_u32(sQ), 16, 1024);
                const uint64_t dk = umma_desc_sw128(smem_u32(sKV), 16, 1024);
                const uint64_t dv = umma_desc_sw128(smem_u32(sKV), PT_SLAB, 1024);
                const bool one = elect_one();
                auto wait = [&](uint64_t* bar, uint32_t parity) {
                    return __all_sync(0xffffffffu, pt_wait(bar, parity, quit, a.err)) != 0;
                };
                bool ok = wait(&q_full, 0);
                tc_fence_after();
                auto wait_tile = [&](int it) {
                    bool o = wait(&kv_full[it % SLOTS], (it / SLOTS) & 1);
                    if (!Q8 && o && cut && it == 2 * n - 1) o = wait(&tail, 0);
                    tc_fence_after();
                    return o;
                };
                // pair `step`: row tile, key tile, and whether no later pair reads the key tile
                auto pair = [&](int step, int& x, int& j, bool& last) {
                    const bool two = step < 2 * both;
                    x = two ? step & 1 : nt[1] > 0;
                    j = two ? step >> 1 : step - both;
                    last = x == 1 || j >= nt[1];
                };
                auto scores = [&](int step) {
                    int x, j;
                    bool last;
                    pair(step, x, j, last);
                    if (!wait_tile(2 * j)) return false;
                    const uint64_t q = dq + x * (SLOT >> 4), k = dk + ((2 * j) % SLOTS) * (SLOT >> 4);
                    const uint32_t to = taddr + 128 * (step % NB);
                    if (one) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            constexpr int S4 = PT_SLAB >> 4;
                            umma_ss(to, q + (kk >> 2) * S4 + (kk & 3) * 2, k + (kk >> 2) * S4 + (kk & 3) * 2, id_s, kk > 0);
                        }
                        umma_commit(&s_full[step % NB]);
                        if (last) umma_commit(&kv_empty[(2 * j) % SLOTS]);
                    }
                    return true;
                };
                for (int i = 0; i < NB && i < steps && ok; ++i) ok = scores(i);
                for (int i = 0; i < steps && ok; ++i) {
                    int x, j;
                    bool last;
                    pair(i, x, j, last);
                    ok = wait_tile(2 * j + 1);
                    const uint64_t v = dv + ((2 * j + 1) % SLOTS) * (SLOT >> 4);
                    const uint32_t ps = taddr + 128 * (i % NB), to = taddr + O_AT + D * x;
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf) {
                        if (ok) ok = wait(&p_full[i % NB][hf], (i / NB) & 1);
                        if (!ok) break;
                        tc_fence_after();
                        if (one) {
#pragma unroll
                            for (int kk = 4 * hf; kk < 4 * hf + 4; ++kk)
                                umma_ts(to, ps + 8 * kk, v + kk * 128, id_o, j > 0 || kk > 0);
                        }
                    }
                    if (!ok) break;
                    if (one) {
                        umma_commit(&o_full[i % NB]);
                        if (j + 1 == (x ? nt[1] : nt[0])) umma_commit(&o_last[x]);
                        if (last) umma_commit(&kv_empty[(2 * j + 1) % SLOTS]);
                    }
                    if (i + NB < steps) ok = scores(i + NB);
                }
                // no MMA is in flight when the TMEM is released
                if (one) umma_commit(&done);
                mbar_wait_bounded(&done, 0);
            }
        } else if (Q8 && warp >= 10) {
            // -------------------------------------------------------- codes -> 16-bit operands
            // A tile is PARTS x 128 chunks of 16 codes.  Warps 12-15 (t = 0..127) take the first five eighths of
            // the parts, warps 10 and 11 the rest, each lane two chunks of a part.  Eight lanes hold four chunks
            // of two rows, so that neither their reads (128-byte swizzle at D = 128) nor their writes share
            // banks: rows r and r ^ 5, or (D = 64) r and r + 1; parts differ by constants.
            constexpr int PARTS = PT_KEYS * D / 16 / 128, FIRST = PARTS * 5 / 8;
            const bool extra = warp < 12;
            const int t = extra ? threadIdx.x - 320 : threadIdx.x - 384;
            auto place = [&](int i, int& from, int& to0, int& to1) {     // chunk i of part 0
                int r, cc;
                if constexpr (D == 128) {
                    r = (i >> 5) * 8 + ((i >> 3) & 3);
                    if (i & 4) r ^= 5;
                    cc = i & 3;
                    from = r * 128 + ((cc ^ (r & 7)) << 4);
                } else {
                    r = i >> 2;
                    cc = i & 3;
                    from = r * 64 + cc * 16;
                }
                to0 = r * 128 + (((2 * cc) ^ (r & 7)) << 4);
                to1 = r * 128 + (((2 * cc + 1) ^ (r & 7)) << 4);
            };
            // D = 128: parts 0-3 are rows +32 each of the low four chunks, 4-7 of the high four (the other slab)
            auto convert = [&](const unsigned char* raw, unsigned char* dst, int part, int from, int to0, int to1, int rows) {
                const int r = (to0 >> 7) + 32 * (part & 3);
                const unsigned char* src = raw + (D == 128 ? (from ^ ((part >> 2) << 6)) + (part & 3) * 32 * 128 : from + part * 32 * 64);
                uint4 u = make_uint4(0, 0, 0, 0);
                if (r < rows) u = *reinterpret_cast<const uint4*>(src);
                constexpr uint32_t S0 = 0x4140, S1 = 0x4342;
                unsigned char* out = dst + (D == 128 ? part >> 2 : 0) * PT_SLAB + (part & 3) * 32 * 128;
                *reinterpret_cast<uint4*>(out + to0) = make_uint4(pt_codes2<DT>(u.x, S0), pt_codes2<DT>(u.x, S1),
                                                                  pt_codes2<DT>(u.y, S0), pt_codes2<DT>(u.y, S1));
                *reinterpret_cast<uint4*>(out + to1) = make_uint4(pt_codes2<DT>(u.z, S0), pt_codes2<DT>(u.z, S1),
                                                                  pt_codes2<DT>(u.w, S0), pt_codes2<DT>(u.w, S1));
            };
            int from[2], to0[2], to1[2];
            place(t, from[0], to0[0], to1[0]);
            place(extra ? t + 64 : t, from[1], to0[1], to1[1]);
            bool ok = true;
            for (int it = 0; it < 2 * n && ok; ++it) {
                const int st = it & 1, slot = it % SLOTS, j = it >> 1;
                ok = pt_wait(&raw_full[st], (it >> 1) & 1, quit, a.err);
                if (ok && it >= SLOTS) ok = pt_wait(&kv_empty[slot], (it / SLOTS - 1) & 1, quit, a.err);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int rows = j + 1 == n ? min(live_last, PT_KEYS) : PT_KEYS;
                if ((it & 1) == 0 && !extra) {
                    // scales of this tile's keys; one behind the sequence contributes nothing
                    float* sc = sSc + (j % PT_SC) * 3 * PT_KEYS;
                    const float ks = sRawSc[t];
                    float vs = sRawSc[PT_KEYS + t];
                    const bool in = t < rows;
                    sc[t] = in ? ks * a.scale_log2 : 0.f;
                    if constexpr (DT == QV_F16) {
                        if (fabsf(vs) < PT_MIN_SCALE) vs = PT_MIN_SCALE;   // also a zero row, whose codes are 0; below: NaN
                        sc[PT_KEYS + t] = in ? log2f(vs) : 0.f;
                        sc[2 * PT_KEYS + t] = in ? 1.f / vs : 0.f;
                    } else {
                        sc[PT_KEYS + t] = in ? vs : 0.f;
                    }
                }
                const unsigned char* raw = sRaw + st * C::RAW;
                unsigned char* dst = sKV + slot * SLOT;
                if (!extra) {
#pragma unroll
                    for (int part = 0; part < FIRST; ++part) convert(raw, dst, part, from[0], to0[0], to1[0], rows);
                } else {
#pragma unroll
                    for (int part = FIRST; part < PARTS; ++part) {
                        convert(raw, dst, part, from[0], to0[0], to1[0], rows);
                        convert(raw, dst, part, from[1], to0[1], to1[1], rows);
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&kv_full[slot]);
                    mbar_arrive(&raw_empty[st]);
                    if ((it & 1) == 0 && !extra) mbar_arrive(&sc_full[j % PT_SC]);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(taddr, 512);
    }
}

// ---------------------------------------------------------------- host
static PFN_cuTensorMapEncodeTiled_v12000 pt_encode() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> found{nullptr};   // calls may come from several threads
    PFN_cuTensorMapEncodeTiled_v12000 fn = found.load(std::memory_order_acquire);
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
            found.store(fn, std::memory_order_release);
        }
    }
    return fn;
}

static CUtensorMapDataType pt_type(int dt) {
    return dt == QV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Pages as (D, page, heads, pages); a box is box_rows rows of one page, 64
// elements wide with the 128-byte swizzle, or whole rows of codes.
bool paged_map_pages(CUtensorMap* m, const void* base, int dt, bool q8, int D, int page, int H, int pages, int box_rows,
                     CUtensorMapSwizzle codes) {
    auto fn = pt_encode();
    if (!fn) return false;
    const cuuint64_t e = q8 ? 1 : 2;
    cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)H, (cuuint64_t)pages};
    cuuint64_t strides[3] = {D * e, D * e * page, D * e * page * H};
    cuuint32_t box[4] = {(cuuint32_t)(q8 ? D : 64), (cuuint32_t)box_rows, 1, 1};
    cuuint32_t es[4] = {1, 1, 1, 1};
    return fn(m, q8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : pt_type(dt), 4, const_cast<void*>(base), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, q8 ? codes : CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Queries as (D, heads, tokens); a box is one row tile: 64 elements x G heads x 128 / G tokens.
static bool pt_map_q(CUtensorMap* m, const PagedArgs& a, int dt, int D) {
    auto fn = pt_encode();
    if (!fn) return false;
    cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)a.H * a.G, (cuuint64_t)a.total_q};
    cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)a.q_stride * 2};
    cuuint32_t box[3] = {64, (cuuint32_t)a.G, (cuuint32_t)(PT_KEYS / a.G)};
    cuuint32_t es[3] = {1, 1, 1};
    return fn(m, pt_type(dt), 3, const_cast<void*>(a.q), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
           CUDA_SUCCESS;
}

template <int DT, int D, bool Q8> static int pt_launch(const PagedArgs& a, int64_t tiles, cudaStream_t s) {
    using C = PtCfg<DT, D, Q8>;
    CUtensorMap mQ, mK, mV;
    const int page = 1 << a.page_shift;
    const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE;
    if (!pt_map_q(&mQ, a, DT, D) || !paged_map_pages(&mK, a.k, DT, Q8, D, page, a.H, a.pages, page, sw) ||
        !paged_map_pages(&mV, a.v, DT, Q8, D, page, a.H, a.pages, page, sw))
        return QV_EINVAL;
    static std::atomic<uint64_t> seen{0};
    const cudaError_t e = paged_smem(paged_tc_kernel<DT, D, Q8>, C::SMEM, &seen);
    if (e != cudaSuccess) return set_cuda_error(e);
    paged_tc_kernel<DT, D, Q8><<<dim3((unsigned)(tiles * a.H), a.splits), C::THREADS, C::SMEM, s>>>(mQ, mK, mV, a);
    return check_launch();
}

template <int DT> static int pt_dispatch(const PagedArgs& a, int D, bool q8, int64_t tiles, cudaStream_t s) {
    if (D == 128) return q8 ? pt_launch<DT, 128, true>(a, tiles, s) : pt_launch<DT, 128, false>(a, tiles, s);
    return q8 ? pt_launch<DT, 64, true>(a, tiles, s) : pt_launch<DT, 64, false>(a, tiles, s);
}

int paged_tc_launch(const PagedArgs& a, int dt, int D, bool q8, int64_t tiles, cudaStream_t s) {
    return dt == QV_BF16 ? pt_dispatch<QV_BF16>(a, D, q8, tiles, s) : pt_dispatch<QV_F16>(a, D, q8, tiles, s);
}

}  // namespace qv
