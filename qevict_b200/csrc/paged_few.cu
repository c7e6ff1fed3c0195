// Paged attention of few query rows (a decode step; a few tokens times the
// heads of a group, up to 16 rows per KV head), bf16 and fp16, pages in the same
// type or INT8.
//
// Bound by HBM: every cached row is read once for at most 16 query rows, two
// orders of magnitude below the tensor cores' balance, so the work is keeping
// loads in flight.  A block takes one KV head of one sequence and a range of its
// keys; each of its four warps walks its own tiles of 16 or 32 keys through a
// ring of its own in shared memory (TMA, one elected lane, one mbarrier per
// stage), so that no barrier couples the warps until their states join at the
// end.  Two blocks share an SM: one's start and end hide behind the other's
// loads.
//
// Per tile: S = Q K^T and O += P V with warp-level MMA (m16n8k16, rows = query
// rows; P goes from accumulator to operand registers as it is), and in base 2
//   P = exp2(S c - m),  l += P,
// where the reference m moves only when a logit exceeds it by 2^8, so that a
// tile needs no row maximum across lanes.  INT8 rows: the codes become exact
// 16-bit integers in registers and the scales stay in fp32,
//   u = S c ks + log2(vs),  P = exp2(u - m),  O += P code,  l += P / vs.
// The contraction over the head's elements may run in any order, and so may the
// columns of O: with INT8 each lane takes 16-byte chunks of a row as the
// elements of its own fragments.
#include <cudaTypedefs.h>
#include <math.h>

#include "paged.cuh"
#include "ptx.cuh"

namespace qv {

constexpr int PF_WARPS = 4;
constexpr int PF_THREADS = 32 * PF_WARPS;
constexpr int PF_PIECE = 16;              // keys per TMA box: never across a page
constexpr float PF_LAZY = 8.f;
constexpr float PF_MIN_SCALE = 7.8886090522101181e-31f;   // 2^-100: a smaller value scale counts as this

template <int D, bool Q8> struct PfCfg {
    static constexpr int KT = D == 128 && !Q8 ? 16 : 32;            // keys per tile
    static constexpr int ROWB = Q8 ? D : 2 * D;                     // bytes of a cached row
    static constexpr int HALF = KT * ROWB, STAGE = 2 * HALF;        // K, V
    static constexpr int STAGES = 24 * 1024 / STAGE;                // 96 KB per block in all
    static constexpr int STATE = 16 * (D + 4) * 4;                  // a warp's output at the end, in its ring's place
    static constexpr size_t SMEM = 1024 + (size_t)PF_WARPS * STAGES * (STAGE + (Q8 ? 2 * KT * 4 : 0));
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
// Codes in bytes 0 and 2 of w as exact 16-bit floats.  fp16: 0x6400 | u is
// 1024 + u, u = code + 128.  bf16: 0x4300 | (code & 127) is 128 + the low seven
// bits and 0x4300 | (code & 128) is 128, or 256 by the exponent's last bit.
template <int DT> __device__ __forceinline__ uint32_t pf_codes(uint32_t w) {
    uint32_t r;
    if (DT == QV_F16) {
        const uint32_t p = ((w ^ 0x00800080u) & 0x00FF00FFu) | 0x64006400u;
        asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(p), "r"(0x64806480u));
    } else {
        const uint32_t lo = (w & 0x007F007Fu) | 0x43004300u, hi = (w & 0x00800080u) | 0x43004300u;
        asm("sub.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(lo), "r"(hi));
    }
    return r;
}

template <int DT, int D, bool Q8>
__global__ void __launch_bounds__(PF_THREADS, 2)
paged_few_kernel(const __grid_constant__ CUtensorMap mK, const __grid_constant__ CUtensorMap mV, const PagedArgs a) {
    using C = PfCfg<D, Q8>;
    using T = typename Elt<DT>::T;
    constexpr int KT = C::KT, NT = KT / 8, KS = D / 16, ND = D / 8;
    extern __shared__ unsigned char pf_raw[];
    unsigned char* sm = pf_raw + ((1024u - (smem_u32(pf_raw) & 1023u)) & 1023u);
    __shared__ __align__(8) uint64_t full[PF_WARPS][C::STAGES];
    __shared__ float s_m[PF_WARPS][16], s_l[PF_WARPS][16];
    __shared__ int s_bad;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, sp = blockIdx.y;
    const PagedSeq s = paged_seq(a, b);
    const int rows = s.live * a.G;
    const bool split = a.splits > 1 && s.kv > a.chunk;
    if (rows == 0 || (!split && sp > 0)) return;
    const int last = paged_limit(a, s, s.live - 1);
    const int k_begin = split ? sp * a.chunk : 0;
    const int k_end = split ? min(last, k_begin + a.chunk) : last;
    if (split && k_begin >= last) return;
    const int tiles = k_end > k_begin ? (k_end - k_begin + KT - 1) / KT : 0;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    unsigned char* ring = sm + warp * C::STAGES * C::STAGE;
    float* ring_sc = reinterpret_cast<float*>(sm + PF_WARPS * C::STAGES * C::STAGE) + warp * C::STAGES * 2 * KT;
    if (threadIdx.x == 0) {
        for (int i = 0; i < PF_WARPS * C::STAGES; ++i) mbar_init(&full[0][0] + i, 1);
        s_bad = 0;
        fence_barrier_init();
        prefetch_tensormap(&mK);
        prefetch_tensormap(&mV);
    }
    __syncthreads();

    // lane 0 loads: tile i of this warp holds the keys from k_begin + (warp + 4 i) KT on
    const int mine = tiles > warp ? (tiles - warp + PF_WARPS - 1) / PF_WARPS : 0;
    constexpr int PP = KT / PF_PIECE;
    int ids[PP];
    auto find_pages = [&](int i) {
        const int k0 = k_begin + (warp + PF_WARPS * i) * KT;
#pragma unroll
        for (int p = 0; p < PP; ++p) ids[p] = i < mine && k0 + p * PF_PIECE < s.kv ? paged_page(a, b, k0 + p * PF_PIECE) : -1;
    };
    auto issue = [&](int i) {
        const int st = i % C::STAGES, k0 = k_begin + (warp + PF_WARPS * i) * KT;
        uint64_t* bar = &full[warp][st];
        unsigned char* dst = ring + st * C::STAGE;
        int n = 0;
#pragma unroll
        for (int p = 0; p < PP; ++p) n += ids[p] >= 0;
        mbar_arrive_expect_tx(bar, n * PF_PIECE * (2 * C::ROWB + (Q8 ? 8 : 0)));
#pragma unroll
        for (int p = 0; p < PP; ++p) {
            if (ids[p] < 0) continue;
            const int off = (k0 + p * PF_PIECE) & ((1 << a.page_shift) - 1);
            if (Q8) {
                tma_load_4d(dst + p * PF_PIECE * D, &mK, 0, off, h, ids[p], bar);
                tma_load_4d(dst + C::HALF + p * PF_PIECE * D, &mV, 0, off, h, ids[p], bar);
                const size_t row = (((size_t)ids[p] * a.H + h) << a.page_shift) + off;
                float* sc = ring_sc + st * 2 * KT + p * PF_PIECE;
                bulk_load(sc, a.k_scale + row, PF_PIECE * 4, bar);
                bulk_load(sc + KT, a.v_scale + row, PF_PIECE * 4, bar);
            } else {
#pragma unroll
                for (int w = 0; w < D / 64; ++w) {
                    tma_load_4d(dst + w * KT * 128 + p * PF_PIECE * 128, &mK, 64 * w, off, h, ids[p], bar);
                    tma_load_4d(dst + C::HALF + w * KT * 128 + p * PF_PIECE * 128, &mV, 64 * w, off, h, ids[p], bar);
                }
            }
        }
    };
    if (lane == 0) {
        for (int i = 0; i < C::STAGES && i < mine; ++i) { find_pages(i); issue(i); }
        find_pages(C::STAGES);
    }

    // query fragments: row g (and g + 8) of the group's rows
    uint32_t qa[KS][4];
    {
        const T* q0 = nullptr;
        const T* q1 = nullptr;
        if (g < rows) q0 = reinterpret_cast<const T*>(a.q) + (size_t)(s.q0 + g / a.G) * a.q_stride + (size_t)(h * a.G + g % a.G) * D;
        if (g + 8 < rows)
            q1 = reinterpret_cast<const T*>(a.q) + (size_t)(s.q0 + (g + 8) / a.G) * a.q_stride + (size_t)(h * a.G + (g + 8) % a.G) * D;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            // elements of the lane's four slots of a k-step: 2t, 2t + 1, 2t + 8, 2t + 9, or with
            // INT8 four consecutive codes of the chunks the lane reads
            const int d0 = Q8 ? 64 * (k >> 2) + 16 * t + 4 * (k & 3) : 16 * k + 2 * t;
            const int d1 = Q8 ? d0 + 2 : d0 + 8;
            qa[k][0] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + d0) : 0u;
            qa[k][1] = q1 ? *reinterpret_cast<const uint32_t*>(q1 + d0) : 0u;
            qa[k][2] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + d1) : 0u;
            qa[k][3] = q1 ? *reinterpret_cast<const uint32_t*>(q1 + d1) : 0u;
        }
    }
    const int lim0 = g < rows ? paged_limit(a, s, g / a.G) : s.kv;
    const int lim1 = g + 8 < rows ? paged_limit(a, s, (g + 8) / a.G) : s.kv;
    const int lim_min = paged_limit(a, s, 0);
    float o[ND][4];
#pragma unroll
    for (int i = 0; i < ND; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    for (int i = 0; i < mine; ++i) {
        const int st = i % C::STAGES, k0 = k_begin + (warp + PF_WARPS * i) * KT;
        bool ok = mbar_wait_bounded(&full[warp][st], (i / C::STAGES) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
            if (lane == 0) { s_bad = 1; if (a.err) set_err(a.err, QV_DERR_TIMEOUT); }
            break;
        }
        unsigned char* kt = ring + st * C::STAGE;
        unsigned char* vt = kt + C::HALF;
        const uint32_t ka = smem_u32(kt), va = smem_u32(vt);
        float x[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
        if constexpr (!Q8) {
            const int r = (lane & 7) + ((lane >> 4) << 3), hi = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const uint32_t ch = (((2 * k) & 7) + hi) ^ (r & 7);
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    uint32_t b0, b1, b2, b3;
                    ldsm_x4(ka + (k >> 2) * KT * 128 + (8 * n + r) * 128 + (ch << 4), b0, b1, b2, b3);
                    pf_mma<DT>(x[n], qa[k], b0, b1);
                    pf_mma<DT>(x[n + 1], qa[k], b2, b3);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int key = 8 * n + g;
#pragma unroll
                for (int c = 0; c < D / 64; ++c) {
                    const int ch = (t + 4 * c) ^ (D == 128 ? key & 7 : (key >> 1) & 3);
                    const uint4 u = *reinterpret_cast<const uint4*>(kt + key * D + (ch << 4));
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(&u);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        pf_mma<DT>(x[n], qa[4 * c + k], pf_codes<DT>(__byte_perm(w[k], 0, 0x4140)),
                                   pf_codes<DT>(__byte_perm(w[k], 0, 0x4342)));
                }
            }
        }
        // base-2 logits; keys behind a row's limit leave
        const bool edge = k0 + KT > min(lim_min, k_end);
        float iv[Q8 ? NT : 1][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int key = k0 + 8 * n + 2 * t;
            if constexpr (Q8) {
                const float* sc = ring_sc + st * 2 * KT + 8 * n + 2 * t;
                float2 ks = *reinterpret_cast<const float2*>(sc);
                float2 vs = *reinterpret_cast<const float2*>(sc + KT);
                vs.x = vs.x < PF_MIN_SCALE ? PF_MIN_SCALE : vs.x;      // also a zero row, whose codes are 0
                vs.y = vs.y < PF_MIN_SCALE ? PF_MIN_SCALE : vs.y;
                if (edge) {
                    if (key >= s.kv) { ks.x = 0.f; vs.x = 1.f; }       // what lies there is not a row
                    if (key + 1 >= s.kv) { ks.y = 0.f; vs.y = 1.f; }
                }
                const float lx = __log2f(vs.x), ly = __log2f(vs.y);
                iv[n][0] = pf_ex2(-lx);
                iv[n][1] = pf_ex2(-ly);
                ks.x *= a.scale_log2;
                ks.y *= a.scale_log2;
                x[n][0] = fmaf(x[n][0], ks.x, lx);
                x[n][1] = fmaf(x[n][1], ks.y, ly);
                x[n][2] = fmaf(x[n][2], ks.x, lx);
                x[n][3] = fmaf(x[n][3], ks.y, ly);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) x[n][j] *= a.scale_log2;
            }
            if (edge) {
                if (key >= min(lim0, k_end)) x[n][0] = -INFINITY;
                if (key + 1 >= min(lim0, k_end)) x[n][1] = -INFINITY;
                if (key >= min(lim1, k_end)) x[n][2] = -INFINITY;
                if (key + 1 >= min(lim1, k_end)) x[n][3] = -INFINITY;
            }
        }
        float a0 = x[0][0], a1 = x[0][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            a0 = fmaxf(a0, fmaxf(x[n][0], x[n][1]));
            a1 = fmaxf(a1, fmaxf(x[n][2], x[n][3]));
        }
        if (__any_sync(0xffffffffu, a0 > m0 + PF_LAZY || a1 > m1 + PF_LAZY)) {
            a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, 1));
            a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, 1));
            a0 = fmaxf(a0, __shfl_xor_sync(0xffffffffu, a0, 2));
            a1 = fmaxf(a1, __shfl_xor_sync(0xffffffffu, a1, 2));
            const float n0 = a0 > m0 + PF_LAZY ? a0 : m0, n1 = a1 > m1 + PF_LAZY ? a1 : m1;
            const float f0 = m0 == -INFINITY ? 1.f : pf_ex2(m0 - n0), f1 = m1 == -INFINITY ? 1.f : pf_ex2(m1 - n1);
            m0 = n0;
            m1 = n1;
            l0 *= f0;
            l1 *= f1;
#pragma unroll
            for (int d = 0; d < ND; ++d) { o[d][0] *= f0; o[d][1] *= f0; o[d][2] *= f1; o[d][3] *= f1; }
        }
        const float b0 = m0 == -INFINITY ? 0.f : m0, b1 = m1 == -INFINITY ? 0.f : m1;
        uint32_t p[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float p0 = pf_ex2(x[n][0] - b0), p1 = pf_ex2(x[n][1] - b0);
            const float p2 = pf_ex2(x[n][2] - b1), p3 = pf_ex2(x[n][3] - b1);
            if constexpr (Q8) {
                l0 = fmaf(p0, iv[n][0], fmaf(p1, iv[n][1], l0));
                l1 = fmaf(p2, iv[n][0], fmaf(p3, iv[n][1], l1));
            } else {
                l0 += p0 + p1;
                l1 += p2 + p3;
            }
            p[n][0] = pf_cvt2<DT>(p0, p1);
            p[n][1] = pf_cvt2<DT>(p2, p3);
        }
        if (!Q8 && k0 + KT > s.kv) {
            // rows behind the sequence may hold anything: 0 times that must be 0
            for (int c = lane; c < KT * (D / 64) * 8; c += 32)
                if (k0 + ((c >> 3) % KT) >= s.kv) *reinterpret_cast<uint4*>(vt + c * 16) = make_uint4(0, 0, 0, 0);
            __syncwarp();
        }
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk) {
            const uint32_t pa[4] = {p[2 * kk][0], p[2 * kk][1], p[2 * kk + 1][0], p[2 * kk + 1][1]};
            if constexpr (!Q8) {
                const int r = 16 * kk + (lane & 7) + (((lane >> 3) & 1) << 3), hi = lane >> 4;
#pragma unroll
                for (int d = 0; d < ND; d += 2) {
                    uint32_t v0, v1, v2, v3;
                    ldsm_x4_t(va + (d >> 3) * KT * 128 + r * 128 + ((((d & 7) + hi) ^ (r & 7)) << 4), v0, v1, v2, v3);
                    pf_mma<DT>(o[d], pa, v0, v1);
                    pf_mma<DT>(o[d + 1], pa, v2, v3);
                }
            } else {
                // lane (g, t): bytes ND g .. of key rows 2t, 2t + 1, 2t + 8, 2t + 9; column n of tile d is element n ND + d
                uint32_t w[4][ND / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = 16 * kk + 2 * t + (e & 1) + 8 * (e >> 1);
                    if constexpr (D == 128) {
                        const uint4 u = *reinterpret_cast<const uint4*>(vt + key * D + ((g ^ (key & 7)) << 4));
                        w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
                    } else {
                        const uint2 u = *reinterpret_cast<const uint2*>(vt + key * D + (((g >> 1) ^ ((key >> 1) & 3)) << 4) + 8 * (g & 1));
                        w[e][0] = u.x; w[e][1] = u.y;
                    }
                }
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const uint32_t sel = (d & 3) | ((d & 3) << 4) | ((4 + (d & 3)) << 8) | ((4 + (d & 3)) << 12);
                    pf_mma<DT>(o[d], pa, pf_codes<DT>(__byte_perm(w[0][d >> 2], w[1][d >> 2], sel)),
                               pf_codes<DT>(__byte_perm(w[2][d >> 2], w[3][d >> 2], sel)));
                }
            }
        }
        __syncwarp();
        if (lane == 0 && i + C::STAGES < mine) {
            issue(i + C::STAGES);
            find_pages(i + C::STAGES + 1);
        }
    }
    // the warps' states join
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
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
    for (int d = 0; d < ND; ++d) {
        const int c0 = Q8 ? 2 * t * ND + d : 8 * d + 2 * t, c1 = Q8 ? c0 + ND : c0 + 1;
        so[g * LD + c0] = o[d][0];
        so[g * LD + c1] = o[d][1];
        so[(g + 8) * LD + c0] = o[d][2];
        so[(g + 8) * LD + c1] = o[d][3];
    }
    if (t == 0) { s_m[warp][g] = m0; s_m[warp][g + 8] = m1; s_l[warp][g] = l0; s_l[warp][g + 8] = l1; }
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

template <int DT, int D, bool Q8> static int pf_launch(const PagedArgs& a, cudaStream_t s) {
    using C = PfCfg<D, Q8>;
    CUtensorMap mK, mV;
    const int page = 1 << a.page_shift;
    const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    if (!paged_map_pages(&mK, a.k, DT, Q8, D, page, a.H, a.pages, PF_PIECE, sw) ||
        !paged_map_pages(&mV, a.v, DT, Q8, D, page, a.H, a.pages, PF_PIECE, sw))
        return QV_EINVAL;
    const cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<DT, D, Q8>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)C::SMEM);
    if (e != cudaSuccess) return set_cuda_error(e);
    paged_few_kernel<DT, D, Q8><<<dim3((unsigned)(a.B * a.H), a.splits), PF_THREADS, C::SMEM, s>>>(mK, mV, a);
    return check_launch();
}

template <int DT> static int pf_dispatch(const PagedArgs& a, int D, bool q8, cudaStream_t s) {
    if (D == 128) return q8 ? pf_launch<DT, 128, true>(a, s) : pf_launch<DT, 128, false>(a, s);
    return q8 ? pf_launch<DT, 64, true>(a, s) : pf_launch<DT, 64, false>(a, s);
}

int paged_few_launch(const PagedArgs& a, int dt, int D, bool q8, cudaStream_t s) {
    return dt == QV_BF16 ? pf_dispatch<QV_BF16>(a, D, q8, s) : pf_dispatch<QV_F16>(a, D, q8, s);
}

}  // namespace qv
