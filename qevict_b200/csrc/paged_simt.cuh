// Paged attention on the CUDA cores, fp32 (pages in fp32 or INT8): exact fp32
// products and sums, which the tensor cores do not give.
//
// A block takes BM query rows (row r of a chunk is token r / G, head r % G of
// one KV head's group, so that the group shares every K and V row it reads)
// and one range of keys, 64 at a time:  S = Q K^T, running maximum m and sum l
// of exp2(S - m), O = O exp2(m_old - m) + P V.  16 x 16 threads, each with
// BM/16 rows x 4 keys of S and BM/16 rows x D/16 columns of O in registers;
// K, V and P tiles in shared memory, P in K's place.  Rows are padded by four
// floats so that the 16-byte reads of eight neighbouring rows fall on
// different banks.
#pragma once

#include "paged.cuh"

namespace qv {

constexpr int PS_KEYS = 64;
constexpr int PS_THREADS = 256;

template <int D, int BM> constexpr size_t paged_simt_smem() {
    return sizeof(float) * (BM + 2 * PS_KEYS) * (D + 4);
}

__device__ __forceinline__ uint64_t ps_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void ps_unpack(uint64_t r, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(r));
}
__device__ __forceinline__ uint64_t ps_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t ps_mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

template <int D, bool Q8, int BM>
__global__ void __launch_bounds__(PS_THREADS, 2) paged_simt_kernel(const PagedArgs a) {
    constexpr int LD = D + 4, RM = BM / 16, NC = D / 64, CH = D / 8, LP = PS_KEYS + 4;
    extern __shared__ __align__(16) float ps_sm[];
    float* sQ = ps_sm;                    // [BM][LD]
    float* sK = sQ + BM * LD;             // [64][LD], then P [BM][PS_KEYS + 4]
    float* sV = sK + PS_KEYS * LD;        // [64][LD]
    float* sP = sK;
    __shared__ int2 s_tile;
    const int h = blockIdx.y, sp = blockIdx.z;
    if (threadIdx.x < 32) {
        const int2 t = paged_find_tile(a, blockIdx.x, a.G, BM);
        if (threadIdx.x == 0) s_tile = t;
    }
    __syncthreads();
    const int b = s_tile.x;
    if (b < 0) return;
    const PagedSeq s = paged_seq(a, b);
    const int row0 = s_tile.y * BM, rows = min(BM, s.live * a.G - row0);
    const int Hq = a.H * a.G;
    // keys of this block: its split, up to what the tile's last row sees
    const int last = paged_limit(a, s, (row0 + rows - 1) / a.G);
    const bool split = a.splits > 1 && s.kv > a.chunk;
    if (!split && sp > 0) return;
    const int k_begin = split ? sp * a.chunk : 0;
    const int k_end = split ? min(last, k_begin + a.chunk) : last;
    if (split && sp > 0 && k_begin >= last) return;
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;

    for (int i = tid; i < BM * CH; i += PS_THREADS) {
        const int r = i / CH, c = 8 * (i % CH);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
        if (r < rows) {
            const int row = row0 + r;
            widen8<QV_F32>(load8<QV_F32>(a.q, (size_t)(s.q0 + row / a.G) * a.q_stride + (size_t)(h * a.G + row % a.G) * D + c), x);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sQ[r * LD + c + j] = x[j];
    }
    int limit[RM];
    float m[RM], l[RM];
    uint64_t o[RM][NC][2];                // pairs of columns
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = row0 + ty * RM + i;
        limit[i] = ty * RM + i < rows ? paged_limit(a, s, r / a.G) : 0;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[i][c][0] = o[i][c][1] = ps_pack(0.f, 0.f);
    }
    // A thread loads 4-element chunk tx of rows ty, ty + 16, ... (and chunk tx + 16): K of the next tile while P V
    // runs, V while Q K^T does, both through registers.  Keys past the range give 0: their P is 0 and V must be
    // finite.
    constexpr int LR = PS_KEYS / 16, LC = D / 64;
    float4 pre[LR][LC];
    auto fetch = [&](const void* pages, const float* scales, int k0) {
#pragma unroll
        for (int r = 0; r < LR; ++r) {
            const int key = k0 + ty + 16 * r;
            const bool in = key < k_end;
            const size_t row = in ? (((size_t)paged_page(a, b, key) * a.H + h) << a.page_shift) + (key & ((1 << a.page_shift) - 1)) : 0;
            float sc = 0.f;
            if (Q8 && in) sc = scales[row];
#pragma unroll
            for (int c = 0; c < LC; ++c) {
                pre[r][c] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (!in) continue;
                if constexpr (Q8) {
                    const char4 e = *reinterpret_cast<const char4*>(reinterpret_cast<const int8_t*>(pages) + row * D + 4 * tx + 64 * c);
                    pre[r][c] = make_float4(e.x * sc, e.y * sc, e.z * sc, e.w * sc);
                } else {
                    pre[r][c] = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(pages) + row * D + 4 * tx + 64 * c);
                }
            }
        }
    };
    auto put = [&](float* dst) {
#pragma unroll
        for (int r = 0; r < LR; ++r)
#pragma unroll
            for (int c = 0; c < LC; ++c) *reinterpret_cast<float4*>(dst + (ty + 16 * r) * LD + 4 * tx + 64 * c) = pre[r][c];
    };

    if (k_begin < k_end) fetch(a.k, a.k_scale, k_begin);
    for (int k0 = k_begin; k0 < k_end; k0 += PS_KEYS) {
        __syncthreads();                  // the last tile's P and V have been read
        put(sK);
        __syncthreads();
        fetch(a.v, a.v_scale, k0);
        uint64_t acc2[RM][4];             // even and odd elements' sums
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc2[i][j] = ps_pack(0.f, 0.f);
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            ulonglong2 q4[RM], k4[4];
#pragma unroll
            for (int i = 0; i < RM; ++i) q4[i] = *reinterpret_cast<const ulonglong2*>(sQ + (ty * RM + i) * LD + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const ulonglong2*>(sK + (tx + 16 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc2[i][j] = ps_fma2(q4[i].y, k4[j].y, ps_fma2(q4[i].x, k4[j].x, acc2[i][j]));
        }
        __syncthreads();                  // K has been read: P takes its place
        put(sV);
        if (k0 + PS_KEYS < k_end) fetch(a.k, a.k_scale, k0 + PS_KEYS);
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            float acc[4], mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float e, f;
                ps_unpack(acc2[i][j], e, f);
                acc[j] = k0 + tx + 16 * j < limit[i] ? (e + f) * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, acc[j]);
            }
#pragma unroll
            for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
            const float base = mx == -INFINITY ? 0.f : mx;   // nothing seen yet: every term is 0
            const float f = exp2f(m[i] - base);
            m[i] = mx;
            l[i] *= f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < 2; ++j) o[i][c][j] = ps_mul2(o[i][c][j], ps_pack(f, f));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(acc[j] - base);
                l[i] += p;
                sP[(ty * RM + i) * LP + tx + 16 * j] = p;
            }
        }
        __syncthreads();
#pragma unroll 2
        for (int k = 0; k < PS_KEYS; k += 4) {
            float4 p4[RM];
#pragma unroll
            for (int i = 0; i < RM; ++i) p4[i] = *reinterpret_cast<const float4*>(sP + (ty * RM + i) * LP + k);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const ulonglong2 v4 = *reinterpret_cast<const ulonglong2*>(sV + (k + kk) * LD + 64 * c + 4 * tx);
#pragma unroll
                    for (int i = 0; i < RM; ++i) {
                        const float p = reinterpret_cast<const float*>(&p4[i])[kk];
                        o[i][c][0] = ps_fma2(ps_pack(p, p), v4.x, o[i][c][0]);
                        o[i][c][1] = ps_fma2(ps_pack(p, p), v4.y, o[i][c][1]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RM; ++i) {
#pragma unroll
        for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
        const int r = ty * RM + i;
        if (r >= rows) continue;
        const int row = row0 + r;
        const size_t orow = (size_t)(s.q0 + row / a.G) * Hq + h * a.G + row % a.G;
        const float inv = split ? 1.f : l[i] > 0.f ? 1.f / l[i] : l[i];   // no key seen: 0 (a NaN sum stays NaN)
        const size_t prow = split ? (size_t)sp * a.total_q * Hq + orow : orow;
        float* out = split ? a.part_o : reinterpret_cast<float*>(a.out);
        if (split && tx == 0) {
            a.part_ml[2 * prow] = m[i];
            a.part_ml[2 * prow + 1] = l[i];
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float4 x;
            ps_unpack(o[i][c][0], x.x, x.y);
            ps_unpack(o[i][c][1], x.z, x.w);
            *reinterpret_cast<float4*>(out + prow * D + 64 * c + 4 * tx) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
    }
}

}  // namespace qv
