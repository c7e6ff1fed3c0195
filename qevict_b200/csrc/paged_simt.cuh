// Paged attention on the CUDA cores (fp32 arithmetic for every type).
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

template <int DT, bool Q8> __device__ __forceinline__ void paged_load8(const void* p, const float* scale, size_t row,
                                                                       int D, int col, float* x) {
    if constexpr (Q8)
        widen8_codes(*reinterpret_cast<const uint2*>(reinterpret_cast<const int8_t*>(p) + row * D + col), scale[row], x);
    else
        widen8<DT>(load8<DT>(p, row * D + col), x);
}

template <int DT, int D, bool Q8, int BM>
__global__ void __launch_bounds__(PS_THREADS) paged_simt_kernel(const PagedArgs a) {
    constexpr int LD = D + 4, RM = BM / 16, NC = D / 64, CH = D / 8;
    extern __shared__ __align__(16) float ps_sm[];
    float* sQ = ps_sm;                    // [BM][LD]
    float* sK = sQ + BM * LD;             // [64][LD], then P [BM][PS_KEYS + 4]
    float* sV = sK + PS_KEYS * LD;        // [64][LD]
    float* sP = sK;
    constexpr int LP = PS_KEYS + 4;
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
            widen8<DT>(load8<DT>(a.q, (size_t)(s.q0 + row / a.G) * a.q_stride + (size_t)(h * a.G + row % a.G) * D + c), x);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) sQ[r * LD + c + j] = x[j];
    }
    int limit[RM];
    float m[RM], l[RM], o[RM][NC][4];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
        const int r = row0 + ty * RM + i;
        limit[i] = ty * RM + i < rows ? paged_limit(a, s, r / a.G) : 0;
        m[i] = -INFINITY;
        l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][c][j] = 0.f;
    }

    for (int k0 = k_begin; k0 < k_end; k0 += PS_KEYS) {
        __syncthreads();
        for (int i = tid; i < PS_KEYS * CH; i += PS_THREADS) {
            const int r = i / CH, c = 8 * (i % CH), key = k0 + r;
            float x[8], y[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = y[j] = 0.f;   // keys past the range: P is 0 and V must be finite
            if (key < k_end) {
                const size_t row = (((size_t)paged_page(a, b, key) * a.H + h) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
                paged_load8<DT, Q8>(a.k, a.k_scale, row, D, c, x);
                paged_load8<DT, Q8>(a.v, a.v_scale, row, D, c, y);
            }
            float4* kd = reinterpret_cast<float4*>(sK + r * LD + c);
            float4* vd = reinterpret_cast<float4*>(sV + r * LD + c);
            kd[0] = make_float4(x[0], x[1], x[2], x[3]);
            kd[1] = make_float4(x[4], x[5], x[6], x[7]);
            vd[0] = make_float4(y[0], y[1], y[2], y[3]);
            vd[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
        __syncthreads();
        float acc[RM][4];
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; d += 4) {
            float4 q4[RM], k4[4];
#pragma unroll
            for (int i = 0; i < RM; ++i) q4[i] = *reinterpret_cast<const float4*>(sQ + (ty * RM + i) * LD + d);
#pragma unroll
            for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * LD + d);
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = fmaf(q4[i].w, k4[j].w, fmaf(q4[i].z, k4[j].z, fmaf(q4[i].y, k4[j].y, fmaf(q4[i].x, k4[j].x, acc[i][j]))));
        }
        __syncthreads();   // K has been read: P takes its place
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[i][j] = k0 + tx + 16 * j < limit[i] ? acc[i][j] * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, acc[i][j]);
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
                for (int j = 0; j < 4; ++j) o[i][c][j] *= f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p = exp2f(acc[i][j] - base);
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
                    const float4 v4 = *reinterpret_cast<const float4*>(sV + (k + kk) * LD + 64 * c + 4 * tx);
#pragma unroll
                    for (int i = 0; i < RM; ++i) {
                        const float p = reinterpret_cast<const float*>(&p4[i])[kk];
                        o[i][c][0] = fmaf(p, v4.x, o[i][c][0]);
                        o[i][c][1] = fmaf(p, v4.y, o[i][c][1]);
                        o[i][c][2] = fmaf(p, v4.z, o[i][c][2]);
                        o[i][c][3] = fmaf(p, v4.w, o[i][c][3]);
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
        if (split) {
            const size_t prow = (size_t)sp * a.total_q * Hq + orow;
            if (tx == 0) {
                a.part_ml[2 * prow] = m[i];
                a.part_ml[2 * prow + 1] = l[i];
            }
#pragma unroll
            for (int c = 0; c < NC; ++c)
                *reinterpret_cast<float4*>(a.part_o + prow * D + 64 * c + 4 * tx) =
                    make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
        } else {
            const float inv = l[i] > 0.f ? 1.f / l[i] : l[i];   // no key seen: 0 (a NaN sum stays NaN)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) st<DT>(a.out, orow * D + 64 * c + 4 * tx + j, o[i][c][j] * inv);
        }
    }
}

}  // namespace qv
