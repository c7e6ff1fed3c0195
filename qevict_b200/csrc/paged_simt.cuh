// Paged attention on the CUDA cores, fp32 (pages in fp32 or INT8): exact fp32
// products and sums, which the tensor cores do not give.
//
// A block takes BM query rows (row r of a chunk is token r / G, head r % G of
// one KV head's group, so that the group shares every K and V row it reads)
// and one range of keys, a tile at a time:  S = Q K^T, running maximum m and sum l
// of exp2(S - m), O = O exp2(m_old - m) + P V.  16 x 16 threads, each with BM/16
// rows of S and O in registers; K, V and P tiles in shared memory, P in K's place.
// Rows are padded by four floats so that the 16-byte reads of eight neighbouring
// rows fall on different banks.
//
// Bound by shared memory's reads: a 16-byte read takes four cycles a warp whether
// lanes share addresses or not, so a 4 x 4 block of S per thread (64 rows) reads
// for twice as long as it multiplies; 8 x 8 (128 rows, 128 keys, one block per SM)
// for as long.
#pragma once

#include "paged.cuh"

namespace qv {

constexpr int PS_THREADS = 256;

// Keys per tile: as many as rows, at least 64.
constexpr int paged_simt_keys(int BM) { return BM > 64 ? BM : 64; }

template <int D, int BM> constexpr size_t paged_simt_smem() {
    const int K = paged_simt_keys(BM), KP = K * (D + 4) > BM * (K + 4) ? K * (D + 4) : BM * (K + 4);   // K, then P
    return sizeof(float) * ((BM + K) * (D + 4) + KP);
}

// 16 bytes into shared memory in the background.
__device__ __forceinline__ void ps_copy16(float* dst, const float* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void ps_copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

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
__global__ void __launch_bounds__(PS_THREADS, BM > 64 ? 1 : 2) paged_simt_kernel(const PagedArgs a) {
    constexpr int LD = D + 4, RM = BM / 16, NC = D / 64, CH = D / 8;
    constexpr int KEYS = paged_simt_keys(BM), RK = KEYS / 16, LP = KEYS + 4;
    constexpr bool AHEAD = KEYS == 64;    // tiles loaded ahead through registers
    // QK sums: even and odd elements in pairs, where the registers allow
    constexpr bool PAIR = RM * RK <= 16;
    extern __shared__ __align__(16) float ps_sm[];
    float* sQ = ps_sm;                    // [BM][LD]
    float* sK = sQ + BM * LD;             // [KEYS][LD], then P [BM][LP]
    float* sV = sK + (KEYS * LD > BM * LP ? KEYS * LD : BM * LP);
    float* sP = sK;
    __shared__ int2 s_tile;
    const int h = blockIdx.y, sp = blockIdx.z;
    if (threadIdx.x < 32) {
        const int2 t = paged_find_tile(a, blockIdx.x, a.G, BM);
        if (threadIdx.x == 0) s_tile = t;
    } else if (threadIdx.x < 64 && blockIdx.x == 0 && h == 0 && sp == 0) {
        paged_check_rows(a, threadIdx.x - 32);
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
    // A thread loads 4-element chunk tx of rows ty, ty + 16, ... (and chunk tx + 16).  Tiles of 64 keys go through
    // registers, K of the next tile while P V runs, V while Q K^T does; larger ones are copied straight to shared
    // memory, V while Q K^T runs.  Keys past the range give 0: their P is 0 and V must be finite.
    constexpr int LR = KEYS / 16, LC = D / 64;
    float4 pre[AHEAD ? LR : 1][LC];
    auto row_of = [&](int key) {
        return (((size_t)paged_page(a, b, key) * a.H + h) << a.page_shift) + (key & ((1 << a.page_shift) - 1));
    };
    auto load4 = [&](const void* pages, float sc, size_t row, int col) {
        if constexpr (Q8) {
            const char4 e = *reinterpret_cast<const char4*>(reinterpret_cast<const int8_t*>(pages) + row * D + col);
            return make_float4(e.x * sc, e.y * sc, e.z * sc, e.w * sc);
        } else {
            return *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(pages) + row * D + col);
        }
    };
    // start: load a tile (ahead: into registers, otherwise towards dst)
    auto start = [&](const void* pages, const float* scales, int k0, float* dst) {
#pragma unroll
        for (int r = 0; r < LR; ++r) {
            const int key = k0 + ty + 16 * r;
            const bool in = key < k_end;
            const size_t row = in ? row_of(key) : 0;
            float sc = 0.f;
            if (Q8 && in) sc = scales[row];
#pragma unroll
            for (int c = 0; c < LC; ++c) {
                float* at = dst + (ty + 16 * r) * LD + 4 * tx + 64 * c;
                if (AHEAD) pre[AHEAD ? r : 0][c] = in ? load4(pages, sc, row, 4 * tx + 64 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
                else if (!Q8 && in) ps_copy16(at, reinterpret_cast<const float*>(pages) + row * D + 4 * tx + 64 * c);
                else *reinterpret_cast<float4*>(at) = in ? load4(pages, sc, row, 4 * tx + 64 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
        }
    };
    // finish: its elements are in dst (this thread's; a barrier follows)
    auto finish = [&](float* dst) {
        if constexpr (AHEAD) {
#pragma unroll
            for (int r = 0; r < LR; ++r)
#pragma unroll
                for (int c = 0; c < LC; ++c) *reinterpret_cast<float4*>(dst + (ty + 16 * r) * LD + 4 * tx + 64 * c) = pre[r][c];
        } else {
            ps_copies_done();
        }
    };

    if (AHEAD && k_begin < k_end) start(a.k, a.k_scale, k_begin, sK);
    for (int k0 = k_begin; k0 < k_end; k0 += KEYS) {
        __syncthreads();                  // the last tile's P and V have been read
        if (!AHEAD) start(a.k, a.k_scale, k0, sK);
        finish(sK);
        __syncthreads();
        start(a.v, a.v_scale, k0, sV);
        float acc[RM][RK];
        if constexpr (PAIR) {
            uint64_t acc2[RM][RK];
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RK; ++j) acc2[i][j] = ps_pack(0.f, 0.f);
#pragma unroll 4
            for (int d = 0; d < D; d += 4) {
                ulonglong2 q4[RM], k4[RK];
#pragma unroll
                for (int i = 0; i < RM; ++i) q4[i] = *reinterpret_cast<const ulonglong2*>(sQ + (ty * RM + i) * LD + d);
#pragma unroll
                for (int j = 0; j < RK; ++j) k4[j] = *reinterpret_cast<const ulonglong2*>(sK + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < RK; ++j)
                        acc2[i][j] = ps_fma2(q4[i].y, k4[j].y, ps_fma2(q4[i].x, k4[j].x, acc2[i][j]));
            }
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RK; ++j) {
                    float e, f;
                    ps_unpack(acc2[i][j], e, f);
                    acc[i][j] = e + f;
                }
        } else {
#pragma unroll
            for (int i = 0; i < RM; ++i)
#pragma unroll
                for (int j = 0; j < RK; ++j) acc[i][j] = 0.f;
            // (two elements at a time: the next ones' reads fit beside the sums)
#pragma unroll 8
            for (int d = 0; d < D; d += 2) {
                float2 q2[RM], k2[RK];
#pragma unroll
                for (int i = 0; i < RM; ++i) q2[i] = *reinterpret_cast<const float2*>(sQ + (ty * RM + i) * LD + d);
#pragma unroll
                for (int j = 0; j < RK; ++j) k2[j] = *reinterpret_cast<const float2*>(sK + (tx + 16 * j) * LD + d);
#pragma unroll
                for (int i = 0; i < RM; ++i)
#pragma unroll
                    for (int j = 0; j < RK; ++j) acc[i][j] = fmaf(q2[i].y, k2[j].y, fmaf(q2[i].x, k2[j].x, acc[i][j]));
            }
        }
        __syncthreads();                  // K has been read: P takes its place
        finish(sV);
        if (AHEAD && k0 + KEYS < k_end) start(a.k, a.k_scale, k0 + KEYS, sK);
#pragma unroll
        for (int i = 0; i < RM; ++i) {
            float mx = m[i];
#pragma unroll
            for (int j = 0; j < RK; ++j) {
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
                for (int j = 0; j < 2; ++j) o[i][c][j] = ps_mul2(o[i][c][j], ps_pack(f, f));
#pragma unroll
            for (int j = 0; j < RK; ++j) {
                const float p = exp2f(acc[i][j] - base);
                l[i] += p;
                sP[(ty * RM + i) * LP + tx + 16 * j] = p;
            }
        }
        __syncthreads();
#pragma unroll 2
        for (int k = 0; k < KEYS; k += 4) {
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
