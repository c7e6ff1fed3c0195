// The paged KV cache: norm and rotation of query / key heads, the same with
// the new keys and values written into pages, and pages read back.
//
// Per head row x of D elements, in fp32 throughout and rounded once at the
// store:
//   norm      y = x * (mean(x^2) + eps)^(-1/2) * w          (optional)
//   rotation  pair (a, b) -> (a c - b s, b c + a s), i < rot/2, with (a, b) =
//             (y[i], y[i + rot/2]) or, interleaved, (y[2i], y[2i+1]); (c, s)
//             from the fp32 table row of the token's position
//   8 bits    scale = max|y| / 127 (fp32), code = rint(y / scale)
//
// All three are bound by HBM: every row is read and written once.  A block
// takes one token, and each of its threads one 8-element chunk position of
// all the token's heads, so that the table row and the norm weights are
// loaded once per token into registers (a table row is two to four times a
// 16-bit head row); the next two rows load while two are worked on.  16383
// tokens of 64 normed fp16 heads: 98 us, 5.5 TB/s (84 % of a copy's rate);
// without the loads ahead 116 us.
#include <math.h>

#include "paged.cuh"

namespace qv {

constexpr int PH_MOST = 256;     // threads of a block, at most
constexpr int PH_ROWS = 2;       // head rows per step of a thread; the next step's are in flight meanwhile

struct HeadArgs {
    const void* q;
    const void* k;
    const void* v;
    int64_t qs, ks, vs;          // token strides in elements
    const void* qw;              // [D] or null
    const void* kw;
    float eps;
    const float* table;          // [max_pos][rot]: cos | sin, or null
    const int32_t* pos;
    int max_pos, rot, interleaved;
    int Hq, H, D;
    void* q_out;                 // [tokens][Hq][D]
    void* k_out;                 // [tokens][H][D] (no pages)
    void* kp;                    // pages
    void* vp;
    float* k_scale;
    float* v_scale;
    const int64_t* slots;
    int64_t n_slots;
    int page_shift;
    int32_t* err;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

enum { PH_ROWS_ONLY = 0, PH_PAGES = 1, PH_PAGES8 = 2 };

// Packed fp32 pairs.
__device__ __forceinline__ uint64_t ph_pack(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void ph_unpack(uint64_t r, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(r));
}
__device__ __forceinline__ uint64_t ph_mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t ph_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t ph_sub2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t ph_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// TPR threads share a head row (8 elements each, TPR a power of two >= D/8).  A
// block walks its token's query, key and value heads one kind after the other
// (gridDim.y = 1), or one kind (blockIdx.y; few tokens).
template <int DT, int TPR, int MODE>
__global__ void __launch_bounds__(PH_MOST, DT == QV_F32 ? 2 : 3) heads_kernel(const __grid_constant__ HeadArgs a) {
    using T = typename Elt<DT>::T;
    constexpr int KINDS = MODE == PH_ROWS_ONLY ? 2 : 3;
    const size_t t = blockIdx.x;
    const int c = threadIdx.x & (TPR - 1), hl = threadIdx.x / TPR, hpb = blockDim.x / TPR;
    const int lane = threadIdx.x & 31, warp_row = (threadIdx.x >> 5) * (32 / TPR);
    const bool on = 8 * c < a.D;
    int kind = gridDim.y == 1 ? 0 : blockIdx.y;
    const int kind_end = gridDim.y == 1 ? KINDS : kind + 1;
    const T* in = nullptr;      // the kind's rows at this thread's chunk, and how many
    int nh = 0;
    auto enter = [&]() {
        in = kind == 0 ? reinterpret_cast<const T*>(a.q) + t * a.qs : kind == 1 ? reinterpret_cast<const T*>(a.k) + t * a.ks
                                                                                : reinterpret_cast<const T*>(a.v) + t * a.vs;
        in += 8 * c;
        nh = kind == 0 ? a.Hq : a.H;
    };
    Chunk8<DT> raw[PH_ROWS], ahead[PH_ROWS];   // a lane behind the head's end holds 0 throughout: row sums include it
#pragma unroll
    for (int i = 0; i < PH_ROWS; ++i)
#pragma unroll
        for (int w = 0; w < (DT == QV_F32 ? 2 : 1); ++w) raw[i].u[w] = ahead[i].u[w] = make_uint4(0, 0, 0, 0);
    auto fetch = [&](int r0, Chunk8<DT>* raw) {
#pragma unroll
        for (int i = 0; i < PH_ROWS; ++i) {
            const int r = r0 + i * hpb + hl;
            if (r < nh && on) raw[i] = load8<DT>(in, (size_t)(r * a.D));
        }
    };
    enter();
    fetch(0, raw);                                            // before anything waits for the position's table row

    int64_t slot = -1;
    if (MODE != PH_ROWS_ONLY) {
        slot = a.slots[t];
        if (slot >= a.n_slots) {
            if (threadIdx.x == 0 && a.err) set_err(a.err, QV_DERR_CAPACITY);
            slot = -1;
        }
    }
    // the thread's rotation factors and where its partner elements sit: 4-element
    // sub-chunk u = 2c + s of a half-layout head pairs with u +- rot/8
    uint64_t cs[4], sn[4];
    bool turn[2] = {false, false};
    int src[2] = {lane, lane};
    const int r8 = a.rot >> 3;
    if (a.table && kind < 2) {
        const int p = a.pos[t];
        const bool ok = (unsigned)p < (unsigned)a.max_pos;
        if (MODE != PH_ROWS_ONLY && !ok && threadIdx.x == 0 && a.err) set_err(a.err, QV_DERR_TABLE);
        const float* row = a.table + (size_t)(ok ? p : 0) * a.rot;
        const float bad = ok ? 0.f : NAN;   // a position outside the table shows as NaN
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int u = 2 * c + s;
            turn[s] = 4 * u < a.rot;
            float4 cv = make_float4(0.f, 0.f, 0.f, 0.f), sv = cv;
            if (turn[s]) {
                // interleaved: both sub-chunks of a thread read their two pairs of the same 4
                const int i0 = a.interleaved ? 4 * c : 4 * (u < r8 ? u : u - r8);
                cv = *reinterpret_cast<const float4*>(row + i0);
                sv = *reinterpret_cast<const float4*>(row + a.rot / 2 + i0);
                if (!a.interleaved) src[s] = lane - c + ((u < r8 ? u + r8 : u - r8) >> 1);
            }
            const float* ce = reinterpret_cast<const float*>(&cv);
            const float* se = reinterpret_cast<const float*>(&sv);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const int j0 = a.interleaved ? 2 * s + (i >> 1) : i, j1 = a.interleaved ? j0 : i + 1;
                const float s0 = se[j0] + bad, s1 = se[j1] + bad;
                cs[2 * s + i / 2] = ph_pack(ce[j0] + bad, ce[j1] + bad);
                sn[2 * s + i / 2] = a.interleaved ? ph_pack(-s0, s0) : u < r8 ? ph_pack(-s0, -s1) : ph_pack(s0, s1);
            }
        }
    }
    const float inv_d = 1.f / (float)a.D;
    const bool swap = r8 & 1;                            // half layout: partners sit in the other sub-chunk

    for (bool again = false; kind < kind_end; ++kind, again = true) {
        if (again) { enter(); fetch(0, raw); }
        const void* weight = kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr;
        const bool rotate = a.table && kind < 2;
        uint64_t w2[4] = {0, 0, 0, 0};
        if (weight && on) {
            float w[8];
            widen8<DT>(load8<DT>(weight, 8 * c), w);
#pragma unroll
            for (int j = 0; j < 4; ++j) w2[j] = ph_pack(w[2 * j], w[2 * j + 1]);
        }
        // where the kind's rows go: contiguous, or the slot's row of each head
        const bool paged = MODE != PH_ROWS_ONLY && kind > 0;
        T* out = kind == 0 ? reinterpret_cast<T*>(a.q_out) + t * a.Hq * a.D : reinterpret_cast<T*>(a.k_out) + t * a.H * a.D;
        size_t row0 = 0;
        if (paged) {
            const size_t pg = (size_t)(slot >> a.page_shift), off = (size_t)slot & ((1u << a.page_shift) - 1);
            row0 = ((pg * a.H) << a.page_shift) + off;
            if (MODE == PH_PAGES) out = reinterpret_cast<T*>(kind == 2 ? a.vp : a.kp) + row0 * a.D;
        }
        out += 8 * c;
        const int step = paged ? a.D << a.page_shift : a.D;   // between heads
        const bool write = on && !(paged && slot < 0);

        for (int r0 = 0; r0 < nh; r0 += hpb * PH_ROWS) {
            if (r0 + warp_row >= nh) break;                   // the same for the whole warp
            fetch(r0 + hpb * PH_ROWS, ahead);
            float xs[PH_ROWS][8];                                   // two rows at a time: their chains overlap
#pragma unroll
            for (int i = 0; i < 2; ++i) widen8<DT>(raw[i], xs[i]);
            if (weight) {
                float ss[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float* x = xs[i];
                    uint64_t s2 = ph_mul2(ph_pack(x[0], x[1]), ph_pack(x[0], x[1]));
#pragma unroll
                    for (int j = 2; j < 8; j += 2) s2 = ph_fma2(ph_pack(x[j], x[j + 1]), ph_pack(x[j], x[j + 1]), s2);
                    float s1;
                    ph_unpack(s2, ss[i], s1);
                    ss[i] += s1;
                }
#pragma unroll
                for (int o = TPR / 2; o > 0; o >>= 1)
#pragma unroll
                    for (int i = 0; i < 2; ++i) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float* x = xs[i];
                    const float inv = rsqrtf(fmaf(ss[i], inv_d, a.eps));
                    const uint64_t inv2 = ph_pack(inv, inv);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        ph_unpack(ph_mul2(ph_mul2(ph_pack(x[2 * j], x[2 * j + 1]), inv2), w2[j]), x[2 * j], x[2 * j + 1]);
                }
            }
            if (rotate) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float* x = xs[i];
                    float y[8];
                    if (a.interleaved) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) y[j] = x[j ^ 1];
                    } else {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            y[j] = __shfl_sync(0xffffffffu, swap ? x[4 + j] : x[j], src[0]);
                            y[4 + j] = __shfl_sync(0xffffffffu, swap ? x[j] : x[4 + j], src[1]);
                        }
                    }
#pragma unroll
                    for (int s = 0; s < 2; ++s)
                        if (turn[s]) {
#pragma unroll
                            for (int j = 4 * s; j < 4 * s + 4; j += 2)
                                ph_unpack(ph_fma2(ph_pack(x[j], x[j + 1]), cs[j / 2], ph_mul2(ph_pack(y[j], y[j + 1]), sn[j / 2])),
                                          x[j], x[j + 1]);
                        }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = r0 + i * hpb + hl;
                float* x = xs[i];
                if (MODE != PH_PAGES8 || kind == 0) {
                    if (write && r < nh) store8<DT>(out, (size_t)((int64_t)r * step), x);
                    continue;
                }
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(x[j]));
#pragma unroll
                for (int o = TPR / 2; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                if (!write || r >= nh) continue;
                const size_t row = row0 + ((size_t)r << a.page_shift);
                const float scale = __fdiv_rn(m, 127.f);
                // x / scale as a product, at most 1.5 ulp off: 1.5 2^-17 below 128.  Where that leaves a code open (within
                // 2^-15 of a tie), or the scale's reciprocal leaves fp32's range, the row's lane divides.  A row that is not
                // finite: codes of 0 and a scale that is not finite read back as NaN
                const bool plain = scale > 1e-37f && scale < INFINITY;
                const float back = plain ? __fdiv_rn(1.f, scale) : 0.f;
                const uint64_t back2 = ph_pack(back, back), high2 = ph_pack(12582912.f, 12582912.f);
                int e[8];
                float off = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    // |f| <= 127 but for its rounding, so the nearest integer is in range; with 1.5 2^23 added it stands in
                    // the low bits
                    const uint64_t f2 = ph_mul2(ph_pack(x[j], x[j + 1]), back2), t2 = ph_add2(f2, high2);
                    float t0, t1, d0, d1;
                    ph_unpack(t2, t0, t1);
                    ph_unpack(ph_sub2(f2, ph_sub2(t2, high2)), d0, d1);
                    off = fmaxf(off, fmaxf(fabsf(d0), fabsf(d1)));
                    e[j] = __float_as_int(t0);
                    e[j + 1] = __float_as_int(t1);
                }
                const bool open = !plain || off > 0.5f - 0x1p-15f;
                if (open) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        // (a subnormal scale is itself rounded: the quotient may pass 127)
                        const float f = scale > 0.f && scale < INFINITY ? fminf(fmaxf(__fdiv_rn(x[j], scale), -127.f), 127.f) : 0.f;
                        e[j] = __float_as_int(__fadd_rn(f, 12582912.f));
                    }
                }
                uint32_t u[2];
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    u[j / 4] = __byte_perm(__byte_perm(e[j], e[j + 1], 0x0040), __byte_perm(e[j + 2], e[j + 3], 0x0040), 0x5410);
                *reinterpret_cast<uint2*>(reinterpret_cast<int8_t*>(kind == 2 ? a.vp : a.kp) + row * a.D + 8 * c) = make_uint2(u[0], u[1]);
                if (c == 0) (kind == 2 ? a.v_scale : a.k_scale)[row] = scale;
            }
#pragma unroll
            for (int i = 0; i < PH_ROWS; ++i) raw[i] = ahead[i];
        }
    }
}

// ---------------------------------------------------------------- read back
constexpr int PG_TOKENS = 8;     // tokens per block
constexpr int PG_THREADS = 256;
// K chunks, and V chunks, in flight per thread: 131072 bf16 tokens of 8 heads of 128 read back in 177 us (6.1 TB/s,
// 92 % of a copy's rate) with two, 187 with four and fewer warps
constexpr int PG_FLIGHT = 2;

struct GatherArgs {
    const void* k;
    const void* v;
    const float* k_scale;
    const float* v_scale;
    int32_t* err;
    const int32_t* block_table;
    const int32_t* kv_lens;
    const int32_t* cu_kv;
    void* k_out;
    void* v_out;
    int pages, H, D, page_shift, max_pages, B, total;
};

template <int DT, bool Q8>
__global__ void __launch_bounds__(PG_THREADS) gather_kernel(const GatherArgs a) {
    __shared__ int64_t s_row[PG_TOKENS];   // the token's row of head 0 in the pages, or -1
    const int t0 = blockIdx.x * PG_TOKENS;
    if (blockIdx.x == 0 && a.err) {        // a sequence cut by the next one's rows, or by the rows there are
        for (int b = threadIdx.x; b < a.B; b += PG_THREADS) {
            const int at = a.cu_kv[b], to = a.cu_kv[b + 1], kv = a.kv_lens[b];
            if (at < 0 || to < at || kv < 0 || kv > to - at || (kv > 0 && at > a.total - kv)) set_err(a.err, QV_DERR_CAPACITY);
        }
    }
    if (threadIdx.x < PG_TOKENS) {
        const int t = t0 + threadIdx.x;
        int64_t row = -1;
        if (t < a.total) {
            const int b = paged_find_token(a.cu_kv, a.B, t);
            const int pos = t - a.cu_kv[b];
            if (t < a.cu_kv[a.B] && pos >= 0 && pos < a.kv_lens[b]) {
                const int pi = pos >> a.page_shift;
                const int pg = pi < a.max_pages ? a.block_table[(size_t)b * a.max_pages + pi] : -1;
                if ((unsigned)pg < (unsigned)a.pages)
                    row = (((int64_t)pg * a.H) << a.page_shift) + (pos & ((1 << a.page_shift) - 1));
                else if (a.err)
                    set_err(a.err, pi < a.max_pages ? QV_DERR_TABLE : QV_DERR_CAPACITY);
            }
        }
        s_row[threadIdx.x] = row;
    }
    __syncthreads();
    const int per_row = a.D >> 3, per_tok = a.H * per_row, n = PG_TOKENS * per_tok;
    for (int i0 = threadIdx.x; i0 < n; i0 += PG_THREADS * PG_FLIGHT) {
        int64_t src[PG_FLIGHT], dst[PG_FLIGHT];
        Chunk8<DT> kr[PG_FLIGHT], vr[PG_FLIGHT];
        uint2 kc[PG_FLIGHT], vc[PG_FLIGHT];
        float kscale[PG_FLIGHT], vscale[PG_FLIGHT];
#pragma unroll
        for (int f = 0; f < PG_FLIGHT; ++f) {
            const int i = i0 + f * PG_THREADS;
            src[f] = -1;
            if (i >= n) continue;
            const int tt = i / per_tok, rem = i - tt * per_tok, h = rem / per_row, c = rem - h * per_row;
            if (s_row[tt] < 0) continue;
            const int64_t row = s_row[tt] + ((int64_t)h << a.page_shift);
            src[f] = row * a.D + 8 * c;
            dst[f] = ((int64_t)(t0 + tt) * a.H + h) * a.D + 8 * c;
            if (Q8) {
                kc[f] = *reinterpret_cast<const uint2*>(reinterpret_cast<const int8_t*>(a.k) + src[f]);
                vc[f] = *reinterpret_cast<const uint2*>(reinterpret_cast<const int8_t*>(a.v) + src[f]);
                kscale[f] = a.k_scale[row];
                vscale[f] = a.v_scale[row];
            } else {
                kr[f] = load8<DT>(a.k, src[f]);
                vr[f] = load8<DT>(a.v, src[f]);
            }
        }
#pragma unroll
        for (int f = 0; f < PG_FLIGHT; ++f) {
            if (src[f] < 0) continue;
            float x[8];
            if (Q8) widen8_codes(kc[f], kscale[f], x); else widen8<DT>(kr[f], x);
            store8<DT>(a.k_out, dst[f], x);
            if (Q8) widen8_codes(vc[f], vscale[f], x); else widen8<DT>(vr[f], x);
            store8<DT>(a.v_out, dst[f], x);
        }
    }
}

// ---------------------------------------------------------------- host
static bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
static bool dtype_ok(int dt) { return dt == QV_F32 || dt == QV_BF16 || dt == QV_F16; }

// The checks every entry point makes of a cache.
int paged_cache_check(const qv_paged_cache* c) {
    if (!c || !c->k || !c->v || !al16(c->k) || !al16(c->v)) return QV_EINVAL;
    if (c->pages <= 0 || c->kv_heads <= 0 || c->head_dim < 8 || c->head_dim > 256 || c->head_dim % 8) return QV_EINVAL;
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return QV_EINVAL;
    if (!dtype_ok(c->dtype) || (c->bits != 0 && c->bits != 8)) return QV_EINVAL;
    if (c->bits == 8 && (!c->k_scale || !c->v_scale || !al16(c->k_scale) || !al16(c->v_scale))) return QV_EINVAL;
    return QV_OK;
}

int paged_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

static int heads_check(const HeadArgs& a, int64_t tokens, int dt) {
    if (tokens < 0 || tokens > 0x7fffffff || a.Hq <= 0 || a.H <= 0 || !dtype_ok(dt)) return QV_EINVAL;
    if (a.D < 8 || a.D > 256 || a.D % 8) return QV_EINVAL;
    const int64_t per16 = 16 / (int64_t)elt_size(dt);
    if (!a.q || !a.k || !a.q_out || !al16(a.q) || !al16(a.k) || !al16(a.q_out)) return QV_EINVAL;
    if (a.qs < (int64_t)a.Hq * a.D || a.ks < (int64_t)a.H * a.D || a.qs % per16 || a.ks % per16) return QV_EINVAL;
    if ((a.qw && !al16(a.qw)) || (a.kw && !al16(a.kw))) return QV_EINVAL;
    if (a.table && (!a.pos || !al16(a.table) || a.max_pos <= 0 || a.rot < 8 || a.rot > a.D || a.rot % 8)) return QV_EINVAL;
    return QV_OK;
}

// Whether outputs share memory with one another or with what the call reads.  A row is read by the block that writes it,
// before it does: the queries (and, without pages, the keys) may be written in place where they are contiguous.
static bool heads_overlap(const HeadArgs& a, int64_t tokens, int dt, const qv_paged_cache* c) {
    const size_t e = elt_size(dt), n = (size_t)tokens, w = (size_t)a.D * e;
    auto rows = [&](const void* p, int64_t stride, int heads) { return span(p, ((n - 1) * (size_t)stride + (size_t)heads * a.D) * e); };
    const Span q = rows(a.q, a.qs, a.Hq), k = rows(a.k, a.ks, a.H), v = rows(a.v, a.vs, a.H);
    const Span qw = span(a.qw, w), kw = span(a.kw, w), table = span(a.table, (size_t)a.max_pos * a.rot * 4);
    const Span pos = span(a.table ? a.pos : nullptr, n * 4), slots = span(a.slots, n * 8), err = span(a.err, 4);
    auto in_place = [&](Span in, Span out) { return in.at == out.at && in.bytes == out.bytes; };
    auto taken = [&](Span o) { return meets(o, {v, qw, kw, table, pos, slots, err}); };
    const Span qo = span(a.q_out, n * a.Hq * w);
    if (taken(qo) || meets(qo, {k}) || (meets(qo, {q}) && !in_place(q, qo))) return true;
    if (!c) {
        const Span ko = span(a.k_out, n * a.H * w);
        return taken(ko) || meets(ko, {q, qo}) || (meets(ko, {k}) && !in_place(k, ko));
    }
    const size_t pb = pool_bytes(c), sb = pool_scale_bytes(c);
    const Span pool[4] = {span(c->k, pb), span(c->v, pb), span(c->k_scale, sb), span(c->v_scale, sb)};
    for (int i = 0; i < 4; ++i) {
        if (taken(pool[i]) || meets(pool[i], {q, k, qo})) return true;
        for (int j = 0; j < i; ++j)
            if (meets(pool[i], {pool[j]})) return true;
    }
    return false;
}

template <int DT, int MODE> static int heads_launch(const HeadArgs& a, int64_t tokens, cudaStream_t s) {
    // Few tokens: large blocks, one for each kind of head (a decode step's latency).  Many: one small block per
    // token, so that a thread has rows enough to pay for the token's table row and slot; 16383 tokens of 64
    // normed heads take 98, 105 and 118 us with 32, 64 and 128 threads, 400 tokens of 48 heads 6.8, 5.2 and 4.7.
    const bool few = tokens < 2 * 148;
    const dim3 g((unsigned)tokens, !few ? 1 : MODE == PH_ROWS_ONLY ? 2 : 3);
    const int n = few ? PH_MOST : tokens < 8 * 148 ? 128 : tokens < 16 * 148 ? 64 : 32;
    if (a.D <= 64) heads_kernel<DT, 8, MODE><<<g, n, 0, s>>>(a);
    else if (a.D <= 128) heads_kernel<DT, 16, MODE><<<g, n, 0, s>>>(a);
    else heads_kernel<DT, 32, MODE><<<g, n, 0, s>>>(a);
    return check_launch();
}
template <int MODE> static int heads_dispatch(const HeadArgs& a, int64_t tokens, int dt, cudaStream_t s) {
    if (dt == QV_F32) return heads_launch<QV_F32, MODE>(a, tokens, s);
    if (dt == QV_BF16) return heads_launch<QV_BF16, MODE>(a, tokens, s);
    return heads_launch<QV_F16, MODE>(a, tokens, s);
}

}  // namespace qv

using namespace qv;

extern "C" int qv_qk_norm_rope(int32_t tokens, int32_t q_heads, int32_t kv_heads, int32_t head_dim, int32_t dtype,
                               const void* q, int64_t q_stride, const void* k, int64_t k_stride, const void* q_weight,
                               const void* k_weight, float eps, const float* table, int32_t max_pos, int32_t rot_dim,
                               int32_t interleaved, const int32_t* positions, void* q_out, void* k_out,
                               qv_stream_t stream) {
    HeadArgs a = {};
    a.q = q; a.k = k; a.qs = q_stride; a.ks = k_stride; a.qw = q_weight; a.kw = k_weight; a.eps = eps;
    a.table = table; a.pos = positions; a.max_pos = max_pos; a.rot = rot_dim; a.interleaved = interleaved != 0;
    a.Hq = q_heads; a.H = kv_heads; a.D = head_dim; a.q_out = q_out; a.k_out = k_out;
    if (tokens == 0) return QV_OK;
    const int rc = heads_check(a, tokens, dtype);
    if (rc != QV_OK) return rc;
    if (!k_out || !al16(k_out) || heads_overlap(a, tokens, dtype, nullptr)) return QV_EINVAL;
    return heads_dispatch<PH_ROWS_ONLY>(a, tokens, dtype, (cudaStream_t)stream);
}

extern "C" int qv_paged_append(const qv_paged_cache* c, int32_t tokens, int32_t q_heads, const void* q,
                               int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                               const void* q_weight, const void* k_weight, float eps, const float* table,
                               int32_t max_pos, int32_t rot_dim, int32_t interleaved, const int32_t* positions,
                               const int64_t* slots, void* q_out, qv_stream_t stream) {
    int rc = paged_cache_check(c);
    if (rc != QV_OK) return rc;
    HeadArgs a = {};
    a.q = q; a.k = k; a.v = v; a.qs = q_stride; a.ks = k_stride; a.vs = v_stride;
    a.qw = q_weight; a.kw = k_weight; a.eps = eps;
    a.table = table; a.pos = positions; a.max_pos = max_pos; a.rot = rot_dim; a.interleaved = interleaved != 0;
    a.Hq = q_heads; a.H = c->kv_heads; a.D = c->head_dim; a.q_out = q_out;
    a.kp = c->k; a.vp = c->v; a.k_scale = c->k_scale; a.v_scale = c->v_scale; a.err = c->err;
    a.slots = slots; a.page_shift = paged_shift(c->page_size);
    a.n_slots = (int64_t)c->pages * c->page_size;
    if (tokens == 0) return QV_OK;
    rc = heads_check(a, tokens, c->dtype);
    if (rc != QV_OK) return rc;
    const int64_t per16 = 16 / (int64_t)elt_size(c->dtype);
    if (!v || !al16(v) || !slots || v_stride < (int64_t)a.H * a.D || v_stride % per16) return QV_EINVAL;
    if (heads_overlap(a, tokens, c->dtype, c)) return QV_EINVAL;
    return c->bits == 8 ? heads_dispatch<PH_PAGES8>(a, tokens, c->dtype, (cudaStream_t)stream)
                        : heads_dispatch<PH_PAGES>(a, tokens, c->dtype, (cudaStream_t)stream);
}

extern "C" int qv_paged_gather(const qv_paged_cache* c, int32_t batch, const int32_t* block_table, int32_t max_pages,
                               const int32_t* kv_lens, const int32_t* cu_kv, int32_t total, void* k_out, void* v_out,
                               qv_stream_t stream) {
    const int rc = paged_cache_check(c);
    if (rc != QV_OK) return rc;
    if (batch < 0 || total < 0) return QV_EINVAL;
    if (batch == 0 || total == 0) return QV_OK;
    if (!block_table || max_pages <= 0 || !kv_lens || !cu_kv || !k_out || !v_out) return QV_EINVAL;
    if (!al16(k_out) || !al16(v_out)) return QV_EINVAL;
    // a block writes rows that others still read: nothing in place
    const size_t out_bytes = (size_t)total * c->kv_heads * c->head_dim * elt_size(c->dtype), sb = pool_scale_bytes(c);
    const Span ko = span(k_out, out_bytes), vo = span(v_out, out_bytes);
    for (const Span& o : {ko, vo})
        if (meets(o, {span(c->k, pool_bytes(c)), span(c->v, pool_bytes(c)), span(c->k_scale, sb), span(c->v_scale, sb),
                      span(block_table, (size_t)batch * max_pages * 4), span(kv_lens, (size_t)batch * 4),
                      span(cu_kv, ((size_t)batch + 1) * 4), span(c->err, 4)}))
            return QV_EINVAL;
    if (meets(ko, {vo})) return QV_EINVAL;
    GatherArgs a = {c->k, c->v, c->k_scale, c->v_scale, c->err, block_table, kv_lens, cu_kv, k_out, v_out,
                    c->pages, c->kv_heads, c->head_dim, paged_shift(c->page_size), max_pages, batch, total};
    const int g = (int)(((int64_t)total + PG_TOKENS - 1) / PG_TOKENS);
    cudaStream_t s = (cudaStream_t)stream;
    const bool q8 = c->bits == 8;
    if (c->dtype == QV_F32) {
        if (q8) gather_kernel<QV_F32, true><<<g, PG_THREADS, 0, s>>>(a);
        else gather_kernel<QV_F32, false><<<g, PG_THREADS, 0, s>>>(a);
    } else if (c->dtype == QV_BF16) {
        if (q8) gather_kernel<QV_BF16, true><<<g, PG_THREADS, 0, s>>>(a);
        else gather_kernel<QV_BF16, false><<<g, PG_THREADS, 0, s>>>(a);
    } else {
        if (q8) gather_kernel<QV_F16, true><<<g, PG_THREADS, 0, s>>>(a);
        else gather_kernel<QV_F16, false><<<g, PG_THREADS, 0, s>>>(a);
    }
    return check_launch();
}
