// Per-head norm of Q and K and the position rotation, in one pass.
//
// For a head's row x of D channels, weight w and the token's angles t:
//   n_c = x_c * w_c / sqrt(mean_c(x_c^2) + eps)
//   (n_a, n_b) -> (n_a cos t_i - n_b sin t_i, n_a sin t_i + n_b cos t_i)
// for the pairs i < rotary / 2: (a, b) = (2i, 2i + 1) or (i, i + rotary / 2).
// Channels behind `rotary` and tokens behind the tables' last row are only
// normed.  All arithmetic is FP32 and rounds once, at the store.
//
// Bound: HBM.  Q and K are read and written once and the tables once (their
// rows are shared by all heads of a token).  Measured, 1 B200: 32768 tokens x 40
// heads x 128, BF16, 237-246 us, 85-89 % of a plain copy's rate; 2 x 24 heads x 4399
// tokens x 96, FP16, 40 us, bound by issue slots (12 of 16 lanes have channels).
//
// Split.  A row of D channels is held by LPR lanes with one 16-byte vector
// each (16 lanes for 128 16-bit channels), so the sum of squares takes
// log2(LPR) shuffles and a pair lies in one lane (adjacent pairs) or one
// shuffle away (half-split pairs).  A warp takes four such vectors of one token
// at a time, all loads issued before the first use, and reads the token's
// angles once for all of them; the eight warps of a CTA take eight consecutive tokens, so that a
// token-major input is read in runs of 4 * 32 * 16 bytes and a head-major
// output written in runs of eight rows.
#include "vcb_internal.h"

namespace vcb {
namespace {

constexpr int kWarps = 8;            // tokens per CTA
constexpr int kLoads = 4;            // row vectors in flight per lane

struct RopeSide {                    // Q or K
    const void* x;
    void* y;
    const void* w;                   // [d] or null
    int w_dtype, w_vec;              // w_vec: 16-byte aligned
    int heads;
    int chunks;                      // warps that share a token's heads
    int64_t xs_b, xs_h, xs_s, ys_b, ys_h, ys_s;
};

struct RopeParams {
    RopeSide side[2];
    const float* cos;
    const float* sin;
    int64_t tokens, rows;            // rows: tokens with a row in the tables
    int64_t ts_b, ts_s;              // table strides (batch 0 when shared)
    int d, half;                     // rotary / 2
    int interleaved, norm;
    int table_vec;                   // the tables allow 16-byte (adjacent fp32: 8-byte) loads
    float eps;
};

__device__ __forceinline__ float load_as_float(const void* p, int64_t i, int dtype) {
    if (dtype == VCB_F32) return __ldg(static_cast<const float*>(p) + i);
    if (dtype == VCB_F16) return __half2float(__ldg(static_cast<const __half*>(p) + i));
    return __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(p) + i));
}

// Not __ldg: the output may be the input (an in-place call).
__device__ __forceinline__ uint4 load16(const void* p) { return *static_cast<const uint4*>(p); }

template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};
template <> struct Vec<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
        const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 v = __half22float2(h[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        uint4 u;
        __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        return u;
    }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& u, float* f) {
        const uint32_t h[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(h[i] << 16);
            f[2 * i + 1] = __uint_as_float(h[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        uint4 u;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        return u;
    }
};

// N consecutive fp32 entries p[i ..]; entries at or behind `limit` read as 0
template <int N>
__device__ __forceinline__ void load_table(const float* p, int i, int limit, bool vec, float* o) {
    if (vec && i + N <= limit) {
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int e = 0; e < N; e += 4) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(p + i + e));
                o[e] = f.x; o[e + 1] = f.y; o[e + 2] = f.z; o[e + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const float2 f = __ldg(reinterpret_cast<const float2*>(p + i + e));
                o[e] = f.x; o[e + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = i + e < limit ? __ldg(p + i + e) : 0.0f;
    }
}

// N consecutive weights from w[i]; ones without weights
template <int N>
__device__ __forceinline__ void load_weights(const RopeSide& s, int i, float* o) {
    if (!s.w) {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = 1.0f;
    } else if (s.w_dtype == VCB_F32 && s.w_vec) {
        load_table<N>(static_cast<const float*>(s.w), i, i + N, true, o);
    } else if (s.w_vec) {
        uint32_t u[N / 2];
        const uint16_t* w = static_cast<const uint16_t*>(s.w) + i;
        if constexpr (N == 8) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(w));
            u[0] = v.x; u[1] = v.y; u[2] = v.z; u[3] = v.w;
        } else {
            const uint2 v = __ldg(reinterpret_cast<const uint2*>(w));
            u[0] = v.x; u[1] = v.y;
        }
#pragma unroll
        for (int e = 0; e < N / 2; ++e) {
            const float2 f = s.w_dtype == VCB_F16 ? __half22float2(*reinterpret_cast<const __half2*>(&u[e]))
                                                  : make_float2(__uint_as_float(u[e] << 16),
                                                                __uint_as_float(u[e] & 0xffff0000u));
            o[2 * e] = f.x; o[2 * e + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = load_as_float(s.w, i + e, s.w_dtype);
    }
}

// 16-byte vectors, LPR lanes per row.  Needs d, the strides and the base
// pointers in whole vectors and, for half-split pairs, rotary / 2 too.
// Weight and angle are multiplied once per token: with A = w cos, B = -+ w' sin
// (w' the partner's weight) a channel is r (x A + x' B), r the row's 1 / rms.
template <typename T, int LPR, bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kWarps, 4) rope_kernel(const __grid_constant__ RopeParams p) {
    pdl_wait();
    pdl_open();
    constexpr int N = Vec<T>::N, P = N / 2;
    constexpr int kRows = 32 / LPR;                  // rows per vector load of the warp
    constexpr int A = INTERLEAVED ? P : N;           // angles per lane
    const int lane = threadIdx.x & 31, li = lane % LPR, sub = lane / LPR;
    const int chunks = p.side[0].chunks + p.side[1].chunks;
    const int block = blockIdx.x / chunks;
    int chunk = blockIdx.x - block * chunks;
    const int64_t s = (int64_t)block * kWarps + (threadIdx.x >> 5);
    if (s >= p.tokens) return;
    const int64_t b = blockIdx.y;
    const int which = chunk >= p.side[0].chunks;
    const RopeSide& sd = p.side[which];
    if (which) chunk -= p.side[0].chunks;
    const int c = li * N;
    const bool has = c < p.d;
    const T* x = static_cast<const T*>(sd.x) + b * sd.xs_b + s * sd.xs_s + c;
    T* y = static_cast<T*>(sd.y) + b * sd.ys_b + s * sd.ys_s + c;
    const int h0 = chunk * (kRows * kLoads) + sub;

    uint4 raw[kLoads];
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        const int h = h0 + u * kRows;
        raw[u] = has && h < sd.heads ? load16(x + h * sd.xs_h) : make_uint4(0, 0, 0, 0);
    }
    // the token's angles and the weights, once for all rows
    const int half = s < p.rows ? p.half : 0;
    const bool low = INTERLEAVED || c < half;        // half-split: this lane's channels are the first of their pairs
    const int a0 = INTERLEAVED ? c / 2 : (low ? c : c - half);
    const bool rot = has && (INTERLEAVED ? a0 < half : c < 2 * half);
    const bool all = rot && a0 + A <= half;          // every channel of this lane turns
    const int shift = half / (INTERLEAVED ? 1 : N);  // half-split: lanes between partners
    const int peer = INTERLEAVED || !rot ? li : (low ? li + shift : li - shift);
    // A and B of channel pairs 2e, 2e + 1; where nothing turns A = w and B = 0, and
    // the partner is taken as 0 too (0 times a NaN or infinity would not be)
    float2 ca[P], cb[P];
    {
        float w[N], cs[A], sn[A], wp[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = 1.0f;
        if (has) load_weights<N>(sd, c, w);
#pragma unroll
        for (int e = 0; e < P; ++e) {
            ca[e] = make_float2(w[2 * e], w[2 * e + 1]);
            cb[e] = make_float2(0.0f, 0.0f);
        }
        if (rot) {
            const int64_t t = b * p.ts_b + s * p.ts_s;
            load_table<A>(p.cos + t, a0, half, p.table_vec, cs);
            load_table<A>(p.sin + t, a0, half, p.table_vec, sn);
            if (!INTERLEAVED) load_weights<N>(sd, peer * N, wp);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                if (INTERLEAVED) {
                    if (a0 + e >= half) break;
                    ca[e] = make_float2(__fmul_rn(w[2 * e], cs[e]), __fmul_rn(w[2 * e + 1], cs[e]));
                    cb[e] = make_float2(-__fmul_rn(w[2 * e + 1], sn[e]), __fmul_rn(w[2 * e], sn[e]));
                } else {
                    const float sg = low ? -1.0f : 1.0f;
                    ca[e] = make_float2(__fmul_rn(w[2 * e], cs[2 * e % A]), __fmul_rn(w[2 * e + 1], cs[(2 * e + 1) % A]));
                    cb[e] = make_float2(__fmul_rn(sg * wp[2 * e], sn[2 * e % A]),
                                        __fmul_rn(sg * wp[2 * e + 1], sn[(2 * e + 1) % A]));
                }
            }
        }
    }
    const float inv_d = 1.0f / (float)p.d;
    const bool warp_all = __all_sync(0xffffffffu, all);      // the common case: no choice per channel
    T* to = y + h0 * sd.ys_h;
    const int64_t step = kRows * sd.ys_h;
#pragma unroll
    for (int u = 0; u < kLoads; ++u, to += step) {
        float f[N];
        Vec<T>::unpack(raw[u], f);
        float r = 1.0f;
        if (p.norm) {
            float2 s2 = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const float2 v = make_float2(f[2 * e], f[2 * e + 1]);
                s2 = ffma2(v, v, s2);
            }
            float ss = __fadd_rn(s2.x, s2.y);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            r = rsqrtf(__fmaf_rn(ss, inv_d, p.eps));
        }
        const float2 rr = make_float2(r, r);
        float g[N];                                  // the partners' channels
        if (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < P; ++e) { g[2 * e] = f[2 * e + 1]; g[2 * e + 1] = f[2 * e]; }
            if (!warp_all) {
#pragma unroll
                for (int e = 0; e < P; ++e)
                    if (a0 + e >= half) g[2 * e] = g[2 * e + 1] = 0.0f;
            }
        } else {
            const int from = peer + sub * LPR;
            uint4 o = make_uint4(__shfl_sync(0xffffffffu, raw[u].x, from), __shfl_sync(0xffffffffu, raw[u].y, from),
                                 __shfl_sync(0xffffffffu, raw[u].z, from), __shfl_sync(0xffffffffu, raw[u].w, from));
            if (!rot) o = make_uint4(0, 0, 0, 0);
            Vec<T>::unpack(o, g);
        }
#pragma unroll
        for (int e = 0; e < P; ++e) {
            float2 o = fmul2(make_float2(g[2 * e], g[2 * e + 1]), cb[e]);
            o = fmul2(ffma2(make_float2(f[2 * e], f[2 * e + 1]), ca[e], o), rr);
            f[2 * e] = o.x; f[2 * e + 1] = o.y;
        }
        if (has && h0 + u * kRows < sd.heads) *reinterpret_cast<uint4*>(to) = Vec<T>::pack(f);
    }
}

template <typename T> __device__ __forceinline__ T from_float(float f);
template <> __device__ __forceinline__ float from_float<float>(float f) { return f; }
template <> __device__ __forceinline__ __half from_float<__half>(float f) { return __float2half_rn(f); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Any width, stride and alignment: the same lanes, channels and order of
// arithmetic as rope_kernel (an output does not depend on the layout), element
// by element; a pair's other channel is read again (from L1).
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) rope_any_kernel(const __grid_constant__ RopeParams p, int lpr) {
    pdl_wait();
    pdl_open();
    constexpr int N = Vec<T>::N;
    const int lane = threadIdx.x & 31, li = lane & (lpr - 1), sub = lane / lpr;
    const int chunks = p.side[0].chunks + p.side[1].chunks;
    const int block = blockIdx.x / chunks;
    int chunk = blockIdx.x - block * chunks;
    const int64_t s = (int64_t)block * kWarps + (threadIdx.x >> 5);
    if (s >= p.tokens) return;
    const int64_t b = blockIdx.y;
    const int which = chunk >= p.side[0].chunks;
    const RopeSide& sd = p.side[which];
    if (which) chunk -= p.side[0].chunks;
    const int h = chunk * (32 / lpr) + sub;
    const bool row = h < sd.heads;
    const T* x = static_cast<const T*>(sd.x) + b * sd.xs_b + h * sd.xs_h + s * sd.xs_s;
    T* y = static_cast<T*>(sd.y) + b * sd.ys_b + h * sd.ys_h + s * sd.ys_s;
    const int half = s < p.rows ? p.half : 0;
    float f[N], g[N];
    float s2[2] = {0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int c = li * N + e;
        const bool in = row && c < p.d;
        f[e] = in ? as_float(x[c]) : 0.0f;
        g[e] = in && c < 2 * half ? as_float(x[p.interleaved ? c ^ 1 : (c < half ? c + half : c - half)]) : 0.0f;
        s2[e & 1] = __fmaf_rn(f[e], f[e], s2[e & 1]);
    }
    float r = 1.0f;
    if (p.norm) {
        float ss = __fadd_rn(s2[0], s2[1]);
        for (int o = lpr / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        r = rsqrtf(__fmaf_rn(ss, 1.0f / (float)p.d, p.eps));
    }
    const int64_t t = b * p.ts_b + s * p.ts_s;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int c = li * N + e;
        if (!row || c >= p.d) continue;
        const float w = sd.w ? load_as_float(sd.w, c, sd.w_dtype) : 1.0f;
        if (c < 2 * half) {
            const int peer = p.interleaved ? c ^ 1 : (c < half ? c + half : c - half);
            const bool first = p.interleaved ? !(c & 1) : c < half;
            const int a = p.interleaved ? c >> 1 : (c < half ? c : c - half);
            const float wp = sd.w ? load_as_float(sd.w, peer, sd.w_dtype) : 1.0f;
            const float ws = __fmul_rn(wp, __ldg(p.sin + t + a));
            f[e] = __fmaf_rn(f[e], __fmul_rn(w, __ldg(p.cos + t + a)), __fmul_rn(g[e], first ? -ws : ws));
        } else {
            f[e] = __fmul_rn(f[e], w);
        }
        f[e] = __fmul_rn(f[e], r);
    }
    __syncwarp();                       // every lane has read its row: it may be the output
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int c = li * N + e;
        if (row && c < p.d) y[c] = from_float<T>(f[e]);
    }
}

template <typename T, int LPR>
cudaError_t launch_vec(RopeParams& p, int64_t batch, cudaStream_t st) {
    constexpr int per = (32 / LPR) * kLoads;
    for (RopeSide& s : p.side) s.chunks = (s.heads + per - 1) / per;
    const int64_t blocks = (p.tokens + kWarps - 1) / kWarps * (p.side[0].chunks + p.side[1].chunks);
    const dim3 grid((unsigned)blocks, (unsigned)batch);
    if (p.interleaved) return launch_pdl(rope_kernel<T, LPR, true>, grid, dim3(32 * kWarps), 0, st, p);
    return launch_pdl(rope_kernel<T, LPR, false>, grid, dim3(32 * kWarps), 0, st, p);
}

template <typename T>
int launch(RopeParams& p, int64_t batch, bool vec, cudaStream_t st) {
    constexpr int N = Vec<T>::N;
    const int lanes = (p.d + N - 1) / N;
    if (!vec) {
        int lpr = 4;
        while (lpr < lanes) lpr *= 2;
        for (RopeSide& s : p.side) s.chunks = (s.heads + 32 / lpr - 1) / (32 / lpr);
        const int64_t blocks = (p.tokens + kWarps - 1) / kWarps * (p.side[0].chunks + p.side[1].chunks);
        VCB_CUDA(launch_pdl(rope_any_kernel<T>, dim3((unsigned)blocks, (unsigned)batch), dim3(32 * kWarps), 0, st, p, lpr));
        return VCB_OK;
    }
    if (lanes <= 4) VCB_CUDA((launch_vec<T, 4>(p, batch, st)));
    else if (lanes <= 8) VCB_CUDA((launch_vec<T, 8>(p, batch, st)));
    else if (lanes <= 16 || N > 4) VCB_CUDA((launch_vec<T, 16>(p, batch, st)));
    else if constexpr (N == 4) VCB_CUDA((launch_vec<T, 32>(p, batch, st)));
    return VCB_OK;
}

bool multiple(int64_t v, int n) { return v % n == 0; }
bool aligned(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace

int rope_run(const vcb_qk_norm_rope_args* a, cudaStream_t st) {
    RopeParams p{};
    const int n = a->dtype == VCB_F32 ? 4 : 8;
    bool vec = multiple(a->d, n) && (a->interleaved || multiple(a->rotary / 2, n));
    for (int i = 0; i < 2; ++i) {
        RopeSide& s = p.side[i];
        s.x = i ? a->k : a->q;
        s.y = i ? a->k_out : a->q_out;
        s.w = i ? a->k_weight : a->q_weight;
        s.w_dtype = a->weight_dtype;
        s.w_vec = aligned(s.w, 16);
        s.heads = (int)(i ? a->k_heads : a->q_heads);
        const int64_t* xs = i ? a->k_stride : a->q_stride;
        const int64_t* ys = i ? a->k_out_stride : a->q_out_stride;
        s.xs_b = xs[0]; s.xs_h = xs[1]; s.xs_s = xs[2];
        s.ys_b = ys[0]; s.ys_h = ys[1]; s.ys_s = ys[2];
        vec = vec && aligned(s.x, 16) && aligned(s.y, 16);
        for (int j = 0; j < 3; ++j) vec = vec && multiple(xs[j], n) && multiple(ys[j], n);
    }
    p.cos = a->cos; p.sin = a->sin;
    p.tokens = a->tokens; p.rows = a->rotary ? a->rows : 0;
    p.ts_b = a->table_stride_b; p.ts_s = a->table_stride_s;
    p.d = a->d; p.half = a->rotary / 2;
    p.interleaved = a->interleaved; p.norm = a->norm; p.eps = a->eps;
    p.table_vec = aligned(a->cos, 16) && aligned(a->sin, 16) && multiple(a->table_stride_b, 4) &&
                  multiple(a->table_stride_s, 4);
    switch (a->dtype) {
        case VCB_F32: return launch<float>(p, a->batch, vec, st);
        case VCB_F16: return launch<__half>(p, a->batch, vec, st);
        default: return launch<__nv_bfloat16>(p, a->batch, vec, st);
    }
}

}  // namespace vcb
