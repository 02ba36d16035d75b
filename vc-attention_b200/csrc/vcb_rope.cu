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
// rows are shared by all heads of a token).
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
    int w_dtype;
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
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) { const float2 v = __bfloat1622float2(h[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        uint4 u;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        return u;
    }
};

// n consecutive table entries starting at p + i
template <int N>
__device__ __forceinline__ void load_table(const float* p, int i, int limit, bool vec, float* o) {
    if (vec && i + N <= limit) {
        if (N % 4 == 0) {
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

// 16-byte vectors, LPR lanes per row.  Needs d, the strides and the base
// pointers in whole vectors and, for half-split pairs, rotary / 2 too.
template <typename T, int LPR, bool INTERLEAVED>
__global__ void __launch_bounds__(32 * kWarps) rope_kernel(const __grid_constant__ RopeParams p) {
    pdl_wait();
    pdl_open();
    constexpr int N = Vec<T>::N;
    constexpr int kRows = 32 / LPR;                  // rows per vector load of the warp
    constexpr int A = INTERLEAVED ? N / 2 : N;       // angles per lane
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
    // the token's angles, once for all rows: a0 is this lane's first
    const bool turned = s < p.rows;
    const int half = turned ? p.half : 0;
    int a0 = INTERLEAVED ? c / 2 : (c >= half ? c - half : c);
    const bool rot = INTERLEAVED ? a0 < half : c < 2 * half;
    float cs[A], sn[A];
    if (rot && has) {
        const int64_t t = b * p.ts_b + s * p.ts_s;
        load_table<A>(p.cos + t, a0, half, p.table_vec, cs);
        load_table<A>(p.sin + t, a0, half, p.table_vec, sn);
    }
    float w[N];
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = sd.w && has ? load_as_float(sd.w, c + e, sd.w_dtype) : 1.0f;
    const float inv_d = 1.0f / (float)p.d;
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
        float f[N];
        Vec<T>::unpack(raw[u], f);
        if (p.norm) {
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < N; ++e) ss = __fmaf_rn(f[e], f[e], ss);
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float r = __frsqrt_rn(__fmaf_rn(ss, inv_d, p.eps));
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = __fmul_rn(__fmul_rn(f[e], r), w[e]);
        } else {
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = __fmul_rn(f[e], w[e]);
        }
        if (INTERLEAVED) {
            if (rot) {
#pragma unroll
                for (int e = 0; e < A; ++e)
                    if (a0 + e < half) {
                        const float a = f[2 * e], q = f[2 * e + 1];
                        f[2 * e] = __fmaf_rn(a, cs[e], -__fmul_rn(q, sn[e]));
                        f[2 * e + 1] = __fmaf_rn(a, sn[e], __fmul_rn(q, cs[e]));
                    }
            }
        } else if (half > 0) {                       // the same for every lane of the warp
            const int shift = half / N;
            const int peer = (rot ? (c < half ? li + shift : li - shift) : li) + sub * LPR;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float o = __shfl_sync(0xffffffffu, f[e], peer);
                if (rot) f[e] = __fmaf_rn(f[e], cs[e], c < half ? -__fmul_rn(o, sn[e]) : __fmul_rn(o, sn[e]));
            }
        }
        const int h = h0 + u * kRows;
        if (has && h < sd.heads) *reinterpret_cast<uint4*>(y + h * sd.ys_h) = Vec<T>::pack(f);
    }
}

template <typename T> __device__ __forceinline__ T from_float(float f);
template <> __device__ __forceinline__ float from_float<float>(float f) { return f; }
template <> __device__ __forceinline__ __half from_float<__half>(float f) { return __float2half_rn(f); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }
__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Any width, stride and alignment: one warp per row, lane l holds channels
// l, l + 32, ...; a pair's other channel is read again (from L1).
template <typename T>
__global__ void __launch_bounds__(32 * kWarps) rope_any_kernel(const __grid_constant__ RopeParams p) {
    pdl_wait();
    pdl_open();
    const int lane = threadIdx.x & 31;
    const int heads = p.side[0].heads + p.side[1].heads;
    const int block = blockIdx.x / heads;
    int h = blockIdx.x - block * heads;
    const int64_t s = (int64_t)block * kWarps + (threadIdx.x >> 5);
    if (s >= p.tokens) return;
    const int64_t b = blockIdx.y;
    const int which = h >= p.side[0].heads;
    const RopeSide& sd = p.side[which];
    if (which) h -= p.side[0].heads;
    const T* x = static_cast<const T*>(sd.x) + b * sd.xs_b + h * sd.xs_h + s * sd.xs_s;
    T* y = static_cast<T*>(sd.y) + b * sd.ys_b + h * sd.ys_h + s * sd.ys_s;
    const int half = s < p.rows ? p.half : 0;
    float f[4], o[4];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        f[i] = c < p.d ? as_float(x[c]) : 0.0f;
        ss = __fmaf_rn(f[i], f[i], ss);
        o[i] = 0.0f;
        if (c < 2 * half) o[i] = as_float(x[p.interleaved ? c ^ 1 : (c < half ? c + half : c - half)]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
    const float r = p.norm ? __frsqrt_rn(__fmaf_rn(ss, 1.0f / (float)p.d, p.eps)) : 1.0f;
    const int64_t t = b * p.ts_b + s * p.ts_s;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        if (c >= p.d) continue;
        f[i] = __fmul_rn(f[i], r);
        if (sd.w) f[i] = __fmul_rn(f[i], load_as_float(sd.w, c, sd.w_dtype));
        if (c < 2 * half) {
            const int peer = p.interleaved ? c ^ 1 : (c < half ? c + half : c - half);
            const bool first = p.interleaved ? !(c & 1) : c < half;
            const int a = p.interleaved ? c >> 1 : (c < half ? c : c - half);
            float q = __fmul_rn(o[i], r);
            if (sd.w) q = __fmul_rn(q, load_as_float(sd.w, peer, sd.w_dtype));
            const float qs = __fmul_rn(q, __ldg(p.sin + t + a));
            f[i] = __fmaf_rn(f[i], __ldg(p.cos + t + a), first ? -qs : qs);
        }
    }
    __syncwarp();                       // every lane has read the row: it may be the output
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = lane + 32 * i;
        if (c < p.d) y[c] = from_float<T>(f[i]);
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
    if (!vec) {
        const int64_t blocks = (p.tokens + kWarps - 1) / kWarps * (p.side[0].heads + p.side[1].heads);
        VCB_CUDA(launch_pdl(rope_any_kernel<T>, dim3((unsigned)blocks, (unsigned)batch), dim3(32 * kWarps), 0, st, p));
        return VCB_OK;
    }
    const int lanes = (p.d + N - 1) / N;
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
