// 16-bit attention over a sliding window with first tokens that stay visible.
// Query i stands at position p = i + offset and sees key j of the first `len`
// keys when
//   (j < sinks or p - left <= j <= p + right) and (not causal or j <= p);
// out = softmax over the seen keys of (scale q . k), times v; 0 for a row that
// sees none.  The seen keys are two runs, [0, sink) and [lo, hi).
#include "vcb_internal.h"

namespace vcb {
namespace {

struct WinParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* kv_lens;
    int64_t qs[3], ks[3], vs[3], os[3];      // batch, head, token
    int64_t sq, sk, heads;
    int64_t left, right, sinks, q_offset;
    int causal, has_offset, d;
    float scale;
};

// The keys that the query at position p sees: [0, sink) and [lo, hi), lo >= sink.
struct Seen {
    int sink, lo, hi;
};
__device__ __forceinline__ Seen seen_at(const WinParams& p, int64_t pos, int64_t len) {
    auto clamp = [&](int64_t x) { return x < 0 ? (int64_t)0 : x > len ? len : x; };
    int64_t lo = p.left < 0 ? 0 : clamp(pos - p.left);
    int64_t hi = p.right < 0 ? len : clamp(pos + p.right + 1);
    int64_t sink = clamp(p.sinks);
    if (p.causal) {
        const int64_t end = clamp(pos + 1);
        hi = hi < end ? hi : end;
        sink = sink < end ? sink : end;
    }
    lo = lo > sink ? lo : sink;
    return {(int)sink, (int)lo, (int)(hi > lo ? hi : lo)};
}

__device__ __forceinline__ int64_t keys_of(const WinParams& p, int64_t b) {
    if (!p.kv_lens) return p.sk;
    const int64_t n = p.kv_lens[b];
    return n < 0 ? 0 : n > p.sk ? p.sk : n;
}

__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float f);
template <> __device__ __forceinline__ __half from_f<__half>(float f) { return __float2half_rn(f); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float f) { return __float2bfloat16_rn(f); }

// One output row by one warp, reading only the keys that the row sees: lane l
// takes every 32nd key's logit, then channels l, l + 32, ... of the sum.
// `qrow` is 128 floats of shared memory of this warp.
template <typename T>
__device__ void window_row(const WinParams& p, int64_t b, int64_t h, int64_t i, float* qrow, int lane) {
    const int64_t len = keys_of(p, b);
    const Seen s = seen_at(p, i + (p.has_offset ? p.q_offset : len - p.sq), len);
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + h * p.ks[1];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + h * p.vs[1];
    __syncwarp();
    for (int c = lane; c < 128; c += 32) qrow[c] = c < p.d ? to_f(q[c]) : 0.0f;
    __syncwarp();
    float m = -INFINITY, den = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int part = 0; part < 2; ++part) {
        const int first = part ? s.lo : 0, last = part ? s.hi : s.sink;
        for (int base = first; base < last; base += 32) {
            const int n = min(32, last - base);
            float logit = -INFINITY;
            if (lane < n) {
                const T* row = k + (int64_t)(base + lane) * p.ks[2];
                float dot = 0.0f;
                for (int c = 0; c < p.d; ++c) dot = __fmaf_rn(qrow[c], to_f(row[c]), dot);
                logit = __fmul_rn(dot, p.scale);
            }
            float top = logit;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float m_new = fmaxf(m, top);
            const float ref = m_new == -INFINITY ? 0.0f : m_new;      // nothing but -inf so far: weights of 0
            const float alpha = expf(m - ref);
            const float w = lane < n ? expf(logit - ref) : 0.0f;
            float sum = w;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            den = __fmaf_rn(den, alpha, sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __fmul_rn(acc[e], alpha);
            for (int j = 0; j < n; ++j) {
                const float wj = __shfl_sync(0xffffffffu, w, j);
                const T* row = v + (int64_t)(base + j) * p.vs[2];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (lane + 32 * e < p.d) acc[e] = __fmaf_rn(wj, to_f(row[lane + 32 * e]), acc[e]);
            }
            m = m_new;
        }
    }
    T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + i * p.os[2];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < p.d) out[lane + 32 * e] = from_f<T>(den == 0.0f ? 0.0f : acc[e] / den);
}

template <typename T>
__global__ void __launch_bounds__(256) window_row_kernel(const __grid_constant__ WinParams p) {
    pdl_wait();
    pdl_open();
    __shared__ float qrow[8][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * 8 + warp;
    if (i >= p.sq) return;
    window_row<T>(p, blockIdx.y / p.heads, blockIdx.y % p.heads, i, qrow[warp], lane);
}

}  // namespace

size_t window_workspace_bytes(const vcb_window_args*) { return 0; }

int window_run(const vcb_window_args* a, cudaStream_t st) {
    WinParams p{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
    p.kv_lens = a->kv_lens;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.os[i] = a->out_stride[i];
    }
    p.sq = a->sq; p.sk = a->sk; p.heads = a->heads;
    p.left = a->left; p.right = a->right; p.sinks = a->sinks;
    p.causal = a->causal; p.has_offset = a->has_offset; p.q_offset = a->q_offset;
    p.d = a->d; p.scale = a->scale;
    const dim3 grid((unsigned)((a->sq + 7) / 8), (unsigned)(a->batch * a->heads));
    if (a->dtype == VCB_BF16) VCB_CUDA(launch_pdl(window_row_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p));
    else VCB_CUDA(launch_pdl(window_row_kernel<__half>, grid, dim3(256), 0, st, p));
    return VCB_OK;
}

}  // namespace vcb
