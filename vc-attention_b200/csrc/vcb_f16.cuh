// Pieces shared by the 16-bit tensor-core kernels (vcb_linear.cu,
// vcb_window.cu): TMA maps of strided 16-bit tensors, kind::f16 descriptors,
// conversions, and the copy that lines up operands which TMA cannot address.
// Every definition has internal linkage.
#pragma once
#include <cstring>

#include "vcb_attn_pair.cuh"

namespace vcb {
namespace {

// Instruction descriptor, kind::f16: F32 D (c_format [4,6) = 1), A and B both
// FP16 (0) or both BF16 (1) at [7,10) and [10,13), A K-major, B K-major or
// (bit 16) N-major.
template <typename T> struct F16;
template <> struct F16<__half> {
    static constexpr int kDtype = VCB_F16;
    static constexpr uint32_t kFormat = 0;
    static __device__ __forceinline__ float to(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half one(float f) { return __float2half_rn(f); }
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 both(uint32_t u) { return __half22float2(*reinterpret_cast<__half2*>(&u)); }
};
template <> struct F16<__nv_bfloat16> {
    static constexpr int kDtype = VCB_BF16;
    static constexpr uint32_t kFormat = 1;
    static __device__ __forceinline__ float to(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 one(float f) { return __float2bfloat16_rn(f); }
    static __device__ __forceinline__ uint32_t two(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ float2 both(uint32_t u) {
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
};
template <typename T> __host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool b_n_major = false) {
    return (1u << 4) | (F16<T>::kFormat << 7) | (F16<T>::kFormat << 10) | ((b_n_major ? 1u : 0u) << 16) |
           ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

int make_map16(CUtensorMap* map, const void* base, bool bf16, int rank, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeTiledFn enc;
    int rc = get_encoder(&enc);
    if (rc) return rc;
    const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
                     const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(VCB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return VCB_OK;
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool by8(int64_t v) { return v % 8 == 0; }
// a stride that TMA can take along an axis of n entries (16-byte steps, forward)
bool tma_stride(int64_t s, int64_t n) { return n == 1 || (by8(s) && s > 0); }

// Rows of `channels` elements ([batch][token][head][head_dim], strides in
// elements) into rows of `pitch` elements, zero behind the last channel.
// Row order: tokens inner, outer (batch or batch x head) outer.
struct PackSide {
    const uint16_t* src;
    uint16_t* dst;
    int64_t rows, tokens;                 // row r is (r / tokens, r % tokens)
    int64_t s_b, s_s;                     // strides of the outer index and of a token
    int64_t inner, s_i;                   // the outer index is (r / tokens / inner, % inner); stride of the latter
    int64_t s_h;                          // stride of a head within a row
    int head_dim;                         // channels per head within a row
};
struct PackParams {
    PackSide side[3];
    int64_t end[3];                       // first block behind side i
    int channels, pitch;
};
__global__ void __launch_bounds__(256) pack_rows_kernel(const __grid_constant__ PackParams p) {
    pdl_wait();
    pdl_open();
    const int64_t block = blockIdx.x;
    const int which = block < p.end[0] ? 0 : block < p.end[1] ? 1 : 2;
    const PackSide& s = p.side[which];
    const int64_t row = (block - (which ? p.end[which - 1] : 0)) * 8 + (threadIdx.x >> 5);
    if (row >= s.rows) return;
    const int64_t o = row / s.tokens, t = row - o * s.tokens;
    const int64_t b = o / s.inner, i = o - b * s.inner;
    const uint16_t* src = s.src + b * s.s_b + i * s.s_i + t * s.s_s;
    uint4* dst = reinterpret_cast<uint4*>(s.dst + row * p.pitch);
    // eight channels per lane, all reads in flight before the 16-byte store
    for (int c = 8 * (threadIdx.x & 31); c < p.pitch; c += 256) {
        uint32_t v[8];
        int h = c / s.head_dim, k = c - h * s.head_dim;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = c + e < p.channels ? src[h * s.s_h + k] : 0u;
            if (++k == s.head_dim) { k = 0; ++h; }
        }
        dst[c / 8] = make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
}
cudaError_t launch_pack(const PackParams& p, cudaStream_t st) {
    return launch_pdl(pack_rows_kernel, dim3((unsigned)p.end[2]), dim3(256), 0, st, p);
}

}  // namespace
}  // namespace vcb
