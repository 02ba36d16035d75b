// Matrix product with bias, activation, gate and residual in its epilogue:
//   y[m, n] = residual[m, n] + gate[m, n] * act(sum_k x[m, k] w[n, k] + bias[n])
// for the projections around the attention.  x is token-major or the
// attention's head-major output, y token-major or the head-major input of the
// attention, so neither side needs a transposing copy.  Products are summed
// in FP32 (tensor memory) and rounded once, at the store.
//
// Bound: the tensor cores (2 M N K operations) once M passes a few hundred
// rows, the weights' N K bytes below.
//
// Work decomposition.  Two CTAs form a cluster; the pair's tile is 256 rows of
// x by BN rows of w, multiplied by tcgen05.mma.cta_group::2 (M = 256), issued
// by one thread of the even CTA.  Each CTA loads its 128 rows of x and half of
// the w rows, 64 channels (128 swizzled bytes) a stage.  K is walked head by
// head: x is [batch, head, token, channel] and w [n, head, channel] to the
// TMA (one head for token-major x), and channels behind a head's last are
// zero-filled on both sides.  The grid is persistent; tiles are walked in
// groups of kGroup row tiles, so that the pairs at work share w tiles and a
// few row tiles in L2.
//
// Roles per CTA (384 threads): warp 0 TMA producer, warp 1 MMA issuer (even
// CTA), warp 2 tensor memory, warps 4-11 epilogue.  Two accumulators alternate
// in tensor memory, so a tile's epilogue runs under the next tile's products.
// Epilogue: a warp owns 32 rows and half the columns; it turns 32 x 32 blocks
// through shared memory (FP32, swizzled, no bank conflicts) so that four lanes
// hold 32 consecutive columns of a row: bias, gate and residual are read and y
// written in 64-byte runs.
//
// Operands that TMA cannot address (rows or bases off the 16-byte grid) are
// first copied, padded, into the caller's workspace.
//
// Every mbarrier wait is bounded (vcb_attn_pair.cuh); a CTA that gives up
// tells its peer, and the pair drains and frees its tensor memory together.
#include "vcb_f16.cuh"

namespace vcb {
namespace {

constexpr int kLinThreads = 384;
constexpr int kBK = 64;                            // channels per stage: 128 bytes
constexpr uint32_t kABytes = 128 * kBK * 2;        // one CTA's x tile of a stage
constexpr int kGroup = 8;                          // row tiles that share their walk over w
constexpr int kEpiWarps = 8;
constexpr uint32_t kEpiBytes = 32 * 32 * 4;        // one epilogue warp's staging block

template <int BN> struct Tile {
    static constexpr uint32_t kBBytes = BN / 2 * kBK * 2;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = BN == 256 ? 6 : BN == 128 ? 7 : 8;
    static constexpr uint32_t kOffEpi = kStages * kStageBytes;
    static constexpr uint32_t kOffBars = kOffEpi + kEpiWarps * kEpiBytes;
    static constexpr int kNumBars = 2 * kStages + 2 + 2 + 1;
    static constexpr uint32_t kOffMisc = kOffBars + kNumBars * 8;
    static constexpr uint32_t kSmem = kOffMisc + 16;
    static constexpr uint32_t kCols = 2 * BN;
    static_assert(kStageBytes % 1024 == 0, "swizzled tiles need 1024-byte aligned stages");
    static_assert(kSmem <= 232448, "shared memory of one CTA");
};

struct LinParams {
    CUtensorMap tm_x;            // [batch][head][token][channel]
    CUtensorMap tm_w;            // [n][head][channel]
    int k_chunks, chunks_per_head;
    int m_tiles, n_tiles, m_tiles_per_batch;
    int64_t rows;                // rows of one walk (tokens, or batch x tokens when collapsed)
    int64_t tokens;
    int collapsed;               // rows run over batch x tokens
    int n, n_head;
    int activation;
    const void* bias;
    const void* gate;
    const void* residual;
    void* y;
    int bias_dtype, gate_dtype;
    int64_t gs_b, gs_s, rs_b, rs_s, ys_b, ys_h, ys_s;
    int vec_y, vec_r, vec_bias, vec_gate;
    int32_t* status;
};

__device__ __forceinline__ void tma_load_4d_pair(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z,
                                                 int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

__device__ __forceinline__ void mma2_f16(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}

struct LinBars {
    uint64_t* full;      // [stages]  even CTA: both CTAs' parts of a stage landed
    uint64_t* empty;     // [stages]  both: the stage's products are done
    uint64_t* acc_full;  // [2]  both: the tile's products are done
    uint64_t* acc_free;  // [2]  even CTA: both CTAs' epilogues have read the accumulator
    uint64_t* drain;     // [1]
};

// Tile t of the walk: groups of kGroup row tiles, w tiles outer within one.
__device__ __forceinline__ void tile_at(const LinParams& p, int t, int& m, int& n) {
    const int per = kGroup * p.n_tiles;
    const int g = t / per, r = t - g * per;
    const int first = g * kGroup;
    const int size = min(kGroup, p.m_tiles - first);
    n = r / size;
    m = first + (r - n * size);
}

template <int BN>
__device__ void lin_producer(const LinParams& p, uint8_t* smem, const LinBars& B, const Waiter& wait, uint32_t rank,
                             int c, int ncl) {
    using L = Tile<BN>;
    prefetch_tmap(&p.tm_x);
    prefetch_tmap(&p.tm_w);
    const uint32_t lead = peer_addr(B.full, 0);
    uint32_t g = 0;
    bool ok = true;
    const int tiles = p.m_tiles * p.n_tiles;
    for (int t = c; ok && t < tiles; t += ncl) {
        int mt, nt;
        tile_at(p, t, mt, nt);
        const int b = mt / p.m_tiles_per_batch;
        const int row = (mt - b * p.m_tiles_per_batch) * 256 + (int)rank * 128;
        const int wrow = nt * BN + (int)rank * (BN / 2);
        int head = 0, x = 0;
        for (int k = 0; k < p.k_chunks; ++k, ++g) {
            const int s = g % L::kStages;
            if (g >= (uint32_t)L::kStages && !wait(&B.empty[s], ((g / L::kStages) - 1) & 1)) {
                ok = false;
                break;
            }
            uint8_t* st = smem + s * L::kStageBytes;
            if (rank == 0) mbar_arrive_expect_tx(&B.full[s], 2 * L::kStageBytes);
            tma_load_4d_pair(st, &p.tm_x, lead + 8 * s, x, row, head, b);
            tma_load_3d_pair(st + kABytes, &p.tm_w, lead + 8 * s, x, head, wrow);
            x += kBK;
            if (x >= p.chunks_per_head * kBK) { x = 0; ++head; }
        }
    }
    if (*wait.abort) {
        // No copy may land after the pair exits: the even CTA's barriers count
        // both CTAs' bytes; the odd CTA gives its copies a bounded millisecond.
        if (rank == 0) {
            for (uint32_t s = 0; s < (uint32_t)L::kStages && s < g; ++s)
                drain_wait(&B.full[s], ((g - 1 - s) / L::kStages) & 1);
        } else {
            const uint64_t t0 = globaltimer();
            while (globaltimer() - t0 < 1000000ull) {
            }
        }
    }
}

template <typename T, int BN>
__device__ void lin_mma(const LinParams& p, uint8_t* smem, const LinBars& B, const Waiter& wait, uint32_t tmem, int c,
                        int ncl) {
    using L = Tile<BN>;
    constexpr uint32_t idesc = idesc_f16<T>(256, BN);
    const uint64_t d64 = smem_desc_k128(smem);
    const uint32_t hi = (uint32_t)(d64 >> 32), lo0 = (uint32_t)d64;
    const int tiles = p.m_tiles * p.n_tiles;
    uint32_t g = 0, li = 0;
    bool ok = true;
    for (int t = c; ok && t < tiles; t += ncl, ++li) {
        const uint32_t buf = li & 1;
        if (li >= 2 && !wait(&B.acc_free[buf], ((li - 2) >> 1) & 1)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        for (int k = 0; k < p.k_chunks; ++k, ++g) {
            const uint32_t s = g % L::kStages;
            if (!wait(&B.full[s], (g / L::kStages) & 1)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t a = lo0 + s * (L::kStageBytes >> 4), w = a + (kABytes >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma2_f16(d, a + 2 * kk, w + 2 * kk, hi, idesc, k > 0 || kk > 0);
            commit_both(&B.empty[s]);
        }
        if (ok) commit_both(&B.acc_full[buf]);
    }
    commit_local_pair(B.drain);
    drain_wait(B.drain, 0);
}

__device__ __forceinline__ float act_of(int kind, float y) {
    switch (kind) {
        case VCB_ACT_SILU: return __fdividef(y, 1.0f + __expf(-y));
        // 0.5 y (1 + erf(y / sqrt 2)), without the cancellation for y < 0
        case VCB_ACT_GELU: return 0.5f * y * erfcf(-0.70710678118654752f * y);
        // 0.5 y (1 + tanh u) = y / (1 + exp(-2 u)), u = sqrt(2/pi) (y + 0.044715 y^3)
        case VCB_ACT_GELU_TANH: {
            const float u2 = 1.5957691216057308f * y * __fmaf_rn(0.044715f * y, y, 1.0f);
            return __fdividef(y, 1.0f + __expf(-u2));
        }
        case VCB_ACT_RELU: return fmax_nan(y, 0.0f);
        default: return y;
    }
}

// Eight consecutive values of a bias, gate or residual row as floats; columns
// at or behind `limit` are not read.
__device__ __forceinline__ void load8_any(const void* p, int64_t i, int dtype, int valid, bool vec, float* o) {
    if (vec && valid >= 8) {
        if (dtype == VCB_F32) {
            const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
            const float4 a = f[0], b = f[1];
            o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float2 f;
                if (dtype == VCB_F16) f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
                else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[e]));
                o[2 * e] = f.x; o[2 * e + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float f = 0.0f;
            if (e < valid) {
                if (dtype == VCB_F32) f = static_cast<const float*>(p)[i + e];
                else if (dtype == VCB_F16) f = __half2float(static_cast<const __half*>(p)[i + e]);
                else f = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i + e]);
            }
            o[e] = f;
        }
    }
}

// Eight accumulated columns n .. n + 7 of one row: act, gate, residual, store.
// f holds the sums with the bias added.
template <typename T>
__device__ __forceinline__ void finish8(const LinParams& p, float* f, int n, int64_t y_off, int64_t g_off,
                                        int64_t r_off) {
    const int valid = p.n - n;
    if (p.activation != VCB_ACT_NONE) {
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = act_of(p.activation, f[e]);
    }
    if (p.gate) {
        float q[8];
        load8_any(p.gate, g_off + n, p.gate_dtype, valid, p.vec_gate, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __fmul_rn(f[e], q[e]);
    }
    if (p.residual) {
        float q[8];
        load8_any(p.residual, r_off + n, F16<T>::kDtype, valid, p.vec_r, q);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = __fadd_rn(f[e], q[e]);
    }
    T* y = static_cast<T*>(p.y) + y_off;
    if (p.vec_y && valid >= 8) {
        const int h = n / p.n_head;
        *reinterpret_cast<uint4*>(y + h * p.ys_h + (n - h * p.n_head)) =
            make_uint4(F16<T>::two(f[0], f[1]), F16<T>::two(f[2], f[3]), F16<T>::two(f[4], f[5]),
                       F16<T>::two(f[6], f[7]));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < valid) {
                const int h = (n + e) / p.n_head;
                y[h * p.ys_h + (n + e - h * p.n_head)] = F16<T>::one(f[e]);
            }
    }
}

template <typename T, int BN>
__device__ void lin_epilogue(const LinParams& p, uint8_t* smem, const LinBars& B, const Waiter& wait, uint32_t tmem,
                             uint32_t rank, int c, int ncl, int ew, int lane) {
    using L = Tile<BN>;
    constexpr int kHalfCols = BN / 2, kChunks = kHalfCols / 32;
    const int quarter = ew & 3, side = ew >> 2;
    const uint32_t lead_free = peer_addr(B.acc_free, 0);
    float4* stage = reinterpret_cast<float4*>(smem + L::kOffEpi + ew * kEpiBytes);
    const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16) + side * kHalfCols;
    const int r0 = lane >> 2, q8 = (lane & 3) * 8;      // this lane's first row and columns in a block
    const int tiles = p.m_tiles * p.n_tiles;
    uint32_t li = 0;
    for (int t = c; t < tiles; t += ncl, ++li) {
        int mt, nt;
        tile_at(p, t, mt, nt);
        const int tb = mt / p.m_tiles_per_batch;
        const int64_t row0 = (int64_t)(mt - tb * p.m_tiles_per_batch) * 256 + rank * 128 + quarter * 32 + r0;
        int64_t y_off[4], g_off[4], r_off[4];
        bool live[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = row0 + 8 * i;
            live[i] = row < p.rows;
            int64_t b = tb, s = row;
            if (p.collapsed) {
                b = p.rows < (1ll << 31) ? (int64_t)((uint32_t)row / (uint32_t)p.tokens) : row / p.tokens;
                s = row - b * p.tokens;
            }
            y_off[i] = b * p.ys_b + s * p.ys_s;
            g_off[i] = b * p.gs_b + s * p.gs_s;
            r_off[i] = b * p.rs_b + s * p.rs_s;
        }
        const uint32_t buf = li & 1;
        if (!wait(&B.acc_full[buf], (li >> 1) & 1)) return;
        tc_fence_after();
#pragma unroll 1
        for (int ch = 0; ch < kChunks; ++ch) {
            uint32_t r[32];
            tmem_ld32_at<0>(trow + buf * BN + ch * 32, r);
            tmem_wait_ld();
            if (ch == kChunks - 1) {
                tc_fence_before();
                __syncwarp();
                mbar_arrive_cluster_if(lead_free + 8 * buf, lane == 0);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                stage[lane * 8 + (j ^ (lane & 7))] =
                    make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]), __uint_as_float(r[4 * j + 2]),
                                __uint_as_float(r[4 * j + 3]));
            __syncwarp();
            const int n = nt * BN + side * kHalfCols + ch * 32 + q8;
            if (n < p.n) {
                float bias[8];
                if (p.bias) load8_any(p.bias, n, p.bias_dtype, p.n - n, p.vec_bias, bias);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r0 + 8 * i;
                    const float4 a = stage[row * 8 + ((q8 >> 2) ^ (row & 7))];
                    const float4 d = stage[row * 8 + (((q8 >> 2) + 1) ^ (row & 7))];
                    float f[8] = {a.x, a.y, a.z, a.w, d.x, d.y, d.z, d.w};
                    if (p.bias) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = __fadd_rn(f[e], bias[e]);
                    }
                    if (live[i]) finish8<T>(p, f, n, y_off[i], g_off[i], r_off[i]);
                }
            }
            __syncwarp();
        }
    }
}

template <typename T, int BN>
__global__ void __launch_bounds__(kLinThreads, 1) linear_kernel(const __grid_constant__ LinParams p) {
    pdl_wait();
    using L = Tile<BN>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) flag_status(p.status, VCB_FLAG_INTERNAL);
        return;
    }
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
    const LinBars B{bars, bars + L::kStages, bars + 2 * L::kStages, bars + 2 * L::kStages + 2,
                    bars + 2 * L::kStages + 4};
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int c = (int)(blockIdx.x >> 1), ncl = (int)(gridDim.x >> 1);
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&B.full[s], 1);
            mbar_init(&B.empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.acc_full[i], 1);
            mbar_init(&B.acc_free[i], 2 * kEpiWarps);
        }
        mbar_init(B.drain, 1);
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 2) {
        tmem_alloc_pair(tmem_slot, L::kCols);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const Waiter wait{abort, peer_addr(const_cast<int*>(abort), rank ^ 1u)};
    if (warp == 0) {
        if (lane == 0) lin_producer<BN>(p, smem, B, wait, rank, c, ncl);
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) lin_mma<T, BN>(p, smem, B, wait, tmem, c, ncl);
    } else if (warp >= 4) {
        lin_epilogue<T, BN>(p, smem, B, wait, tmem, rank, c, ncl, warp - 4, lane);
    }
    tc_fence_before();
    __syncwarp();
    cluster_sync_all();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, L::kCols);
    }
    if (threadIdx.x == 0 && *abort) flag_status(p.status, VCB_FLAG_TIMEOUT);
}

template <typename T, int BN>
int launch_tiles(LinParams& p, cudaStream_t st) {
    static int max_pairs[64] = {};
    using L = Tile<BN>;
    auto kernel = linear_kernel<T, BN>;
    int dev = 0;
    VCB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(VCB_ERR_INVALID_ARGUMENT, "device ordinal %d out of range", dev);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // the kernel begins with pdl_wait()
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(kLinThreads);
    cfg.dynamicSmemBytes = L::kSmem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (max_pairs[dev] == 0) {
        VCB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem));
        cfg.gridDim = dim3(2 * 148);
        int n = 0;
        VCB_CUDA(cudaOccupancyMaxActiveClusters(&n, kernel, &cfg));
        if (n < 1) return fail(VCB_ERR_CUDA, "the projection kernel's CTA pairs do not fit on this GPU");
        max_pairs[dev] = n;
    }
    p.n_tiles = (p.n + BN - 1) / BN;
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles;
    cfg.gridDim = dim3((unsigned)(2 * (tiles < max_pairs[dev] ? tiles : max_pairs[dev])));
    cfg.numAttrs = 2;
    VCB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    return VCB_OK;
}

struct LinPlan {
    bool pack_x, pack_w;
    int64_t pitch;               // elements of a packed row
    size_t off_w, total;
};

LinPlan plan(const vcb_linear_args* a) {
    LinPlan q{};
    const int64_t k = a->heads_in * a->k_head;
    q.pitch = (k + 7) / 8 * 8;
    q.pack_w = !on16(a->w) || !tma_stride(a->w_stride, a->n);
    q.pack_x = !on16(a->x) || (a->heads_in > 1 && !by8(a->k_head)) || !tma_stride(a->x_stride_s, a->tokens) ||
               !tma_stride(a->x_stride_h, a->heads_in) || !tma_stride(a->x_stride_b, a->batch);
    auto r = [](size_t v) { return (v + 255) & ~size_t(255); };
    q.off_w = q.pack_x ? r((size_t)(a->batch * a->tokens * q.pitch) * 2) : 0;
    q.total = q.off_w + (q.pack_w ? r((size_t)(a->n * q.pitch) * 2) : 0);
    return q;
}

}  // namespace

size_t linear_workspace_bytes(const vcb_linear_args* a) { return plan(a).total; }

int linear_run(const vcb_linear_args* a, cudaStream_t st) {
    const LinPlan q = plan(a);
    const int64_t k = a->heads_in * a->k_head;
    const void* x = a->x;
    const void* w = a->w;
    int64_t heads = a->heads_in, k_head = a->k_head, w_stride = a->w_stride;
    int64_t xb = a->x_stride_b, xh = a->x_stride_h, xs = a->x_stride_s;
    if (q.pack_x || q.pack_w) {
        PackParams pk{};
        pk.channels = (int)k;
        pk.pitch = (int)q.pitch;
        char* ws = static_cast<char*>(a->workspace);
        int64_t blocks = 0;
        if (q.pack_x) {
            const int64_t rows = a->batch * a->tokens;
            pk.side[0] = {static_cast<const uint16_t*>(x), reinterpret_cast<uint16_t*>(ws), rows, a->tokens, xb, xs, 1,
                          0, xh, (int)a->k_head};
            blocks += (rows + 7) / 8;
            x = ws;
            xs = q.pitch; xh = k; xb = a->tokens * q.pitch;
        }
        pk.end[0] = blocks;
        if (q.pack_w) {
            pk.side[1] = {static_cast<const uint16_t*>(w), reinterpret_cast<uint16_t*>(ws + q.off_w), a->n, a->n, 0,
                          a->w_stride, 1, 0, k, (int)k};
            blocks += (a->n + 7) / 8;
            w = ws + q.off_w;
            w_stride = q.pitch;
        }
        pk.end[1] = pk.end[2] = blocks;
        if (q.pack_x) { heads = 1; k_head = k; }      // a packed row has its heads joined
        VCB_CUDA(launch_pack(pk, st));
    }
    LinParams p;
    memset(&p, 0, sizeof(p));
    const bool bf16 = a->dtype == VCB_BF16;
    // one walk over batch x tokens where the rows are evenly spaced
    p.collapsed = heads == 1 && (a->batch == 1 || a->tokens == 1 || xb == a->tokens * xs);
    if (p.collapsed && a->tokens == 1 && a->batch > 1) xs = xb;
    const int64_t rows = p.collapsed ? a->batch * a->tokens : a->tokens;
    const int64_t batches = p.collapsed ? 1 : a->batch;
    // strides of axes of length one are never taken: any legal value will do
    const int64_t row = (k_head + 7) / 8 * 8;
    if (rows == 1) xs = row;
    if (heads == 1) xh = row;
    if (batches == 1) xb = row;
    if (a->n == 1) w_stride = row * heads;
    {
        const cuuint64_t dims[4] = {(cuuint64_t)k_head, (cuuint64_t)rows, (cuuint64_t)heads, (cuuint64_t)batches};
        const cuuint64_t strides[3] = {(cuuint64_t)xs * 2, (cuuint64_t)xh * 2, (cuuint64_t)xb * 2};
        const cuuint32_t box[4] = {kBK, 128, 1, 1};
        int rc = make_map16(&p.tm_x, x, bf16, 4, dims, strides, box);
        if (rc) return rc;
    }
    const int64_t m_per_batch = (rows + 255) / 256;
    const int64_t m_tiles = m_per_batch * batches;
    // Tile width: 256 columns need the fewest loads per product; narrower ones
    // give small products a tile for more of the SM pairs.
    const int pairs = sm_count() / 2;
    int bn = 256;
    if (m_tiles * ((a->n + 255) / 256) < pairs) bn = m_tiles * ((a->n + 127) / 128) < pairs ? 64 : 128;
    {
        const cuuint64_t dims[3] = {(cuuint64_t)k_head, (cuuint64_t)heads, (cuuint64_t)a->n};
        const cuuint64_t strides[2] = {(cuuint64_t)row * 2, (cuuint64_t)w_stride * 2};
        const cuuint32_t box[3] = {kBK, 1, (cuuint32_t)(bn / 2)};
        int rc = make_map16(&p.tm_w, w, bf16, 3, dims, strides, box);
        if (rc) return rc;
    }
    p.chunks_per_head = (int)((k_head + kBK - 1) / kBK);
    p.k_chunks = (int)(p.chunks_per_head * heads);
    if (m_tiles * ((a->n + 63) / 64) >= (1ll << 30) || ((m_tiles * ((a->n + bn - 1) / bn) + 73) / 74) * p.k_chunks >= (1ll << 31))
        return fail(VCB_ERR_INVALID_ARGUMENT, "product too large for the projection kernel's tile counters");
    p.m_tiles = (int)m_tiles;
    p.m_tiles_per_batch = (int)m_per_batch;
    p.rows = rows;
    p.tokens = a->tokens;
    p.n = (int)a->n;
    p.n_head = (int)a->n_head;
    p.activation = a->activation;
    p.bias = a->bias; p.bias_dtype = a->bias_dtype;
    p.gate = a->gate; p.gate_dtype = a->gate_dtype; p.gs_b = a->gate_stride_b; p.gs_s = a->gate_stride_s;
    p.residual = a->residual; p.rs_b = a->residual_stride_b; p.rs_s = a->residual_stride_s;
    p.y = a->y; p.ys_b = a->y_stride_b; p.ys_h = a->y_stride_h; p.ys_s = a->y_stride_s;
    p.vec_y = on16(a->y) && by8(a->n_head) && by8(a->y_stride_b) && by8(a->y_stride_h) && by8(a->y_stride_s);
    p.vec_r = on16(a->residual) && by8(a->residual_stride_b) && by8(a->residual_stride_s);
    p.vec_bias = on16(a->bias);
    p.vec_gate = on16(a->gate) && by8(a->gate_stride_b) && by8(a->gate_stride_s);
    p.status = a->status;
    if (bf16) {
        if (bn == 256) return launch_tiles<__nv_bfloat16, 256>(p, st);
        if (bn == 128) return launch_tiles<__nv_bfloat16, 128>(p, st);
        return launch_tiles<__nv_bfloat16, 64>(p, st);
    }
    if (bn == 256) return launch_tiles<__half, 256>(p, st);
    if (bn == 128) return launch_tiles<__half, 128>(p, st);
    return launch_tiles<__half, 64>(p, st);
}

}  // namespace vcb
