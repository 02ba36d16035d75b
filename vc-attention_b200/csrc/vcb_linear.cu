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
// x by bn rows of w (a multiple of 32, up to 256, chosen in plan()), multiplied by
// tcgen05.mma.cta_group::2 (M = 256), issued by an elected lane of a converged warp
// of the even CTA: the loop of a lone thread took 570 clocks per 64 channels.
// Each CTA loads its 128 rows of x and half of the w rows, 64 channels (128 swizzled bytes) a stage.  K is walked head by
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
// Tiles that do not fill the last round of pairs are cut along K: their 64-channel
// chunks are dealt evenly to all pairs (LinWork), a piece that is not a whole
// tile goes to the workspace in FP32, and linear_join_kernel adds a tile's
// pieces in order and runs the epilogue.
//
// Up to kFewRows rows the product is a stream over w: linear_few_kernel reads w
// straight into mma.sync fragments (tcgen05 would spend its 128-row tile on
// them), 16 rows of w per CTA, K dealt to its eight warps.
//
// Measured, 1 B200, BF16: 32768 x 5120 x 15360 3.72-3.92 ms (1315-1384 TFLOP/s) at
// the power limit; 8192 x 5120 x 5120 273 us with the tensor pipe 90 % active;
// 64 rows 15.6 us; one row 15.6 us cold (52 MB), 10.2 us with w in L2; 771 x 1147 x
// 2049 with GELU and residual, off the 16-byte grid, 25.5 us after a copy of 8 us.
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
// Row tiles that share their walk over w.  32768 x 5120 x 15360 BF16, seconds on end
// at the power limit, with an earlier issue loop (now 3.72-3.92 ms at 12): 4 tiles
// 4.60 ms, 8 4.18, 12 4.12, 16 4.16, 24 4.32, 32 4.57.
constexpr int kGroup = 12;
constexpr int kEpiWarps = 8;
constexpr uint32_t kEpiBytes = 32 * 32 * 4;        // one epilogue warp's staging block

// Shared and tensor memory for tiles of up to BN columns (a launch's are p.bn).
template <int BN> struct Tile {
    static constexpr uint32_t kBBytes = BN / 2 * kBK * 2;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = BN == 256 ? 6 : 7;
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
    int bn;                      // columns of a tile: a multiple of 32
    int k_chunks, chunks_per_head;
    int m_tiles, n_tiles, m_tiles_per_batch;
    int64_t rows;                // rows of one walk (tokens, or batch x tokens when collapsed)
    int64_t tokens;
    int collapsed;               // rows run over batch x tokens
    int n, n_head;
    int dp_tiles;                // tiles walked whole; the rest is cut along K
    int cut_units, cut_each;     // chunks of the cut tiles, and of one pair's share
    float* part;                 // [2 per pair][256][bn]
    int activation;
    const void* bias;
    const void* gate;
    const void* residual;
    void* y;
    int bias_dtype, gate_dtype;
    int64_t gs_b, gs_s, rs_b, rs_s, ys_b, ys_h, ys_s;
    int vec;                     // y, bias, gate and residual in whole, aligned 16-byte runs
    int32_t* status;
};

// One stage, by the elected lane of a converged warp (operands in uniform
// registers, as for the MMAs): expect the pair's bytes (even CTA), load this
// CTA's x rows and w rows.
__device__ __forceinline__ void load_stage(uint32_t dst_x, uint32_t dst_w, const CUtensorMap* mx, const CUtensorMap* mw,
                                           uint32_t own_bar, uint32_t bytes, uint32_t bar, int k, int row, int wrow, int head,
                                           int batch) {
    asm volatile(
        "{\n\t.reg .pred q, e;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "setp.ne.and.u32 e, %5, 0, q;\n\t"
        "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%4], %5;\n\t"
        "@q cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%2, {%7, %8, %10, %11}], [%6];\n\t"
        "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%1], [%3, {%7, %10, %9}], [%6];\n\t}"
        ::"r"(dst_x), "r"(dst_w), "l"(mx), "l"(mw), "r"(own_bar), "r"(bytes), "r"(bar), "r"(k), "r"(row), "r"(wrow),
          "r"(head), "r"(batch)
        : "memory");
}

// The whole warp runs the issue loop and one elected lane issues, so that the
// operands stay in uniform registers: a lone thread's were moved there before
// every MMA, and a chunk of four took 570 clocks to issue whatever its width.
__device__ __forceinline__ void mma2_f16(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                         uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}

// commits of the elected lane's MMAs (the same lane every time)
__device__ __forceinline__ void commit_both_elected(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}"
        ::"r"(smem_u32(bar)), "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void commit_local_elected(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(smem_u32(bar))
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

// The i-th piece of work of pair c: a tile and its chunks [k0, k1); slot < 0
// for a whole tile, else its place among the partial sums.  First every
// ncl-th whole tile, then the pair's share of the cut tiles, which covers the
// end of one tile, whole tiles and the beginning of another: two slots suffice.
struct LinWork {
    int tile, k0, k1, slot;
    __device__ __forceinline__ bool get(const LinParams& p, int c, int ncl, int i) {
        const int whole = local_items(p.dp_tiles, c, ncl);
        if (i < whole) {
            tile = c + i * ncl;
            k0 = 0; k1 = p.k_chunks; slot = -1;
            return true;
        }
        const int64_t a64 = (int64_t)c * p.cut_each;
        if (a64 >= p.cut_units) return false;
        const int a = (int)a64, b = min(p.cut_units - a, p.cut_each) + a;
        const int t = a / p.k_chunks + i - whole;
        const int begin = max(a, t * p.k_chunks), end = min(b, (t + 1) * p.k_chunks);
        if (begin >= end) return false;
        tile = p.dp_tiles + t;
        k0 = begin - t * p.k_chunks; k1 = end - t * p.k_chunks;
        slot = k1 - k0 == p.k_chunks ? -1 : 2 * c + (begin == a ? 0 : 1);
        return true;
    }
};

template <int BN>
__device__ void lin_producer(const LinParams& p, uint8_t* smem, const LinBars& B, const Waiter& wait, uint32_t rank,
                             int c, int ncl) {
    using L = Tile<BN>;
    const uint32_t lead = __shfl_sync(0xffffffffu, peer_addr(B.full, 0), 0), full0 = smem_u32(B.full), base = smem_u32(smem);
    const uint32_t bytes = 2 * (kABytes + (uint32_t)p.bn / 2 * kBK * 2);
    uint32_t g = 0;
    bool ok = true;
    LinWork wk;
    for (int i = 0; ok && wk.get(p, c, ncl, i); ++i) {
        int mt, nt;
        tile_at(p, wk.tile, mt, nt);
        const int b = mt / p.m_tiles_per_batch;
        const int row = (mt - b * p.m_tiles_per_batch) * 256 + (int)rank * 128;
        const int wrow = nt * p.bn + (int)rank * (p.bn / 2);
        int head = wk.k0 / p.chunks_per_head, x = (wk.k0 - head * p.chunks_per_head) * kBK;
        for (int k = wk.k0; k < wk.k1; ++k, ++g) {
            const int s = g % L::kStages;
            if (g >= (uint32_t)L::kStages && !wait.parked(&B.empty[s], ((g / L::kStages) - 1) & 1)) {
                ok = false;
                break;
            }
            const uint32_t st = base + s * L::kStageBytes;
            load_stage(st, st + kABytes, &p.tm_x, &p.tm_w, full0 + 8 * s, rank == 0 ? bytes : 0u, lead + 8 * s, x, row, wrow,
                       head, b);
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
__device__ void lin_mma(const LinParams& p, uint8_t* smem, const LinBars& B, const Waiter& wait, uint32_t tmem0, int c,
                        int ncl) {
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem0, 0);      // uniform
    using L = Tile<BN>;
    const uint32_t idesc = idesc_f16<T>(256, p.bn);
    const uint64_t d64 = smem_desc_k128(smem);
    const uint32_t hi = (uint32_t)(d64 >> 32), lo0 = (uint32_t)d64;
    uint32_t g = 0;
    bool ok = true;
    LinWork wk;
    for (int i = 0; ok && wk.get(p, c, ncl, i); ++i) {
        const uint32_t buf = i & 1;
        if (i >= 2 && !wait(&B.acc_free[buf], ((i - 2) >> 1) & 1)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * BN;
        for (int k = wk.k0; k < wk.k1; ++k, ++g) {
            const uint32_t s = g % L::kStages;
            if (!wait(&B.full[s], (g / L::kStages) & 1)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t a = lo0 + s * (L::kStageBytes >> 4), w = a + (kABytes >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) mma2_f16(d, a + 2 * kk, w + 2 * kk, hi, idesc, k > wk.k0 || kk > 0);
            commit_both_elected(&B.empty[s]);
        }
        if (ok) commit_both_elected(&B.acc_full[buf]);
    }
    commit_local_elected(B.drain);
    drain_wait(B.drain, 0);
}

// 0.5 y (1 + erf(y / sqrt 2)) without the cancellation for y < 0: with
// z = |y| / sqrt 2 and t = 1 / (1 + 0.45 z), erfc(z) = t q(t) exp(-z^2), q a degree-7
// fit to erfc(z) exp(z^2) / t over z in [0, 60] (least squares reweighted towards
// the largest relative error, which is 6.7e-7).  No branches.
__device__ __forceinline__ float gelu_erf(float y) {
    const float z = 0.70710678118654752f * fabsf(y);
    const float t = __fdividef(1.0f, __fmaf_rn(0.45f, z, 1.0f));
    float q = 0.0671004429f;
    q = __fmaf_rn(q, t, -0.242869869f);
    q = __fmaf_rn(q, t, 0.216092497f);
    q = __fmaf_rn(q, t, 0.0311580617f);
    q = __fmaf_rn(q, t, 0.194682702f);
    q = __fmaf_rn(q, t, 0.225934967f);
    q = __fmaf_rn(q, t, 0.254018039f);
    q = __fmaf_rn(q, t, 0.253882557f);
    const float e = 0.5f * t * q * __expf(-z * z);
    return y * (y < 0.0f ? e : 1.0f - e);
}

__device__ __forceinline__ float silu(float y) { return __fdividef(y, 1.0f + __expf(-y)); }
// 0.5 y (1 + tanh u) = y / (1 + exp(-2 u)), u = sqrt(2/pi) (y + 0.044715 y^3)
__device__ __forceinline__ float gelu_tanh(float y) {
    return __fdividef(y, 1.0f + __expf(-1.5957691216057308f * y * __fmaf_rn(0.044715f * y, y, 1.0f)));
}

template <int N> __device__ __forceinline__ void activate(int kind, float (&f)[N]) {
    switch (kind) {                     // the same for all threads
        case VCB_ACT_SILU:
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = silu(f[e]);
            break;
        case VCB_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = gelu_erf(f[e]);
            break;
        case VCB_ACT_GELU_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = gelu_tanh(f[e]);
            break;
        case VCB_ACT_RELU:
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = fmax_nan(f[e], 0.0f);
            break;
        default: break;
    }
}

__device__ __forceinline__ float load1_any(const void* p, int64_t i, int dtype) {
    if (dtype == VCB_F32) return static_cast<const float*>(p)[i];
    if (dtype == VCB_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Eight consecutive values of a bias or gate row as floats: 16-byte aligned
// (VEC), or one by one and none at or behind `valid`.
template <bool VEC>
__device__ __forceinline__ void load8_any(const void* p, int64_t i, int dtype, int valid, float* o) {
    if (!VEC) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = e < valid ? load1_any(p, i + e, dtype) : 0.0f;
    } else if (dtype == VCB_F32) {
        const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
        const float4 a = f[0], b = f[1];
        o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w; o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = dtype == VCB_F16 ? F16<__half>::both(w[e]) : F16<__nv_bfloat16>::both(w[e]);
            o[2 * e] = f.x; o[2 * e + 1] = f.y;
        }
    }
}

// Where a row's output, gate and residual begin.
struct RowAt {
    int64_t y, g, r;
    bool live;
};
__device__ __forceinline__ RowAt row_at(const LinParams& p, int64_t b, int64_t row) {
    int64_t s = row;
    if (p.collapsed) {
        b = (uint32_t)row / (uint32_t)p.tokens;
        s = row - b * p.tokens;
    }
    return {b * p.ys_b + s * p.ys_s, b * p.gs_b + s * p.gs_s, b * p.rs_b + s * p.rs_s, row < p.rows};
}

// Bias, activation and gate on ROWS rows of a 32 x 32 block, eight columns
// n .. n + 7 of each (fewer at the last column when not VEC).
template <bool VEC, int ROWS = 4>
__device__ __forceinline__ void finish_rows(const LinParams& p, float (&f)[4][8], int n, const RowAt* at) {
    float bias[8];
    if (p.bias) load8_any<VEC>(p.bias, n, p.bias_dtype, p.n - n, bias);
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        float gate[8];
        if (p.gate && at[i].live) load8_any<VEC>(p.gate, at[i].g + n, p.gate_dtype, p.n - n, gate);
        if (p.bias) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i][e] = __fadd_rn(f[i][e], bias[e]);
        }
        activate(p.activation, f[i]);
        if (p.gate && at[i].live) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[i][e] = __fmul_rn(f[i][e], gate[e]);
        }
    }
}
template <typename T> __device__ __forceinline__ void add_residual(float (&f)[8], const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 q = F16<T>::both(w[e]);
        f[2 * e] = __fadd_rn(f[2 * e], q.x);
        f[2 * e + 1] = __fadd_rn(f[2 * e + 1], q.y);
    }
}
template <typename T> __device__ __forceinline__ uint4 pack8(const float (&f)[8]) {
    return make_uint4(F16<T>::two(f[0], f[1]), F16<T>::two(f[2], f[3]), F16<T>::two(f[4], f[5]), F16<T>::two(f[6], f[7]));
}

// One sum's epilogue, for outputs off the 16-byte grid and the small kernels:
// column n = head h, channel col.
template <typename T>
__device__ __forceinline__ float finish1(const LinParams& p, float f, float bias, int n, const RowAt& at, float residual) {
    float v[1] = {__fadd_rn(f, bias)};
    activate(p.activation, v);
    f = v[0];
    if (p.gate) f = __fmul_rn(f, load1_any(p.gate, at.g + n, p.gate_dtype));
    return p.residual ? __fadd_rn(f, residual) : f;
}

// VEC: bias, gate, residual and y on the 16-byte grid.  (One kernel for both kept
// the registers of the other way too: 4096 x 1280 x 5120 58 us instead of 46.)
template <typename T, int BN, bool VEC>
__device__ void lin_epilogue(const LinParams& p, uint8_t* smem, const LinBars& B, const Waiter& wait, uint32_t tmem,
                             uint32_t rank, int c, int ncl, int ew, int lane) {
    using L = Tile<BN>;
    const int quarter = ew & 3, side = ew >> 2;
    const uint32_t lead_free = peer_addr(B.acc_free, 0);
    float4* stage = reinterpret_cast<float4*>(smem + L::kOffEpi + ew * kEpiBytes);
    const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16);
    const int chunks = p.bn / 32;                       // 32-column blocks; this warp takes every second one
    const int r0 = lane >> 2, q8 = (lane & 3) * 8;      // this lane's first row and columns in a block
    LinWork wk;
    for (int li = 0; wk.get(p, c, ncl, li); ++li) {
        int mt, nt;
        tile_at(p, wk.tile, mt, nt);
        const int tb = mt / p.m_tiles_per_batch;
        const int64_t row0 = (int64_t)(mt - tb * p.m_tiles_per_batch) * 256 + rank * 128 + quarter * 32 + r0;
        RowAt at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) at[i] = row_at(p, tb, row0 + 8 * i);
        float* part = wk.slot < 0 ? nullptr
                                  : p.part + ((int64_t)wk.slot * 256 + rank * 128 + quarter * 32 + r0) * p.bn +
                                        4 * (lane & 3);
        const uint32_t buf = li & 1;
        // Off the 16-byte grid the residual and y are read and written one column
        // per lane: lane r knows where row r of the block begins.
        RowAt mine{};
        if constexpr (!VEC) mine = row_at(p, tb, row0 - r0 + lane);
        const int live = (int)max((int64_t)0, min((int64_t)32, p.rows - (row0 - r0)));
        // the residual's runs of the next block, a block ahead (no other block's
        // output touches them, so y may be the residual itself); off the grid this
        // lane's column, rows 2 i and 2 i + 1 in word i
        const bool ahead = p.residual && !part;
        uint4 next[4];
        auto fetch = [&](int ch) {
            const int n = nt * p.bn + ch * 32 + q8;
            if constexpr (!VEC) {
                if (!ahead) return;
                const int nl = nt * p.bn + ch * 32 + lane;
                const uint16_t* src = static_cast<const uint16_t*>(p.residual) + nl;
                uint32_t v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int64_t o0 = __shfl_sync(0xffffffffu, mine.r, 2 * i);
                    const int64_t o1 = __shfl_sync(0xffffffffu, mine.r, 2 * i + 1);
                    const uint32_t lo = nl < p.n && 2 * i < live ? src[o0] : 0;
                    const uint32_t hi = nl < p.n && 2 * i + 1 < live ? src[o1] : 0;
                    v[i] = lo | hi << 16;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) next[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            } else if (ahead && n < p.n) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at[i].live) next[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) + at[i].r + n);
            }
        };
        fetch(side);
        if (!wait.parked(&B.acc_full[buf], (li >> 1) & 1)) return;
        tc_fence_after();
        if (side >= chunks) mbar_arrive_cluster_if(lead_free + 8 * buf, lane == 0);
#pragma unroll 1
        for (int ch = side; ch < chunks; ch += 2) {
            uint4 res[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) res[i] = next[i];
            if (ch + 2 < chunks) fetch(ch + 2);
            uint32_t r[32];
            tmem_ld32_at<0>(trow + buf * BN + ch * 32, r);
            tmem_wait_ld();
            if (ch + 2 >= chunks) {
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
            const int n0 = nt * p.bn + ch * 32;
            if (part) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r0 + 8 * i;
                    if (!at[i].live) continue;
                    float4* to = reinterpret_cast<float4*>(part + (int64_t)(8 * i) * p.bn + ch * 32);
                    to[0] = stage[row * 8 + ((lane & 3) ^ (row & 7))];             // 64-byte runs of a row
                    to[4] = stage[row * 8 + (((lane & 3) + 4) ^ (row & 7))];
                }
            } else {
                const int n = n0 + q8;
                float f[4][8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int row = r0 + 8 * i;
                    const float4 a = stage[row * 8 + ((q8 >> 2) ^ (row & 7))];
                    const float4 d = stage[row * 8 + (((q8 >> 2) + 1) ^ (row & 7))];
                    f[i][0] = a.x; f[i][1] = a.y; f[i][2] = a.z; f[i][3] = a.w;
                    f[i][4] = d.x; f[i][5] = d.y; f[i][6] = d.z; f[i][7] = d.w;
                }
                if constexpr (VEC) {
                    if (n < p.n) {
                        finish_rows<true>(p, f, n, at);
                        const int h = n / p.n_head;
                        T* y = static_cast<T*>(p.y) + h * p.ys_h + (n - h * p.n_head);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (p.residual) add_residual<T>(f[i], res[i]);
                            if (at[i].live) *reinterpret_cast<uint4*>(y + at[i].y) = pack8<T>(f[i]);
                        }
                    }
                } else {
                    // Off the 16-byte grid: the residual comes in and y goes out one
                    // column per lane (64-byte runs), through the same block.
                    uint16_t* block = reinterpret_cast<uint16_t*>(stage);       // [32 rows][32 columns]
                    const int nl = n0 + lane;
                    __syncwarp();
                    if (p.residual) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t v[4] = {res[i].x, res[i].y, res[i].z, res[i].w};
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                block[(8 * i + 2 * e) * 32 + lane] = (uint16_t)v[e];
                                block[(8 * i + 2 * e + 1) * 32 + lane] = (uint16_t)(v[e] >> 16);
                            }
                        }
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 4; ++i) res[i] = *reinterpret_cast<const uint4*>(block + (r0 + 8 * i) * 32 + q8);
                    }
                    finish_rows<false>(p, f, n, at);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (p.residual) add_residual<T>(f[i], res[i]);
                        *reinterpret_cast<uint4*>(block + (r0 + 8 * i) * 32 + q8) = pack8<T>(f[i]);
                    }
                    __syncwarp();
                    const int h = nl / p.n_head;
                    uint16_t* dst = static_cast<uint16_t*>(p.y) + h * p.ys_h + (nl - h * p.n_head);
#pragma unroll
                    for (int r8 = 0; r8 < 32; r8 += 8) {
                        uint16_t v[8];                          // (shared loads before any store: they may not pass it)
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] = block[(r8 + e) * 32 + lane];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int64_t off = __shfl_sync(0xffffffffu, mine.y, r8 + e);
                            if (nl < p.n && r8 + e < live) dst[off] = v[e];
                        }
                    }
                }
            }
            __syncwarp();
        }
    }
}

template <typename T, int BN, bool VEC>
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
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;      // warp: uniform
    const uint32_t rank = __shfl_sync(0xffffffffu, cluster_rank(), 0);
    const int c = (int)(blockIdx.x >> 1), ncl = (int)(gridDim.x >> 1);
    if (threadIdx.x == 32) {             // while the barriers are set up
        prefetch_tmap(&p.tm_x);
        prefetch_tmap(&p.tm_w);
    }
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
        lin_producer<BN>(p, smem, B, wait, rank, c, ncl);
    } else if (warp == 1) {
        if (rank == 0) lin_mma<T, BN>(p, smem, B, wait, tmem, c, ncl);
    } else if (warp >= 4) {
        lin_epilogue<T, BN, VEC>(p, smem, B, wait, tmem, rank, c, ncl, warp - 4, lane);
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

// A cut tile's pieces, added in the order of their chunks, then the epilogue;
// one thread per row and eight columns.
template <typename T>
__global__ void __launch_bounds__(256) linear_join_kernel(const __grid_constant__ LinParams p) {
    pdl_wait();
    pdl_open();
    const int groups = p.bn / 8, id = blockIdx.x * 256 + threadIdx.x;
    const int t = id / (256 * groups), in = id - t * (256 * groups);      // cut tile
    const int row = in / groups, col = (in - row * groups) * 8;
    const int first = t * p.k_chunks, last = first + p.k_chunks - 1;
    const int c0 = first / p.cut_each, c1 = last / p.cut_each;
    if (c0 == c1) return;                                     // one pair had the whole tile
    int mt, nt;
    tile_at(p, p.dp_tiles + t, mt, nt);
    const int tb = mt / p.m_tiles_per_batch;
    const RowAt at = row_at(p, tb, (int64_t)(mt - tb * p.m_tiles_per_batch) * 256 + row);
    const int n = nt * p.bn + col;
    if (!at.live || n >= p.n) return;
    float f[4][8] = {};                                       // one row of finish_rows' four
#pragma unroll 4
    for (int c = c0; c <= c1; ++c) {                          // (four pieces' reads in flight)
        const int slot = 2 * c + (first > c * p.cut_each ? 1 : 0);
        const float4* q = reinterpret_cast<const float4*>(p.part + ((int64_t)slot * 256 + row) * p.bn + col);
        const float4 a = q[0], b = q[1];
        f[0][0] += a.x; f[0][1] += a.y; f[0][2] += a.z; f[0][3] += a.w;
        f[0][4] += b.x; f[0][5] += b.y; f[0][6] += b.z; f[0][7] += b.w;
    }
    const T* res = static_cast<const T*>(p.residual) + at.r + n;
    T* y = static_cast<T*>(p.y) + at.y;
    if (p.vec) {
        const uint4 add = p.residual ? *reinterpret_cast<const uint4*>(res) : make_uint4(0, 0, 0, 0);
        finish_rows<true, 1>(p, f, n, &at);
        if (p.residual) add_residual<T>(f[0], add);
        const int h = n / p.n_head;
        *reinterpret_cast<uint4*>(y + h * p.ys_h + (n - h * p.n_head)) = pack8<T>(f[0]);
        return;
    }
    finish_rows<false, 1>(p, f, n, &at);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (n + e >= p.n) break;
        const int h = (n + e) / p.n_head;
        y[h * p.ys_h + (n + e - h * p.n_head)] =
            F16<T>::one(p.residual ? __fadd_rn(f[0][e], F16<T>::to(res[e])) : f[0][e]);
    }
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

struct FewParams {
    LinParams l;                 // the epilogue's part
    const uint16_t* x;
    const uint16_t* w;
    int64_t xs_b, xs_h, xs_s, w_stride;
    int k, k_head;
};

// Few rows (8 NT at most): y^T = w x^T, 16 rows of w per CTA.  A lane reads
// 16-byte runs of w rows (lane / 4) and (lane / 4 + 8), eight channels each, four
// lanes 64 consecutive bytes, kFewK / 32 runs in flight; x's rows are read with
// the same assignment of channels to fragment positions (any bijection gives
// the same sum over k).  Warp i takes every eighth run of kFewK channels, and
// the eight partial sums meet in shared memory, added in warp order.
// Bound: HBM, w's bytes.
constexpr int kFewK = 128;

template <typename T, int NT>
__global__ void __launch_bounds__(256) linear_few_kernel(const __grid_constant__ FewParams p) {
    pdl_wait();
    pdl_open();
    constexpr int kU = kFewK / 32;
    __shared__ float part[8][16][NT * 8 + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * 16;
    const int rows = (int)p.l.rows;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    const uint16_t* wrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) wrow[i] = p.w + (int64_t)(n0 + 8 * i + g) * p.w_stride;
    const uint16_t* xrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int r = 8 * j + g, b = r / (int)p.l.tokens;
        xrow[j] = p.x + b * p.xs_b + (r - b * (int)p.l.tokens) * p.xs_s;
    }
    float acc[NT][4] = {};
    // unsigned: k is below 2^31, and the step past its end must not wrap
    for (uint32_t k0 = warp * kFewK; k0 < (uint32_t)p.k; k0 += 8 * kFewK) {
        uint4 wv[kU][2], xv[kU][NT];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const uint32_t k = k0 + 32 * u + 8 * t;
            const bool in = k < (uint32_t)p.k;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                wv[u][i] = in && n0 + 8 * i + g < p.l.n ? __ldg(reinterpret_cast<const uint4*>(wrow[i] + k)) : zero;
            const uint32_t h = k / (uint32_t)p.k_head;
#pragma unroll
            for (int j = 0; j < NT; ++j)
                xv[u][j] = in && 8 * j + g < rows
                               ? __ldg(reinterpret_cast<const uint4*>(xrow[j] + h * p.xs_h + (k - h * p.k_head)))
                               : zero;
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const uint32_t a0[4] = {wv[u][0].x, wv[u][1].x, wv[u][0].y, wv[u][1].y};
            const uint32_t a1[4] = {wv[u][0].z, wv[u][1].z, wv[u][0].w, wv[u][1].w};
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                mma16816<T>(acc[j], a0, xv[u][j].x, xv[u][j].y);
                mma16816<T>(acc[j], a1, xv[u][j].z, xv[u][j].w);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) part[warp][g + 8 * (e >> 1)][8 * j + 2 * t + (e & 1)] = acc[j][e];
    __syncthreads();
    // one thread per output element; consecutive threads, consecutive columns of y
    for (int o = threadIdx.x; o < 16 * NT * 8; o += 256) {
        const int r = o / 16, c = o - r * 16, n = n0 + c;
        if (r >= rows || n >= p.l.n) continue;
        float f = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) f += part[q][c][r];
        const RowAt at = row_at(p.l, 0, r);
        const float bias = p.l.bias ? load1_any(p.l.bias, n, p.l.bias_dtype) : 0.0f;
        const float res = p.l.residual ? F16<T>::to(static_cast<const T*>(p.l.residual)[at.r + n]) : 0.0f;
        const int h = n / p.l.n_head;
        static_cast<T*>(p.l.y)[at.y + h * p.l.ys_h + (n - h * p.l.n_head)] =
            F16<T>::one(finish1<T>(p.l, f, bias, n, at, res));
    }
}

template <typename T, int NT> int launch_few(const FewParams& p, cudaStream_t st) {
    VCB_CUDA(launch_pdl(linear_few_kernel<T, NT>, dim3((unsigned)((p.l.n + 15) / 16)), dim3(256), 0, st, p));
    return VCB_OK;
}
template <typename T> int launch_few_any(const FewParams& p, cudaStream_t st) {
    return p.l.rows <= 8 ? launch_few<T, 1>(p, st) : launch_few<T, 2>(p, st);
}

template <typename T, int BN, bool VEC>
int launch_tiles_as(const LinParams& p, int grid_pairs, cudaStream_t st) {
    static bool ready[64] = {};
    using L = Tile<BN>;
    auto kernel = linear_kernel<T, BN, VEC>;
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
    cfg.numAttrs = 2;
    if (!ready[dev]) {
        VCB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem));
        ready[dev] = true;
    }
    cfg.gridDim = dim3((unsigned)(2 * grid_pairs));
    VCB_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
    if (p.cut_units) {
        const int tiles = p.cut_units / p.k_chunks;
        VCB_CUDA(launch_pdl(linear_join_kernel<T>, dim3((unsigned)tiles * (p.bn / 8)), dim3(256), 0, st, p));
    }
    return VCB_OK;
}

template <typename T, int BN> int launch_tiles(const LinParams& p, int grid_pairs, cudaStream_t st) {
    return p.vec ? launch_tiles_as<T, BN, true>(p, grid_pairs, st) : launch_tiles_as<T, BN, false>(p, grid_pairs, st);
}

// Up to this many rows of x the product streams w through linear_few_kernel.
constexpr int kFewRows = 16;

struct LinPlan {
    bool pack_x, pack_w;
    int64_t pitch;                        // elements of a packed row
    int64_t heads, k_head, w_stride;      // operands as the kernels read them
    int64_t xs_b, xs_h, xs_s;
    bool few, collapsed;
    int64_t rows, batches, m_tiles;
    int bn, chunks_per_head, k_chunks, grid_pairs;
    int64_t tiles, dp_tiles, cut_units, cut_each;
    size_t off_w, off_part, total;
};

LinPlan plan(const vcb_linear_args* a) {
    LinPlan q{};
    const int64_t k = a->heads_in * a->k_head;
    q.pitch = (k + 7) / 8 * 8;
    q.pack_w = !on16(a->w) || !tma_stride(a->w_stride, a->n);
    q.pack_x = !on16(a->x) || (a->heads_in > 1 && !by8(a->k_head)) || !tma_stride(a->x_stride_s, a->tokens) ||
               !tma_stride(a->x_stride_h, a->heads_in) || !tma_stride(a->x_stride_b, a->batch);
    q.heads = a->heads_in; q.k_head = a->k_head; q.w_stride = a->w_stride;
    q.xs_b = a->x_stride_b; q.xs_h = a->x_stride_h; q.xs_s = a->x_stride_s;
    if (q.pack_x) {                       // a packed row has its heads joined
        q.heads = 1; q.k_head = k;
        q.xs_s = q.pitch; q.xs_h = q.pitch; q.xs_b = a->tokens * q.pitch;
    }
    if (q.pack_w) q.w_stride = q.pitch;
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    q.off_w = q.pack_x ? up((size_t)(a->batch * a->tokens * q.pitch) * 2) : 0;
    q.off_part = q.total = q.off_w + (q.pack_w ? up((size_t)(a->n * q.pitch) * 2) : 0);
    // (16-byte runs of a row must not pass its end)
    q.few = a->batch * a->tokens <= kFewRows && (by8(k) || (q.pack_x && q.pack_w));
    if (q.few) return q;

    // one walk over batch x tokens where the rows are evenly spaced
    q.collapsed = q.heads == 1 && (a->batch == 1 || a->tokens == 1 || q.xs_b == a->tokens * q.xs_s);
    if (q.collapsed && a->tokens == 1 && a->batch > 1) q.xs_s = q.xs_b;
    q.rows = q.collapsed ? a->batch * a->tokens : a->tokens;
    q.batches = q.collapsed ? 1 : a->batch;
    // strides of axes of length one are never taken: any legal value will do
    const int64_t row = (q.k_head + 7) / 8 * 8;
    if (q.rows == 1) q.xs_s = row;
    if (q.heads == 1) q.xs_h = row;
    if (q.batches == 1) q.xs_b = row;
    if (a->n == 1) q.w_stride = row * q.heads;
    q.chunks_per_head = (int)((q.k_head + kBK - 1) / kBK);
    q.k_chunks = (int)(q.chunks_per_head * q.heads);
    q.m_tiles = (q.rows + 255) / 256 * q.batches;
    // Tile width, and whether the tiles of the last, partly filled round are
    // cut along K.  Cost in clocks, fitted to timelines of one pair: a 64-channel
    // chunk takes the longer of its products (2.2 a column) and its loads (100
    // bytes a clock); the last epilogue 25 a column; a cut writes its sums (28 a
    // column) and is joined by a second launch (24000).  It leaves out the launch,
    // the first loads and the clocks under load, so it ranks widths and is below
    // the time of a call: for K = N = 5120 at 1.9 GHz 11.0 us of 15.6 at 64 rows,
    // 17.8 of 23.2 at 512, 32.2 of 45.9 at 1024.  A width that fills the last round
    // is mostly better than a cut: 256 x 5120 x 5120 BF16 takes 24.6 us cut at 256
    // columns, 16.0 whole at 96.  Long sums over few tiles are cut (40 x 20000 x 96),
    // and a few tiles behind a full round (6273 x 12040 x 272).
    const int64_t pairs = sm_count() / 2;
    const int64_t tile_rows = q.rows < 128 ? q.rows : 128;
    double best = 0;
    for (int bn = 256; bn >= 32; bn -= 32) {
        const int64_t tiles = q.m_tiles * ((a->n + bn - 1) / bn), rem = tiles % pairs;
        const double mul = 2.2 * bn, ld = (128.0 * (double)tile_rows + 64.0 * bn) / 100;
        const double chunk = (mul > ld ? mul : ld) + 20, tile = chunk * q.k_chunks;
        const double whole = (double)((tiles + pairs - 1) / pairs) * tile + 25 * bn;
        int64_t each = (rem * q.k_chunks + pairs - 1) / pairs;
        if (each < 4) each = 4;
        const double cut = (double)(tiles / pairs) * tile + (double)each * chunk + 28 * bn + 24000;
        // (the kernels count a cut's chunks in 32 bits)
        const bool use_cut = rem && each < q.k_chunks && cut < whole && rem * q.k_chunks + each < (1ll << 31);
        const double cost = use_cut ? cut : whole;
        if (best > 0 && cost >= best) continue;
        best = cost;
        q.bn = bn;
        q.tiles = tiles;
        q.dp_tiles = use_cut ? tiles - rem : tiles;
        q.cut_units = use_cut ? rem * q.k_chunks : 0;
        q.cut_each = use_cut ? each : 1;
        const int64_t shares = use_cut ? (q.cut_units + each - 1) / each : 0;
        q.grid_pairs = (int)(q.dp_tiles >= pairs ? pairs : use_cut ? shares : tiles);
    }
    if (q.cut_units) q.total = q.off_part + (size_t)2 * pairs * 256 * q.bn * 4;
    return q;
}

}  // namespace

size_t linear_workspace_bytes(const vcb_linear_args* a) { return plan(a).total; }

int linear_run(const vcb_linear_args* a, cudaStream_t st) {
    const LinPlan q = plan(a);
    const int64_t k = a->heads_in * a->k_head;
    const void* x = a->x;
    const void* w = a->w;
    char* ws = static_cast<char*>(a->workspace);
    if (q.tiles >= (1ll << 30) || (q.tiles / 74 + 2) * q.k_chunks >= (1ll << 31))
        return fail(VCB_ERR_INVALID_ARGUMENT, "product too large for the projection kernel's tile counters");
    if (q.pack_x || q.pack_w) {
        PackParams pk{};
        pk.channels = (int)k;
        pk.pitch = (int)q.pitch;
        int64_t blocks = 0;
        if (q.pack_x) {
            const int64_t rows = a->batch * a->tokens;
            pk.side[0] = {static_cast<const uint16_t*>(x), reinterpret_cast<uint16_t*>(ws), rows, a->tokens,
                          a->x_stride_b, a->x_stride_s, 1, 0, a->x_stride_h, (int)a->k_head};
            blocks += (rows + 7) / 8;
            x = ws;
        }
        pk.end[0] = blocks;
        if (q.pack_w) {
            pk.side[1] = {static_cast<const uint16_t*>(w), reinterpret_cast<uint16_t*>(ws + q.off_w), a->n, a->n, 0,
                          a->w_stride, 1, 0, k, (int)k};
            blocks += (a->n + 7) / 8;
            w = ws + q.off_w;
        }
        pk.end[1] = pk.end[2] = blocks;
        VCB_CUDA(launch_pack(pk, st));
    }
    LinParams p;
    memset(&p, 0, sizeof(p));
    const bool bf16 = a->dtype == VCB_BF16;
    p.tokens = a->tokens;
    p.n = (int)a->n;
    p.n_head = (int)a->n_head;
    p.activation = a->activation;
    p.bias = a->bias; p.bias_dtype = a->bias_dtype;
    p.gate = a->gate; p.gate_dtype = a->gate_dtype; p.gs_b = a->gate_stride_b; p.gs_s = a->gate_stride_s;
    p.residual = a->residual; p.rs_b = a->residual_stride_b; p.rs_s = a->residual_stride_s;
    p.y = a->y; p.ys_b = a->y_stride_b; p.ys_h = a->y_stride_h; p.ys_s = a->y_stride_s;
    p.vec = on16(a->y) && by8(a->n_head) && by8(a->y_stride_b) && by8(a->y_stride_h) && by8(a->y_stride_s) &&
            (!a->bias || on16(a->bias)) &&
            (!a->gate || (on16(a->gate) && by8(a->gate_stride_b) && by8(a->gate_stride_s))) &&
            (!a->residual || (on16(a->residual) && by8(a->residual_stride_b) && by8(a->residual_stride_s)));
    p.status = a->status;
    if (q.few) {
        FewParams f;
        f.l = p;
        f.l.rows = a->batch * a->tokens;
        f.l.collapsed = 1;
        f.x = static_cast<const uint16_t*>(x);
        f.w = static_cast<const uint16_t*>(w);
        f.xs_b = q.xs_b; f.xs_h = q.xs_h; f.xs_s = q.xs_s; f.w_stride = q.w_stride;
        f.k = (int)(by8(k) ? k : q.pitch);
        f.k_head = (int)(q.heads > 1 ? q.k_head : f.k);
        return bf16 ? launch_few_any<__nv_bfloat16>(f, st) : launch_few_any<__half>(f, st);
    }
    {
        const cuuint64_t dims[4] = {(cuuint64_t)q.k_head, (cuuint64_t)q.rows, (cuuint64_t)q.heads, (cuuint64_t)q.batches};
        const cuuint64_t strides[3] = {(cuuint64_t)q.xs_s * 2, (cuuint64_t)q.xs_h * 2, (cuuint64_t)q.xs_b * 2};
        const cuuint32_t box[4] = {kBK, 128, 1, 1};
        int rc = make_map16(&p.tm_x, x, bf16, 4, dims, strides, box);
        if (rc) return rc;
    }
    {
        const cuuint64_t dims[3] = {(cuuint64_t)q.k_head, (cuuint64_t)q.heads, (cuuint64_t)a->n};
        const cuuint64_t head_stride = (cuuint64_t)((q.k_head + 7) / 8 * 8) * 2;
        const cuuint64_t strides[2] = {head_stride, (cuuint64_t)q.w_stride * 2};
        const cuuint32_t box[3] = {kBK, 1, (cuuint32_t)(q.bn / 2)};
        int rc = make_map16(&p.tm_w, w, bf16, 3, dims, strides, box);
        if (rc) return rc;
    }
    p.bn = q.bn;
    p.chunks_per_head = q.chunks_per_head;
    p.k_chunks = q.k_chunks;
    p.m_tiles = (int)q.m_tiles;
    p.n_tiles = (int)((a->n + q.bn - 1) / q.bn);
    p.m_tiles_per_batch = (int)((q.rows + 255) / 256);
    p.rows = q.rows;
    p.collapsed = q.collapsed;
    p.dp_tiles = (int)q.dp_tiles;
    p.cut_units = (int)q.cut_units;
    p.cut_each = (int)q.cut_each;
    p.part = reinterpret_cast<float*>(ws + q.off_part);
    if (q.bn > 128)
        return bf16 ? launch_tiles<__nv_bfloat16, 256>(p, q.grid_pairs, st) : launch_tiles<__half, 256>(p, q.grid_pairs, st);
    return bf16 ? launch_tiles<__nv_bfloat16, 128>(p, q.grid_pairs, st) : launch_tiles<__half, 128>(p, q.grid_pairs, st);
}

}  // namespace vcb
