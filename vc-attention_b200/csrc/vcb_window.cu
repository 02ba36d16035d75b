// 16-bit attention over a sliding window with first tokens that stay visible.
// Query i stands at position p = i + offset and sees key j of the first `len`
// keys when
//   (j < sinks or p - left <= j <= p + right) and (not causal or j <= p);
// out = softmax over the seen keys of (scale q . k), times v; 0 for a row that
// sees none.  The seen keys are two runs, [0, sink) and [lo, hi), so a CTA
// walks the 128-key tiles of two runs and skips all others.
//
// Bound: the tensor cores (4 D operations a pair) and the exponentials (16 a
// clock and SM: as long as the two products of a 128-wide head), for few
// queries the bytes of K and V.
//
// Work decomposition.  A CTA owns NQ (1 or 2) tiles of 128 queries of one
// head; items that would not fill the last round of CTAs are cut along their
// keys, and window_join_kernel joins the parts in a fixed order.  Per key tile and query
// tile: S = Q K^T into tensor memory (tcgen05, 128 x 128), the query tile's
// eight softmax warps (two lanes per row, 64 keys each) turn S into P = 2^(s - m)
// in 16 bits over S's own columns, and O += P V adds onto the row's sums in
// tensor memory.  V stays [key][channel] as it comes: it is the N-major B
// operand.  With two query tiles one tile's products run under the other's
// softmax; the issue order PV_0(j), QK_0(j+1), PV_1(j), QK_1(j+1) makes S_w(j+1)
// follow P_w(j) in the same columns without a further wait.
//
// P = 2^(s - m).  The reference m moves only when a row's maximum passes it by
// more than 2^8: until then P just grows, and O is not rescaled.  A softmax warp
// rescales O itself, between the commit that follows PV_w(j-1) and its own
// arrival for PV_w(j).
//
// P has fewer bits than S: it is the A operand of a 16-bit product.  The row sum
// adds it in FP32, before its rounding, so an output is off by the roundings of P:
// half a step each, (eps / 2) sum_j w_j |v_j|.  (Summing the rounded P costs one
// instruction per score and 5 % of the time: the kernel runs at the power limit,
// where every instruction counts.)  BF16 has FP32's exponents.  FP16 ends at 2^-24,
// so there m lies 2^7 below the maximum and P reaches 2^15 (the largest FP16 is
// 65504): weights below 2^-21 of the maximum are off by up to 2^-32 of it, and
// only those below 2^-32 are lost to the product (2^-25 with m at the maximum,
// where 60000 keys at 2^-26 lost their whole share).  The sums carry the same
// factor, so it cancels.
//
// Measured, 1 B200: 40 heads of 32768 tokens, window 4096 + 4096, 1024 first
// tokens, BF16: 5.10-5.19 ms back to back, 1108-1126 TFLOP/s at the 1000 W limit
// and 1.56-1.60 GHz.  Tried without gain: the keys'
// tiles on CTA pairs with two S and two P buffers (5.72 ms), one thread per row
// (5.96), no maximum but a check of the sums (5.26, no gain
// for a second path), part of the exponentials as polynomials (5.15-5.17 against 5.19).
//
// A masked key has P = 0, but 0 times a NaN or infinity in its V row would
// still reach O.  Rows behind a batch entry's last key are therefore cleared in
// shared memory, and a row whose sums are not finite is computed again by
// window_row, which reads only the keys that the row sees.  Finite values near
// the end of BF16's range take that way too: P V sums them before the division.
//
// Roles (128 + 256 NQ threads): warp 0 TMA producer, warp 1 MMA issuer, warp 2
// clears V rows behind the last key, warp 3 tensor memory; then eight softmax
// warps (two warpgroups) per query tile, which also write the output.  Every
// mbarrier wait is bounded; a CTA that gives up drains and frees its tensor memory.
#include "vcb_f16.cuh"

namespace vcb {
namespace {

struct WinParams {
    CUtensorMap tm_q, tm_k, tm_v;            // [batch][head][token][channel]
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
    float c;                                 // scale log2(e)
    int q_tiles, vec_out;
    int whole, splits;                       // items of one CTA; parts of each item behind them
    int64_t part_rows;                       // rows of those items
    float* part;                             // [splits][part_rows][HD] sums
    float2* part_ml;                         // [splits][part_rows] maximum (log2) and row sum
    int32_t* status;
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

// One output row by one warp, reading only the keys that the row sees: lane l
// takes every 32nd key's logit, then channels l, l + 32, ... of the mean of V so
// far: a mean of finite values is finite where their sum may not be.  0 for a row
// that sees no key; a row whose logits are all -inf is 0 / 0, a NaN.
// `qrow` is 128 floats of shared memory of this warp.
template <typename T>
__device__ void window_row(const WinParams& p, int64_t b, int64_t h, int64_t i, float* qrow, int lane) {
    const int64_t len = keys_of(p, b);
    const Seen s = seen_at(p, i + (p.has_offset ? p.q_offset : len - p.sq), len);
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[1] + i * p.qs[2];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + h * p.ks[1];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + h * p.vs[1];
    __syncwarp();
    for (int c = lane; c < 128; c += 32) qrow[c] = c < p.d ? F16<T>::to(q[c]) : 0.0f;
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
                for (int c = 0; c < p.d; ++c) dot = __fmaf_rn(qrow[c], F16<T>::to(row[c]), dot);
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
            const float total = __fmaf_rn(den, alpha, sum);
            // (a correctly rounded reciprocal here spilled two registers of the softmax warps,
            // as did an early end at a row of NaNs: 6 % of the whole kernel's time.  One Newton
            // step takes the approximate one to about half a step)
            float inv = total == 0.0f ? 0.0f : __fdividef(1.0f, total);
            inv = __fmaf_rn(__fmaf_rn(-total, inv, 1.0f), inv, inv);
            const float keep = __fmul_rn(__fmul_rn(den, alpha), inv), share = __fmul_rn(w, inv);
            float some[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int j = 0; j < n; ++j) {
                const float wj = __shfl_sync(0xffffffffu, share, j);
                const T* row = v + (int64_t)(base + j) * p.vs[2];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (lane + 32 * e < p.d) some[e] = __fmaf_rn(wj, F16<T>::to(row[lane + 32 * e]), some[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] = __fmaf_rn(acc[e], keep, some[e]);
            den = total;
            m = m_new;
        }
    }
    const bool sees = s.sink > 0 || s.hi > s.lo;
    const float one = __fdiv_rn(den, den);                        // NaN where no logit was above -inf
    T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + i * p.os[2];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (lane + 32 * e < p.d) out[lane + 32 * e] = F16<T>::one(sees ? __fmul_rn(acc[e], one) : 0.0f);
}

constexpr int kKT = 128;                           // keys per tile

template <int HD, int NQ> struct WinTile {
    static constexpr int kBoxes = HD / 64;                       // 64-channel (128-byte) boxes of a row
    static constexpr uint32_t kBox = 128 * 128;                  // 128 rows of a box
    static constexpr uint32_t kBytes = kBoxes * kBox;            // one Q, K or V tile
    static constexpr int kStages = NQ == 2 ? (HD == 128 ? 5 : 8) : (HD == 128 ? 2 : 5);
    static constexpr uint32_t kOffKV = NQ * kBytes;
    static constexpr uint32_t kOffBars = kOffKV + kStages * kBytes;
    static constexpr int kNumBars = 1 + 2 * kStages + 4 * 2 + 1 + 1;
    static constexpr uint32_t kOffMisc = kOffBars + kNumBars * 8;
    static constexpr uint32_t kSmem = kOffMisc + 16;
    static constexpr int kThreads = 128 + 256 * NQ;
    static constexpr int kCtas = NQ == 2 ? 1 : 2;                // per SM
    // tensor memory: S (P over it) and O of each query tile
    static constexpr uint32_t kCols = NQ == 2 ? 512 : 256;
    static constexpr uint32_t kColO = NQ * 128;
    // setmaxnreg shares: control warps, softmax warps (64 / 104 with two query
    // tiles: 5.23 ms against 5.15).  With one tile, two CTAs per SM leave 80 a thread
    // at launch: 20 bytes spill, 368 with 64 / 88.
    static constexpr int kRegsCtl = 32, kRegsSoft = NQ == 2 ? 112 : 104;
    static constexpr int kRegSplit = 128 * kRegsCtl + 256 * NQ * kRegsSoft;
    static_assert(kSmem <= 232448 / kCtas - (kCtas - 1) * 1024, "shared memory of one CTA");
};

struct WinBars {
    uint64_t* q_full;
    uint64_t* kv_full;    // [stages]
    uint64_t* kv_empty;   // [stages]  the stage's products are done
    uint64_t* s_full;     // [2]  S_w(j) is there, and PV_w(j-1) done
    uint64_t* p_half;     // [2]  P_w(j) of the keys 0-31 and 64-95 is there, O_w rescaled
    uint64_t* p_full;     // [2]  all of P_w(j)
    uint64_t* o_full;     // [2]  the last PV_w is done
    uint64_t* v_last;     // [1]  the V tile that holds the last key landed; warp 2 clears the rows behind it
                          //      and arrives on that stage's kv_full itself
    uint64_t* drain;      // [1]
};
template <typename L> __device__ __forceinline__ WinBars win_bars(uint8_t* smem) {
    uint64_t* b = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
    WinBars r;
    r.q_full = b; b += 1;
    r.kv_full = b; b += L::kStages;
    r.kv_empty = b; b += L::kStages;
    r.s_full = b; b += 2;
    r.p_half = b; b += 2;
    r.p_full = b; b += 2;
    r.o_full = b; b += 2;
    r.v_last = b; b += 1;
    r.drain = b;
    return r;
}

// What a CTA works on: queries [row0, row0 + 128 nq) of head (b, h) and the
// key tiles begin .. begin + count - 1 of its list, tiles 0 .. n1 - 1 and then
// from w0 on.
struct WinItem {
    int64_t b, h, row0, len, offset;
    int64_t part_at;             // first row among the parts' rows, -1 for a whole item
    int nq, n1, w0, begin, count;
    __device__ __forceinline__ int tile(int j) const {
        const int i = begin + j;
        return i < n1 ? i : w0 + i - n1;
    }
};
template <int NQ> __device__ __forceinline__ WinItem win_item(const WinParams& p) {
    WinItem it;
    int r = blockIdx.x, split = 0, splits = 1;
    it.part_at = -1;
    if (r >= p.whole && p.splits > 1) {
        const int o = r - p.whole;
        splits = p.splits;
        split = o % splits;
        it.part_at = split * p.part_rows + (int64_t)(o / splits) * (128 * NQ);
        r = p.whole + o / splits;
    }
    const int qt = p.q_tiles - 1 - r % p.q_tiles;               // late (longer) causal tiles first
    const int64_t bh = r / p.q_tiles;
    it.b = bh / p.heads;
    it.h = bh - it.b * p.heads;
    it.row0 = (int64_t)qt * (128 * NQ);
    it.nq = NQ == 2 && it.row0 + 128 < p.sq ? 2 : 1;
    it.len = keys_of(p, it.b);
    it.offset = p.has_offset ? p.q_offset : it.len - p.sq;
    const int64_t last = min(it.row0 + 128 * NQ, p.sq) - 1;
    const Seen a = seen_at(p, it.row0 + it.offset, it.len), z = seen_at(p, last + it.offset, it.len);
    // sink, lo and hi grow with the position
    it.n1 = (z.sink + kKT - 1) / kKT;
    it.w0 = max(it.n1, a.lo / kKT);
    const int w1 = z.hi > a.lo ? (z.hi + kKT - 1) / kKT : 0;
    const int total = it.n1 + max(0, w1 - it.w0);
    it.begin = (int)((int64_t)total * split / splits);
    it.count = (int)((int64_t)total * (split + 1) / splits) - it.begin;
    return it;
}

// The whole warp runs the load loop and one elected lane issues, as for the MMAs.
__device__ __forceinline__ void expect_elected(uint32_t bar, uint32_t bytes) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}"
        ::"r"(bar), "r"(bytes)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z, int w) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5, %6}], [%2];\n\t}"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
// D[128 x N] (+)= A B, A and B in shared memory.  The whole warp runs the issue
// loop and one elected lane issues: its operands then stay in uniform registers.
// (A lone thread's operands were moved there one by one before every MMA, and
// next to the busy softmax warps of its scheduler an MMA of 64 clocks took 80
// to 100 to issue.)  Descriptors differ in the low word only.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "mov.b64 da, {%1, %3};\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// the same with A in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 16 lanes x (N columns, and N columns SPLIT behind): thread t < 16 of the warp
// has lane base + t and the first run, thread t + 16 the same lane and the second
template <int SPLIT> __device__ __forceinline__ void tmem_ld16x2_32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x32bx2.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32], %33;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr), "n"(SPLIT));
}
template <int SPLIT> __device__ __forceinline__ void tmem_st16x2_32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x32bx2.x32.b32 [%0], %33, {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
          "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
          "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "n"(SPLIT)
        : "memory");
}
template <int SPLIT, int OFF, int N> __device__ __forceinline__ void tmem_st16x2_16(uint32_t taddr, const uint32_t (&r)[N]) {
    static_assert(OFF + 16 <= N, "range");
    asm volatile(
        "tcgen05.st.sync.aligned.16x32bx2.x16.b32 [%0], %17, {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
        "%13, %14, %15, %16};"
        ::"r"(taddr), "r"(r[OFF + 0]), "r"(r[OFF + 1]), "r"(r[OFF + 2]), "r"(r[OFF + 3]), "r"(r[OFF + 4]),
          "r"(r[OFF + 5]), "r"(r[OFF + 6]), "r"(r[OFF + 7]), "r"(r[OFF + 8]), "r"(r[OFF + 9]), "r"(r[OFF + 10]),
          "r"(r[OFF + 11]), "r"(r[OFF + 12]), "r"(r[OFF + 13]), "r"(r[OFF + 14]), "r"(r[OFF + 15]), "n"(SPLIT)
        : "memory");
}

// commit of the elected lane's MMAs (the same lane every time)
__device__ __forceinline__ void mma_commit_elected(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(smem_u32(bar))
        : "memory");
}

template <typename L>
__device__ void win_producer(const WinParams& p, const WinItem& it, int fix, uint8_t* smem, const WinBars& B, volatile int* abort) {
    prefetch_tmap(&p.tm_q);
    prefetch_tmap(&p.tm_k);
    prefetch_tmap(&p.tm_v);
    const uint32_t base = smem_u32(smem), q_bar = smem_u32(B.q_full), full0 = smem_u32(B.kv_full), last = smem_u32(B.v_last);
    const int h = (int)it.h, b = (int)it.b;
    expect_elected(q_bar, it.nq * L::kBytes);
    for (int w = 0; w < it.nq; ++w)
        for (int x = 0; x < L::kBoxes; ++x)
            tma_load_4d(base + w * L::kBytes + x * L::kBox, &p.tm_q, q_bar, 64 * x, (int)it.row0 + 128 * w, h, b);
    int issued = 0;
    for (int g = 0; g < 2 * it.count; ++g) {                     // K_0, V_0, K_1, V_1, ...
        const int s = g % L::kStages;
        if (g >= L::kStages && !mbar_wait(&B.kv_empty[s], ((g / L::kStages) - 1) & 1, abort)) break;
        const int key = it.tile(g >> 1) * kKT;
        const uint32_t bar = g == 2 * fix + 1 ? last : full0 + 8 * s, st = base + L::kOffKV + s * L::kBytes;
        expect_elected(bar, L::kBytes);
#pragma unroll
        for (int x = 0; x < L::kBoxes; ++x)
            tma_load_4d(st + x * L::kBox, g & 1 ? &p.tm_v : &p.tm_k, bar, 64 * x, key, h, b);
        issued = g + 1;
    }
    if (*abort) {                                                // no copy may land after the CTA exits
        drain_wait(B.q_full, 0);
        if (fix >= 0 && issued > 2 * fix + 1) drain_wait(B.v_last, 0);
        for (int s = 0; s < L::kStages && s < issued; ++s)
            drain_wait(&B.kv_full[s], ((issued - 1 - s) / L::kStages) & 1);
    }
}

template <typename T, int HD, int NQ>
__device__ void win_mma(const WinItem& it, uint8_t* smem, const WinBars& B, uint32_t tmem0, volatile int* abort) {
    const uint32_t tmem = __shfl_sync(0xffffffffu, tmem0, 0);      // uniform
    using L = WinTile<HD, NQ>;
    constexpr uint32_t idesc_qk = idesc_f16<T>(128, kKT), idesc_pv = idesc_f16<T>(128, HD, true);
    const uint64_t k64 = smem_desc_k128(smem + L::kOffKV);
    const uint32_t hi = (uint32_t)(k64 >> 32), q0 = (uint32_t)smem_desc_k128(smem), k0 = (uint32_t)k64;
    // V tile as the N-major operand: 64-channel blocks a box apart (leading
    // offset, bits [16, 30)), groups of 8 keys 1024 bytes apart (stride offset)
    const uint32_t v0 = (k0 & 0xffffu) | ((L::kBox >> 4) << 16);
    auto qk = [&](int w, int s) {
        const uint32_t q = q0 + w * (L::kBytes >> 4), k = k0 + s * (L::kBytes >> 4);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            const uint32_t step = (kk / 4) * (L::kBox >> 4) + 2 * (kk % 4);
            mma_ss(tmem + 128 * w, q + step, k + step, hi, idesc_qk, kk > 0);
        }
    };
    auto pv = [&](int w, int s, int kk, bool accumulate) {
        mma_ts(tmem + L::kColO + 128 * w, tmem + 128 * w + 8 * kk, v0 + s * (L::kBytes >> 4) + 128 * kk, hi, idesc_pv,
               accumulate);
    };
    bool ok = mbar_wait(B.q_full, 0, abort) && mbar_wait(&B.kv_full[0], 0, abort);
    if (ok) {
        tc_fence_after();
        for (int w = 0; w < it.nq; ++w) {
            qk(w, 0);
            mma_commit_elected(&B.s_full[w]);
        }
        mma_commit_elected(&B.kv_empty[0]);
    }
    for (int j = 0; ok && j < it.count; ++j) {
        const int gv = 2 * j + 1, gk = 2 * j + 2;
        const int sv = gv % L::kStages, sk = gk % L::kStages;
        const bool more = j + 1 < it.count;
        ok = mbar_wait(&B.kv_full[sv], (gv / L::kStages) & 1, abort);
        for (int w = 0; ok && w < it.nq; ++w) {
            if (!mbar_wait(&B.p_half[w], j & 1, abort)) { ok = false; break; }
            tc_fence_after();
            pv(w, sv, 0, j > 0); pv(w, sv, 1, true); pv(w, sv, 4, true); pv(w, sv, 5, true);
            if (!mbar_wait(&B.p_full[w], j & 1, abort)) { ok = false; break; }
            tc_fence_after();
            pv(w, sv, 2, true); pv(w, sv, 3, true); pv(w, sv, 6, true); pv(w, sv, 7, true);
            if (w == it.nq - 1) mma_commit_elected(&B.kv_empty[sv]);
            if (more) {
                if (w == 0 && !mbar_wait(&B.kv_full[sk], (gk / L::kStages) & 1, abort)) { ok = false; break; }
                tc_fence_after();
                qk(w, sk);
                mma_commit_elected(&B.s_full[w]);
                if (w == it.nq - 1) mma_commit_elected(&B.kv_empty[sk]);
            } else {
                mma_commit_elected(&B.o_full[w]);
            }
        }
    }
    mma_commit_elected(B.drain);
    drain_wait(B.drain, 0);
}

// The lowest x bits (none for x <= 0, all for x >= 32).
__device__ __forceinline__ uint32_t bits_below(int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; }

// Warp (quarter, sub) of query tile w owns rows 32 quarter + 16 sub + [0, 16);
// lanes t and t + 16 share a row, keys [0, 64) and [64, 128) of each tile.
template <typename T, int HD, int NQ>
__device__ void win_softmax(const WinParams& p, const WinItem& it, uint8_t* smem, const WinBars& B, uint32_t tmem, int w,
                            int quarter, int sub, int lane, volatile int* abort) {
    using L = WinTile<HD, NQ>;
    const int half = lane >> 4;
    const int64_t tile_row = it.row0 + 128 * w;
    const int64_t row0 = tile_row + quarter * 32 + sub * 16, row = row0 + (lane & 15);
    const bool valid = row < p.sq;
    const bool warp_live = row0 < p.sq;
    const int64_t last = min(tile_row + 128, p.sq) - 1;
    const Seen none{0, 0, 0};
    const Seen mine = valid ? seen_at(p, row + it.offset, it.len) : none;
    const bool sees = mine.sink > 0 || mine.hi > mine.lo;
    // tiles that all rows of the query tile see whole: keys up to sink_all, and
    // from lo_all up to hi_all
    int sink_all, lo_all, hi_all;
    {
        const Seen first = seen_at(p, tile_row + it.offset, it.len), end = seen_at(p, last + it.offset, it.len);
        sink_all = first.sink;
        hi_all = first.hi;
        lo_all = end.lo <= first.sink ? 0 : end.lo;
    }
    const uint32_t trow = tmem + ((uint32_t)(quarter * 32 + sub * 16) << 16);
    const uint32_t ts = trow + 128 * w, to = trow + L::kColO + 128 * w;
    const float c = p.c;
    constexpr float kUp = F16<T>::kDtype == VCB_F16 ? 7.0f : 0.0f;      // log2 of P at the row's maximum
    float m = -INFINITY, den = 0.0f;
    for (int j = 0; j < it.count; ++j) {
        if (!mbar_wait(&B.s_full[w], j & 1, abort)) return;
        tc_fence_after();
        if (!warp_live) {
            tc_fence_before();
            __syncwarp();
            mbar_arrive_if(&B.p_half[w], lane == 0);
            mbar_arrive_if(&B.p_full[w], lane == 0);
            continue;
        }
        uint32_t r[64];
        tmem_ld16x2_at<0>(ts, r);                                // keys 0-31 | 64-95
        tmem_ld16x2_at<32>(ts + 32, r);                          // keys 32-63 | 96-127
        tmem_wait_ld();
        const int k0 = it.tile(j) * kKT, k1 = k0 + kKT;
        if (!(k1 <= sink_all || (k1 <= hi_all && k0 >= lo_all))) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int o = k0 + 64 * half + 32 * q;
                const uint32_t seen = bits_below(mine.sink - o) | (bits_below(mine.hi - o) & ~bits_below(mine.lo - o));
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (!(seen & (1u << e))) r[32 * q + e] = 0xff800000u;
            }
        }
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
#pragma unroll
        for (int t = 1; t < 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                mx[e] = fmax3(mx[e], __uint_as_float(r[8 * t + 2 * e]), __uint_as_float(r[8 * t + 2 * e + 1]));
        float top = fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
        top = __fmul_rn(fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16)), c);
        const float m_new = top > m + (8.0f + kUp) ? top - kUp : m;
        const float alpha = m_new == m ? 1.0f : ex2_ftz(m - m_new);
        const bool moved = __any_sync(0xffffffffu, m_new != m);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float2 cc = make_float2(c, c), rr = make_float2(-ref, -ref);
        if (moved && j > 0) {                                    // PV_w(j-1) is done: s_full follows it
#pragma unroll 1
            for (int q = 0; q < HD / 64; ++q) {
                uint32_t o[32];
                tmem_ld16x2_32<HD / 2>(to + 32 * q, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__fmul_rn(__uint_as_float(o[e]), alpha));
                tmem_st16x2_32<HD / 2>(to + 32 * q, o);
            }
        }
        float2 sum[2] = {};
        uint32_t pk[32];
        auto weights = [&](int e) {
            float2 x = ffma2(make_float2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1])), cc, rr);
            x = make_float2(ex2_ftz(x.x), ex2_ftz(x.y));
            sum[e & 1] = fadd2(sum[e & 1], x);
            pk[e] = F16<T>::two(x.x, x.y);
        };
#pragma unroll
        for (int e = 0; e < 16; ++e) weights(e);
        tmem_st16x2_16<32, 0>(ts, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(&B.p_half[w], lane == 0);
#pragma unroll
        for (int e = 16; e < 32; ++e) weights(e);
        tmem_st16x2_16<32, 16>(ts + 16, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        mbar_arrive_if(&B.p_full[w], lane == 0);
        sum[0] = fadd2(sum[0], sum[1]);
        den = __fmaf_rn(den, alpha, __fadd_rn(sum[0].x, sum[0].y));
        m = m_new;
    }
    if (!warp_live) return;
    den += __shfl_xor_sync(0xffffffffu, den, 16);
    if (it.count > 0) {
        if (!mbar_wait(&B.o_full[w], 0, abort)) return;
        tc_fence_after();
    }
    const int ch0 = half * (HD / 2);                             // this lane's channels: ch0 + 32 q + [0, 32)
    if (it.part_at >= 0) {
        const int64_t at = it.part_at + (row - it.row0);
        if (it.count > 0) {
            float4* dst = reinterpret_cast<float4*>(p.part + at * HD + ch0);
#pragma unroll 1
            for (int q = 0; q < HD / 64; ++q) {
                uint32_t o[32];
                tmem_ld16x2_32<HD / 2>(to + 32 * q, o);
                tmem_wait_ld();
                if (valid) {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        dst[8 * q + e] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                                     __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
                }
            }
        }
        if (valid && half == 0) p.part_ml[at] = make_float2(m, den);
        return;
    }
    // out = O / den; a row that sees nothing is 0
    const float inv = sees ? __frcp_rn(den) : 0.0f;
    T* out = static_cast<T*>(p.out) + it.b * p.os[0] + it.h * p.os[1] + row * p.os[2];
    bool bad = false;
#pragma unroll 1
    for (int q = 0; q < HD / 64; ++q) {
        uint32_t o[32];
        if (it.count > 0) {
            tmem_ld16x2_32<HD / 2>(to + 32 * q, o);
            tmem_wait_ld();
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
            const float f = sees ? __fmul_rn(__uint_as_float(o[e]), inv) : 0.0f;
            bad |= !finite_f(f);
            o[e] = __float_as_uint(f);
        }
        const int ch = ch0 + 32 * q;
        if (valid) {
            if (p.vec_out) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (ch + 8 * e < p.d) {
                        auto two = [&](int i) {
                            return F16<T>::two(__uint_as_float(o[8 * e + i]), __uint_as_float(o[8 * e + i + 1]));
                        };
                        *reinterpret_cast<uint4*>(out + ch + 8 * e) = make_uint4(two(0), two(2), two(4), two(6));
                    }
            } else {
#pragma unroll
                for (int e = 0; e < 32; ++e)
                    if (ch + e < p.d) out[ch + e] = F16<T>::one(__uint_as_float(o[e]));
            }
        }
    }
    // rows with a NaN or infinity among the tiles' keys (or no finite logit)
    unsigned again = __ballot_sync(0xffffffffu, valid && sees && bad);
    again = (again | (again >> 16)) & 0xffffu;
    if (again) {
        float* qrow = reinterpret_cast<float*>(smem + w * L::kBytes) + 128 * (2 * quarter + sub);   // Q_w is no longer read
        for (; again; again &= again - 1) window_row<T>(p, it.b, it.h, row0 + __ffs(again) - 1, qrow, lane);
    }
}

template <typename T, int HD, int NQ>
__global__ void __launch_bounds__(WinTile<HD, NQ>::kThreads, WinTile<HD, NQ>::kCtas)
    window_kernel(const __grid_constant__ WinParams p) {
    pdl_wait();
    using L = WinTile<HD, NQ>;
    extern __shared__ __align__(1024) uint8_t smem[];
    if (smem_u32(smem) & 1023u) {
        if (threadIdx.x == 0) flag_status(p.status, VCB_FLAG_INTERNAL);
        return;
    }
    const WinBars B = win_bars<L>(smem);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffMisc);
    volatile int* abort = reinterpret_cast<volatile int*>(smem + L::kOffMisc + 4);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;      // warp: uniform
    const WinItem it = win_item<NQ>(p);
    if (threadIdx.x == 0) {
        mbar_init(B.q_full, 1);
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&B.kv_full[s], 1);
            mbar_init(&B.kv_empty[s], 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(&B.s_full[w], 1);
            mbar_init(&B.p_half[w], 8);
            mbar_init(&B.p_full[w], 8);
            mbar_init(&B.o_full[w], 1);
        }
        mbar_init(B.v_last, 1);
        mbar_init(B.drain, 1);
        *abort = 0;
        fence_barrier_init();
    }
    if (warp == 3) {
        tmem_alloc(tmem_slot, L::kCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // the place in this CTA's list of the tile that holds keys on both sides
    // of the entry's length, when the tensor has rows there
    int fix = -1;
    if (it.len < p.sk && it.len % kKT && it.count > 0) {
        const int t = (int)(it.len / kKT);
        if (it.tile(it.count - 1) == t) fix = it.count - 1;
    }
    if (warp < 4) {
        reg_dealloc<L::kRegsCtl>();
        if (it.count > 0) {
            if (warp == 0) win_producer<L>(p, it, fix, smem, B, abort);
            if (warp == 1) win_mma<T, HD, NQ>(it, smem, B, tmem, abort);
            if (warp == 2 && fix >= 0) {
                const int s = (2 * fix + 1) % L::kStages;
                if (mbar_wait(B.v_last, 0, abort)) {
                    // whole 128-byte lines: the swizzle moves bytes within a line only
                    const int first = (int)(it.len % kKT);
                    for (int x = 0; x < L::kBoxes; ++x) {
                        uint4* box = reinterpret_cast<uint4*>(smem + L::kOffKV + s * L::kBytes + x * L::kBox);
                        for (int i = first * 8 + lane; i < kKT * 8; i += 32) box[i] = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    mbar_arrive_if(&B.kv_full[s], lane == 0);
                }
            }
        }
    } else {
        reg_alloc<L::kRegsSoft>();
        const int w = (warp - 4) >> 3;
        if (w < it.nq) win_softmax<T, HD, NQ>(p, it, smem, B, tmem, w, warp & 3, ((warp - 4) >> 2) & 1, lane, abort);
    }
    tc_fence_before();
    __syncwarp();
    __syncthreads();
    if (warp == 3) {
        tc_fence_after();
        tmem_dealloc(tmem, L::kCols);
    }
    if (threadIdx.x == 0 && *abort) flag_status(p.status, VCB_FLAG_TIMEOUT);
}

// One warp per row: out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) den_s over
// the parts in order.
template <typename T, int HD, int NQ>
__global__ void __launch_bounds__(256) window_join_kernel(const __grid_constant__ WinParams p) {
    pdl_wait();
    pdl_open();
    __shared__ float qrow[8][128];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a row of the items behind the whole ones; with one query tile per head an
    // item has sq rows only
    const int per = p.q_tiles == 1 ? (int)p.sq : 128 * NQ;
    const int64_t n = (int64_t)blockIdx.x * 8 + warp;
    const int cut = (int)(n / per), in = (int)(n - (int64_t)cut * per), item = p.whole + cut;
    if ((int64_t)cut * (128 * NQ) >= p.part_rows) return;
    const int64_t bh = item / p.q_tiles, b = bh / p.heads, h = bh - b * p.heads;
    const int64_t i = (int64_t)(p.q_tiles - 1 - item % p.q_tiles) * (128 * NQ) + in;
    if (i >= p.sq) return;
    const int64_t rows = p.part_rows, r = (int64_t)cut * (128 * NQ) + in;
    const int64_t len = keys_of(p, b);
    const Seen s = seen_at(p, i + (p.has_offset ? p.q_offset : len - p.sq), len);
    const bool sees = s.sink > 0 || s.hi > s.lo;
    constexpr int kPer = HD / 32;                                // channels per lane
    // lane q holds part q's maximum and weight (32 parts at most)
    const float2 ml = lane < p.splits ? p.part_ml[lane * rows + r] : make_float2(-INFINITY, 0.0f);
    float top = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // a part that sees no key of the row has no weight, whatever its sums hold
    const bool has = !(ml.x == -INFINITY && ml.y == 0.0f);
    const float mine = has ? ex2_ftz(ml.x - top) : 0.0f;
    const unsigned parts = __ballot_sync(0xffffffffu, has);
    float acc[kPer] = {}, den = 0.0f;
#pragma unroll 8
    for (int q = 0; q < p.splits; ++q) {
        const float w = __shfl_sync(0xffffffffu, mine, q), d = __shfl_sync(0xffffffffu, ml.y, q);
        const bool on = parts >> q & 1u;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const float o = on ? p.part[(q * rows + r) * HD + lane + 32 * e] : 0.0f;
            acc[e] = __fmaf_rn(o, w, acc[e]);
        }
        den = __fmaf_rn(d, w, den);
    }
    T* out = static_cast<T*>(p.out) + b * p.os[0] + h * p.os[1] + i * p.os[2];
    bool bad = false;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        const float f = sees ? __fdiv_rn(acc[e], den) : 0.0f;
        bad |= !finite_f(f);
        if (lane + 32 * e < p.d) out[lane + 32 * e] = F16<T>::one(f);
    }
    if (__any_sync(0xffffffffu, bad)) window_row<T>(p, b, h, i, qrow[warp], lane);
}

struct WinPlan {
    int hd, nq, q_tiles, splits;
    int64_t items, whole;
    int pitch;                   // channels of a packed row
    bool pack[3];                // Q, K, V
    size_t off[3], off_part, off_ml, total;
};

WinPlan plan(const vcb_window_args* a) {
    WinPlan r{};
    r.hd = a->d <= 64 ? 64 : 128;
    r.nq = a->sq <= 128 ? 1 : 2;
    r.pitch = (a->d + 7) / 8 * 8;
    const int64_t rows = 128 * r.nq;
    r.q_tiles = (int)((a->sq + rows - 1) / rows);
    const int64_t bh = a->batch * a->heads;
    // Key tiles of a query tile (an upper bound where lengths are on the device).
    auto tiles = [](int64_t n) { return (n + kKT - 1) / kKT; };
    const int64_t all = tiles(a->sk);
    const int64_t right = a->causal ? 0 : a->right;
    int64_t t = all;
    if (a->left >= 0 && right >= 0) {
        const int64_t span = tiles(a->left + right + (a->sq < rows ? a->sq : rows)) + 1;
        const int64_t sink = tiles(a->sinks);
        if (sink + span < all) t = sink + span;
    }
    // Items that do not fill the last round of CTAs are cut along their keys,
    // into as many parts as make the time of the rounds least: a part costs its
    // tiles and about four tiles' time, the join of all parts about four more.
    const int64_t slots = (int64_t)sm_count() * (r.nq == 1 ? 2 : 1);
    r.items = bh * r.q_tiles;
    const int64_t rest = r.items % slots;
    r.splits = 1;
    r.whole = r.items;
    int64_t best = rest ? t + 4 : 0;
    for (int64_t s = 2; rest && s <= 32 && s <= t; ++s) {
        const int64_t cost = (rest * s + slots - 1) / slots * ((t + s - 1) / s + 4) + 4;
        if (cost < best) {
            best = cost;
            r.splits = (int)s;
            r.whole = r.items - rest;
        }
    }
    const void* base[3] = {a->q, a->k, a->v};
    const int64_t* st[3] = {a->q_stride, a->k_stride, a->v_stride};
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    size_t o = 0;
    for (int i = 0; i < 3; ++i) {
        const int64_t n = i ? a->sk : a->sq;
        r.pack[i] = !on16(base[i]) || !tma_stride(st[i][0], a->batch) || !tma_stride(st[i][1], a->heads) ||
                    !tma_stride(st[i][2], n);
        r.off[i] = o;
        if (r.pack[i]) o += up((size_t)(bh * n * r.pitch) * 2);
    }
    r.off_part = o;
    const int64_t part_rows = r.splits * (r.items - r.whole) * rows;
    o += up((size_t)(part_rows * r.hd) * 4);
    r.off_ml = o;
    o += up((size_t)part_rows * 8);
    r.total = o;
    return r;
}

template <typename T, int HD, int NQ> int launch(const WinParams& p, const WinPlan& r, cudaStream_t st) {
    using L = WinTile<HD, NQ>;
    static bool ready[64] = {};
    auto kernel = window_kernel<T, HD, NQ>;
    int dev = 0;
    VCB_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(VCB_ERR_INVALID_ARGUMENT, "device ordinal %d out of range", dev);
    if (!ready[dev]) {
        VCB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::kSmem));
        cudaFuncAttributes fa;
        VCB_CUDA(cudaFuncGetAttributes(&fa, kernel));
        // a setmaxnreg.inc that the launch's registers cannot serve would wait forever
        if (fa.numRegs * L::kThreads < L::kRegSplit)
            return fail(VCB_ERR_CUDA, "window kernel launched with %d registers x %d threads, below its %d-register split",
                        fa.numRegs, L::kThreads, L::kRegSplit);
        ready[dev] = true;
    }
    const int64_t cut = r.items - r.whole;
    VCB_CUDA(launch_pdl(window_kernel<T, HD, NQ>, dim3((unsigned)(r.whole + cut * r.splits)), dim3(L::kThreads), L::kSmem,
                        st, p));
    if (cut) {
        const int64_t rows = cut * (p.q_tiles == 1 ? p.sq : 128 * NQ);
        VCB_CUDA(launch_pdl(window_join_kernel<T, HD, NQ>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p));
    }
    return VCB_OK;
}
template <typename T> int launch_any(const WinParams& p, const WinPlan& r, cudaStream_t st) {
    if (r.hd == 128) return r.nq == 1 ? launch<T, 128, 1>(p, r, st) : launch<T, 128, 2>(p, r, st);
    return r.nq == 1 ? launch<T, 64, 1>(p, r, st) : launch<T, 64, 2>(p, r, st);
}

}  // namespace

size_t window_workspace_bytes(const vcb_window_args* a) { return plan(a).total; }

int window_run(const vcb_window_args* a, cudaStream_t st) {
    const WinPlan r = plan(a);
    const int64_t bh = a->batch * a->heads;
    if (r.items >= (1ll << 30)) return fail(VCB_ERR_INVALID_ARGUMENT, "too many query tiles for one grid");
    WinParams p;
    memset(&p, 0, sizeof(p));
    p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
    p.kv_lens = a->kv_lens;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = a->q_stride[i]; p.ks[i] = a->k_stride[i]; p.vs[i] = a->v_stride[i]; p.os[i] = a->out_stride[i];
    }
    p.sq = a->sq; p.sk = a->sk; p.heads = a->heads;
    p.left = a->left; p.right = a->right; p.sinks = a->sinks;
    p.causal = a->causal; p.has_offset = a->has_offset; p.q_offset = a->q_offset;
    p.d = a->d; p.scale = a->scale;
    p.c = (float)((double)a->scale * 1.4426950408889634);
    p.q_tiles = r.q_tiles;
    p.whole = (int)r.whole; p.splits = r.splits;
    p.part_rows = (r.items - r.whole) * 128 * r.nq;
    p.vec_out = on16(a->out) && by8(a->d) && by8(a->out_stride[0]) && by8(a->out_stride[1]) && by8(a->out_stride[2]);
    char* ws = static_cast<char*>(a->workspace);
    p.part = reinterpret_cast<float*>(ws + r.off_part);
    p.part_ml = reinterpret_cast<float2*>(ws + r.off_ml);
    p.status = a->status;
    const void* base[3] = {a->q, a->k, a->v};
    const int64_t* strides[3] = {a->q_stride, a->k_stride, a->v_stride};
    CUtensorMap* maps[3] = {&p.tm_q, &p.tm_k, &p.tm_v};
    PackParams pk{};
    pk.channels = a->d;
    pk.pitch = r.pitch;
    int64_t blocks = 0;
    for (int i = 0; i < 3; ++i) {
        const int64_t n = i ? a->sk : a->sq;
        const void* at = base[i];
        int64_t sb = strides[i][0], sh = strides[i][1], ss = strides[i][2];
        if (r.pack[i]) {
            pk.side[i] = {static_cast<const uint16_t*>(at), reinterpret_cast<uint16_t*>(ws + r.off[i]), bh * n, n, sb, ss,
                          a->heads, sh, 0, a->d};
            blocks += (bh * n + 7) / 8;
            at = ws + r.off[i];
            ss = r.pitch; sh = n * ss; sb = a->heads * sh;
        }
        pk.end[i] = blocks;
        // strides of axes of length one are never taken: any legal value will do
        if (n == 1) ss = r.pitch;
        if (a->heads == 1) sh = r.pitch;
        if (a->batch == 1) sb = r.pitch;
        const cuuint64_t dims[4] = {(cuuint64_t)a->d, (cuuint64_t)n, (cuuint64_t)a->heads, (cuuint64_t)a->batch};
        const cuuint64_t bytes[3] = {(cuuint64_t)ss * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
        const cuuint32_t box[4] = {64, 128, 1, 1};
        int rc = make_map16(maps[i], at, a->dtype == VCB_BF16, 4, dims, bytes, box);
        if (rc) return rc;
    }
    if (blocks >= (1ll << 31)) return fail(VCB_ERR_INVALID_ARGUMENT, "too many rows for one grid");
    if (blocks) VCB_CUDA(launch_pack(pk, st));
    return a->dtype == VCB_BF16 ? launch_any<__nv_bfloat16>(p, r, st) : launch_any<__half>(p, r, st);
}

}  // namespace vcb
