// Attention's backward pass on the sm_100a tensor cores, probabilities recomputed from the saved
// log-sum-exp:
//
//   P_ij = exp(scale q_i k_j - lse_i), 0 where masked      delta_i = sum_d dO_id O_id
//   dV = P^T dO     dS = P * (dO V^T - delta)     dQ = scale dS K     dK = scale dS^T Q
//
// A key/value head shared by several query heads sums over them. P and dS are rounded to bf16, the type
// of the tensor cores' operands here; every sum is fp32. The roundings (relative 2^-8 each) average out
// over the terms of a sum. Where some sum of a CTA has fewer than kRows terms (the first queries and the
// last keys of a causal sequence, short sequences) the CTA carries P and dS as two bf16 terms, value and
// remainder, which keeps 16 bits; it runs at most four steps a head, so that costs next to nothing.
//
// Two kinds of CTA in one launch. A key CTA owns 128 keys of one key/value head and streams Q and dO in
// steps of 64 queries over every query head that shares it (4 products a step); a query CTA owns 128
// queries of one head and streams K and V in steps of 64 keys (3 products). Together 7 products where
// the mathematics needs 5: S and dO V^T are formed twice, but no gradient is summed across CTAs, so
// there are no atomics, no fp32 copy of dQ in memory, and the result does not depend on scheduling.
//
// Both kinds have one row (a key or a query) per TMEM lane, two score stages, and the same roles:
//   warps 0-3 / 4-7   even / odd steps: read S and dP (64 columns each), form P and dS, store them as
//                     bf16 into the stage's S columns for the products that follow
//   warp 8            issues the products:  S, dP of step i+2 after those that use P, dS of step i
//   warp 9            fills the ring of streamed tiles by TMA
// TMEM (512 columns): query CTA  Q 0-63, dO 64-127 (both as A operands), dQ 128-255, then per stage S and dP;
// key CTA  dV 0-127, dK 128-255, S of both stages 256-383, dP 384-447, V 448-511 (A operand); K, the A
// operand of S, is in shared memory. An A operand in TMEM halves what a product of 64 columns reads of
// shared memory, which otherwise bounds it (6 KB a 16-wide step against 128 B a cycle).
//
// Every wait is bounded; one that runs out sets the attention fault bit and the CTA's abort flag, the
// roles stop at their next wait and the outputs stay unwritten.
#include "attn.cuh"

namespace nb200 {
namespace {

constexpr int kRows = 128;  // rows a CTA owns (= TMEM lanes)
constexpr int kStep = 64;   // streamed rows a step
constexpr int kStages = 5;  // ring of streamed tiles
constexpr uint32_t kTileBytes = kStep * kDim * 2;  // 16 KB
constexpr uint32_t kHalfBytes = kTileBytes / 2;    // 64 columns: the TMA box
constexpr uint32_t kStatBytes = kStep * 4;         // one fp32 per streamed row
constexpr uint32_t kStageBytes = 2 * kTileBytes + 1024;  // two tiles and two statistics rows
constexpr uint32_t kFillBytes = 2 * kTileBytes;
constexpr uint32_t kOwnBytes = 2 * kTileBytes;     // a key CTA's K tile: two halves of 128 rows
constexpr uint32_t kOffOwn = 0;
constexpr uint32_t kOffRing = kOffOwn + kOwnBytes;
constexpr uint32_t kOffBar = kOffRing + kStages * kStageBytes;
constexpr int kMmaWarp = 8;
constexpr int kThreads = 320;  // warp 9, the last, is the producer
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kIdescScores = tc::idesc_bf16(128, kStep, false);
constexpr uint32_t kIdescGrads = tc::idesc_bf16(128, kDim, true);
// Query CTA: A operands, accumulator and stages.
constexpr uint32_t kColQ = 0, kColDO = 64, kColDQ = 128, kColStageQ = 256;  // stage: S, then dP at + 64
// Key CTA.
constexpr uint32_t kColDV = 0, kColDK = 128, kColStageK = 256, kColDP = 384, kColV = 448;

struct Bars {
    uint64_t full[kStages];
    uint64_t empty[kStages];
    uint64_t scores[2];   // S and dP of a stage are in TMEM
    uint64_t grads[2];    // P and dS of a stage are in TMEM (one arrival per warp)
    uint64_t dp_read;     // a key CTA's one dP buffer has been read (one arrival per warp)
    uint64_t own;         // the CTA's own operands: K in shared memory
    uint64_t own_tmem;    // ... and the A operands in TMEM (one arrival per warp)
    uint64_t done;
    uint64_t tail;        // a streamed tile with masked rows, before it is published
    uint32_t tmem_base;
    int abort;
};
constexpr uint32_t kSmemBytes = kOffBar + sizeof(Bars) + 1024;  // + alignment slack

struct BwdArgs {
    int S, Spad, H, Hk, group, key_ctas, key_blocks, query_blocks, causal;
    float scale, sl2;
    const int* lens;
    const __nv_bfloat16 *q, *v, *go;
    __nv_bfloat16 *dq, *dk, *dv;
    nb200_attn_strides sq, sv, sgo, sdq, sdk, sdv;
    const float* nlse2;   // [batch, heads, Spad]: -lse log2(e), -inf where the row sees nothing
    const float* ndelta;  // [batch, heads, Spad]: -delta
};

struct Maps {
    CUtensorMap q, k, v, go;
};

__device__ __forceinline__ int64_t offset(const nb200_attn_strides& s, int64_t b, int64_t h, int64_t i) {
    return b * s.batch + h * s.head + i * s.seq;
}

// ------------------------------------------------------------------ row statistics
// -lse log2(e) and -delta of every query row, padded to whole steps with -inf and 0, so that the
// probabilities of rows past the sequence come out as 2^-inf = 0 without a test. Half a warp per row.
constexpr int kStatThreads = 256;
constexpr int kStatRows = kStatThreads / 16;
struct StatArgs {
    const __nv_bfloat16 *o, *go;
    const float* lse;
    const int* lens;
    nb200_attn_strides so, sgo;
    int64_t rows;  // batch * heads * Spad
    int S, Spad, H;
    float *nlse2, *ndelta;
};

__global__ void __launch_bounds__(kStatThreads) bwd_stats_kernel(StatArgs a) {
    pdl_trigger();
    const int64_t row = (int64_t)blockIdx.x * kStatRows + threadIdx.x / 16;
    const int part = threadIdx.x % 16;
    const int64_t bh = row / a.Spad, b = bh / a.H, h = bh % a.H;
    const int i = (int)(row % a.Spad);
    float d = 0.f, l = -NB200_INF;
    if (row < a.rows && i < tokens_of(a.lens, (int)b, a.S)) {
        float o[8], g[8];
        Elem<__nv_bfloat16>::unpack(ld_stream(a.o + offset(a.so, b, h, i) + 8 * part), o);
        Elem<__nv_bfloat16>::unpack(ld_keep(a.go + offset(a.sgo, b, h, i) + 8 * part), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) d = fmaf(o[e], g[e], d);
        l = a.lse[bh * a.S + i];
        l = l == -NB200_INF ? l : -l * kLog2e;
    }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) d += __shfl_xor_sync(0xffffffffu, d, s);
    if (part == 0 && row < a.rows) {
        a.nlse2[row] = l;
        a.ndelta[row] = -d;
    }
}

// ------------------------------------------------------------------ products
// S-shaped product of a stage: 128 rows x kStep columns over the head dimension, eight K = 16 steps of
// 32 bytes inside a half's 128-byte rows. A from TMEM.
__device__ __forceinline__ void scores_ts(uint32_t d, uint32_t a, uint64_t b) {
    constexpr uint32_t h = kHalfBytes >> 4;
    tc::mma_ts_at<0, 0>(d, a, b, kIdescScores, 0u);
    tc::mma_ts_at<8, 2>(d, a, b, kIdescScores, 1u);
    tc::mma_ts_at<16, 4>(d, a, b, kIdescScores, 1u);
    tc::mma_ts_at<24, 6>(d, a, b, kIdescScores, 1u);
    tc::mma_ts_at<32, h + 0>(d, a, b, kIdescScores, 1u);
    tc::mma_ts_at<40, h + 2>(d, a, b, kIdescScores, 1u);
    tc::mma_ts_at<48, h + 4>(d, a, b, kIdescScores, 1u);
    tc::mma_ts_at<56, h + 6>(d, a, b, kIdescScores, 1u);
}
// The same with A in shared memory (halves of 128 rows).
__device__ __forceinline__ void scores_ss(uint32_t d, uint64_t a, uint64_t b) {
    constexpr uint32_t h = kHalfBytes >> 4, g = kTileBytes >> 4;
    tc::mma_ss_at<0, 0>(d, a, b, kIdescScores, 0u);
    tc::mma_ss_at<2, 2>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<4, 4>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<6, 6>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<g + 0, h + 0>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<g + 2, h + 2>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<g + 4, h + 4>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<g + 6, h + 6>(d, a, b, kIdescScores, 1u);
}
// Gradient-shaped product: 128 rows x 128 head columns (+)= A[128, kStep] (bf16 in TMEM) * streamed tile,
// read MN-major: 16 streamed rows = 2048 bytes a K = 16 step, the second 64 columns one half further.
__device__ __forceinline__ void grads_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t acc) {
    tc::mma_ts_at<0, 0>(d, a, b, kIdescGrads, acc);
    tc::mma_ts_at<8, 128>(d, a, b, kIdescGrads, 1u);
    tc::mma_ts_at<16, 256>(d, a, b, kIdescGrads, 1u);
    tc::mma_ts_at<24, 384>(d, a, b, kIdescGrads, 1u);
}

// Descriptors of the streamed tiles in the ring: as K-major and as MN-major B operands.
struct RingDesc {
    uint64_t k, mn;
    __device__ __forceinline__ explicit RingDesc(uint8_t* smem)
        : k(tc::sw128_desc(smem_u32(smem + kOffRing), 16, 1024)),
          mn(tc::sw128_desc(smem_u32(smem + kOffRing), kHalfBytes, 1024)) {}
    // tile 0: K or Q, tile 1: V or dO
    __device__ __forceinline__ static uint64_t step(int s, int tile) {
        return (uint64_t)((s * kStageBytes + tile * kTileBytes) >> 4);
    }
};

__device__ __forceinline__ void issue_query(uint8_t* smem, Bars* b, uint32_t tmem, int n, bool pair) {
    volatile int* abort = &b->abort;
    const RingDesc rd(smem);
    Ring<kStages> front, back;  // next tile for S and dP; next tile for dQ
    bool ok = wait_bar(&b->own_tmem, 0, abort);
    auto scores = [&](int st) {
        if (!wait_bar(&b->full[front.s], front.ph, abort)) return false;
        tc::fence_after();
        const uint32_t d = tmem + kColStageQ + 128 * st;
        scores_ts(d, tmem + kColQ, rd.k + RingDesc::step(front.s, 0));
        scores_ts(d + 64, tmem + kColDO, rd.k + RingDesc::step(front.s, 1));
        tc::commit(&b->scores[st]);
        front.next();
        return true;
    };
    ok = ok && scores(0);
    if (ok && n > 1) ok = scores(1);
    for (int j = 0; ok && j < n; ++j) {
        const int st = j & 1;
        if (!(ok = wait_bar(&b->grads[st], (j >> 1) & 1u, abort))) break;
        tc::fence_after();
        const uint32_t ds = tmem + kColStageQ + 128 * st;
        grads_ts(tmem + kColDQ, ds, rd.mn + RingDesc::step(back.s, 0), j > 0);
        if (pair) grads_ts(tmem + kColDQ, ds + 32, rd.mn + RingDesc::step(back.s, 0), 1u);
        tc::commit(&b->empty[back.s]);
        back.next();
        if (j + 2 < n) ok = scores(st);
    }
    tc::commit(&b->done);
    drain_bar(&b->done, 0);
}

// With pairs the remainders of P and dS take the dP buffer, so the next dP waits for the products of this
// step: S and dP of one step are issued at a time instead of two.
__device__ __forceinline__ void issue_key(uint8_t* smem, Bars* b, uint32_t tmem, int n, bool pair) {
    volatile int* abort = &b->abort;
    const RingDesc rd(smem);
    const uint64_t own = tc::sw128_desc(smem_u32(smem + kOffOwn), 16, 1024);
    Ring<kStages> front, back;
    bool ok = wait_bar(&b->own_tmem, 0, abort) && wait_bar(&b->own, 0, abort);
    // S and dP of step i; the one dP buffer is free once the warps have read step i - 1 out of it.
    auto scores = [&](int i) {
        if (!wait_bar(&b->full[front.s], front.ph, abort)) return false;
        tc::fence_after();
        scores_ss(tmem + kColStageK + 64 * (i & 1), own, rd.k + RingDesc::step(front.s, 0));
        if (i > 0 && !wait_bar(&b->dp_read, (i - 1) & 1u, abort)) return false;
        tc::fence_after();
        scores_ts(tmem + kColDP, tmem + kColV, rd.k + RingDesc::step(front.s, 1));
        tc::commit(&b->scores[i & 1]);
        front.next();
        return true;
    };
    const int ahead = pair ? 1 : 2;
    ok = ok && scores(0);
    if (ok && n > 1 && !pair) ok = scores(1);
    for (int i = 0; ok && i < n; ++i) {
        const int st = i & 1;
        if (!(ok = wait_bar(&b->grads[st], (i >> 1) & 1u, abort))) break;
        tc::fence_after();
        const uint32_t p = tmem + kColStageK + 64 * st;
        grads_ts(tmem + kColDV, p, rd.mn + RingDesc::step(back.s, 1), i > 0);
        grads_ts(tmem + kColDK, p + 32, rd.mn + RingDesc::step(back.s, 0), i > 0);
        if (pair) {
            grads_ts(tmem + kColDV, tmem + kColDP, rd.mn + RingDesc::step(back.s, 1), 1u);
            grads_ts(tmem + kColDK, tmem + kColDP + 32, rd.mn + RingDesc::step(back.s, 0), 1u);
        }
        tc::commit(&b->empty[back.s]);
        back.next();
        if (i + ahead < n) ok = scores(i + ahead);
    }
    tc::commit(&b->done);
    drain_bar(&b->done, 0);
}

// ------------------------------------------------------------------ the CTA's own operands
// One row of 128 bf16 per lane into 64 TMEM columns (two elements a column); zeros without a row.
__device__ __forceinline__ void own_row(uint32_t col, const __nv_bfloat16* row) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 u = row ? ld_keep(row + 64 * c + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
            w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
        __syncwarp();
        tc::tmem_st32(col + 32 * c, w);
    }
}

// kCols accumulator columns of this lane's row, times `scale`, to `row` as bf16 (zeros if the row is
// masked; nothing without a row).
template <int kCols>
__device__ __forceinline__ void write_row(uint32_t col, __nv_bfloat16* row, bool live, float scale) {
#pragma unroll
    for (int c = 0; c < kCols / 32; ++c) {
        uint32_t v[32];
        __syncwarp();
        tc::tmem_ld32(col + 32 * c, v);
        if (!row) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = live ? tc::pack_bf16(__uint_as_float(v[8 * i + 2 * e]) * scale,
                                            __uint_as_float(v[8 * i + 2 * e + 1]) * scale)
                            : 0u;
            *reinterpret_cast<uint4*>(row + 32 * c + 8 * i) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// Two fp32 values as bf16 pairs: rounded, and (kPair) what the rounding left.
template <bool kPair>
__device__ __forceinline__ void round_pair(uint64_t x, uint32_t& hi, uint32_t& lo) {
    hi = tc::pack_bf16(f2lo(x), f2hi(x));
    if constexpr (kPair)
        lo = tc::pack_bf16(f2lo(x) - __uint_as_float(hi << 16), f2hi(x) - __uint_as_float(hi & 0xffff0000u));
}

__device__ __forceinline__ void publish(uint64_t* bar, int lane) {
    tc::fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// ------------------------------------------------------------------ softmax warps
template <bool kPair>
__device__ __forceinline__ void query_warps(Bars* b, uint32_t tmem, const BwdArgs& a, int batch, int head, int len,
                                            int q0, int n) {
    volatile int* abort = &b->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const int row = q0 + (warp & 3) * 32 + lane;
    const bool live = row < len;
    const uint32_t t = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const __nv_bfloat16* src = half ? a.go + offset(a.sgo, batch, head, row) : a.q + offset(a.sq, batch, head, row);
    own_row(t + (half ? kColDO : kColQ), live ? src : nullptr);
    tc::tmem_wait_st();
    publish(&b->own_tmem, lane);
    const int64_t stat = ((int64_t)batch * a.H + head) * a.Spad + row;
    const float nl = live ? a.nlse2[stat] : -NB200_INF, nd = live ? a.ndelta[stat] : 0.f;
    const uint64_t nl2 = f2(nl, nl), nd2 = f2(nd, nd), sl2 = f2(a.sl2, a.sl2);
    const int lim = a.causal ? min(row, len - 1) : len - 1;  // last key this row sees
    const uint32_t tS = t + kColStageQ + 128 * half;
    bool ok = true;
    for (int j = half; j < n; j += 2) {
        if (!(ok = __all_sync(0xffffffffu, wait_bar(&b->scores[half], (j >> 1) & 1u, abort)))) break;
        tc::fence_after();
        uint32_t s[64], d[64];
        tc::tmem_ld64(tS, s);
        tc::tmem_ld64(tS + 64, d);
        const int room = lim - j * kStep;  // columns past it are masked
        if (__any_sync(0xffffffffu, room < kStep - 1)) {
#pragma unroll
            for (int c = 0; c < 64; ++c)
                if (c > room) s[c] = __float_as_uint(-NB200_INF);
        }
        uint32_t w[32], lo[32];
#pragma unroll
        for (int c = 0; c < 32; ++c) {
            const uint64_t x = fma2(f2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1])), sl2, nl2);
            const uint64_t p = f2(ex2_ftz(f2lo(x)), ex2_ftz(f2hi(x)));
            const uint64_t g = mul2(p, add2(f2(__uint_as_float(d[2 * c]), __uint_as_float(d[2 * c + 1])), nd2));
            round_pair<kPair>(g, w[c], lo[c]);
        }
        tc::tmem_st32(tS, w);
        if constexpr (kPair) tc::tmem_st32(tS + 32, lo);
        tc::tmem_wait_st();
        publish(&b->grads[half], lane);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_bar(&b->done, 0, abort));
    if (!ok) return;
    tc::fence_after();
    __nv_bfloat16* out = row < a.S ? a.dq + offset(a.sdq, batch, head, row) + 64 * half : nullptr;
    write_row<64>(t + kColDQ + 64 * half, out, live, a.scale);
}

template <bool kPair>
__device__ __forceinline__ void key_warps(uint8_t* smem, Bars* b, uint32_t tmem, const BwdArgs& a, int batch, int head,
                                          int len, int k0, int first, int per_head, int n) {
    volatile int* abort = &b->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const int row = k0 + (warp & 3) * 32 + lane;
    const bool live = row < len;
    const uint32_t t = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    if (half == 0) {
        own_row(t + kColV, live ? a.v + offset(a.sv, batch, head, row) : nullptr);
        tc::tmem_wait_st();
    }
    publish(&b->own_tmem, lane);
    const uint64_t sl2 = f2(a.sl2, a.sl2);
    const uint32_t tS = t + kColStageK + 64 * half;
    Ring<kStages> r;
    if (half) r.next();
    bool ok = true;
    int step = first + half;  // query step inside its head
    for (int i = half; i < n; i += 2, step += 2) {
        while (step >= first + per_head) step -= per_head;
        ok = wait_bar(&b->scores[half], (i >> 1) & 1u, abort) && wait_bar(&b->full[r.s], r.ph, abort);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc::fence_after();
        uint32_t s[64], d[64];
        tc::tmem_ld64(t + kColDP, d);
        publish(&b->dp_read, lane);
        tc::tmem_ld64(tS, s);
        const int hidden = a.causal ? row - step * kStep : 0;  // columns before it are masked
        if (__any_sync(0xffffffffu, hidden > 0)) {
#pragma unroll
            for (int c = 0; c < 64; ++c)
                if (c < hidden) s[c] = __float_as_uint(-NB200_INF);
        }
        const float4* nl = reinterpret_cast<const float4*>(smem + kOffRing + r.s * kStageBytes + 2 * kTileBytes);
        const float4* nd = nl + kStep / 4;
        uint32_t w[32], plo[32], wlo[32];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            const float4 l4 = nl[c], d4 = nd[c];
            const uint64_t l2[2] = {f2(l4.x, l4.y), f2(l4.z, l4.w)}, e2[2] = {f2(d4.x, d4.y), f2(d4.z, d4.w)};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = 4 * c + 2 * e;
                const uint64_t x = fma2(f2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), sl2, l2[e]);
                const uint64_t p = f2(ex2_ftz(f2lo(x)), ex2_ftz(f2hi(x)));
                const uint64_t g = mul2(p, add2(f2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])), e2[e]));
                round_pair<kPair>(p, s[k / 2], plo[k / 2]);
                round_pair<kPair>(g, w[k / 2], wlo[k / 2]);
            }
        }
        tc::tmem_st32(tS, s);
        tc::tmem_st32(tS + 32, w);
        if constexpr (kPair) {
            tc::tmem_st32(t + kColDP, plo);
            tc::tmem_st32(t + kColDP + 32, wlo);
        }
        tc::tmem_wait_st();
        publish(&b->grads[half], lane);
        r.next();
        r.next();
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_bar(&b->done, 0, abort));
    if (!ok) return;
    tc::fence_after();
    const nb200_attn_strides& so = half ? a.sdk : a.sdv;
    __nv_bfloat16* out = row < a.S ? (half ? a.dk : a.dv) + offset(so, batch, head, row) : nullptr;
    write_row<128>(t + (half ? kColDK : kColDV), out, live, half ? a.scale : 1.f);
}

// ------------------------------------------------------------------ producer (a whole warp; lane 0 issues)
// Streams n tile pairs: steps first .. first + per_head - 1 of heads head0, head0 + 1, ... Rows past the
// sequence in a head's last step are zeroed before the step is published (`tail` rows remain; 0: none
// to zero): they enter sums over the streamed rows, where a coefficient of 0 times an infinity or NaN
// would still poison the result. With statistics (a key CTA) their two rows come along.
__device__ __forceinline__ void produce(const CUtensorMap* mx, const CUtensorMap* my, uint8_t* smem, Bars* b,
                                        int batch, int head0, int first, int per_head, int n, int tail,
                                        const float* nlse2, const float* ndelta, const BwdArgs& a, int lane) {
    volatile int* abort = &b->abort;
    Ring<kStages> r;
    int it = 0, head = head0, step = first;
    uint32_t tail_ph = 0;
    bool ok = true;
    for (; it < n; ++it, r.next()) {
        ok = __all_sync(0xffffffffu, lane != 0 || wait_bar(&b->empty[r.s], r.ph ^ 1u, abort));
        if (!ok) break;
        uint8_t* dst = smem + kOffRing + r.s * kStageBytes;
        const bool cut = tail && step == first + per_head - 1;
        if (lane == 0) {
            uint64_t* bar = cut ? &b->tail : &b->full[r.s];
            mbar_expect_tx(bar, kFillBytes + (nlse2 ? 2 * kStatBytes : 0));
            const int row = step * kStep;
            tc::tma_load_4d(dst, mx, 0, row, head, batch, bar);
            tc::tma_load_4d(dst + kHalfBytes, mx, kDim / 2, row, head, batch, bar);
            tc::tma_load_4d(dst + kTileBytes, my, 0, row, head, batch, bar);
            tc::tma_load_4d(dst + kTileBytes + kHalfBytes, my, kDim / 2, row, head, batch, bar);
            if (nlse2) {
                const int64_t at = ((int64_t)batch * a.H + head) * a.Spad + row;
                bulk_load(dst + 2 * kTileBytes, nlse2 + at, kStatBytes, bar);
                bulk_load(dst + 2 * kTileBytes + kStatBytes, ndelta + at, kStatBytes, bar);
            }
        }
        if (cut) {
            ok = __all_sync(0xffffffffu, wait_bar(&b->tail, tail_ph, abort));
            if (!ok) break;
            tail_ph ^= 1u;
            zero_tail(dst, kStep, tail, lane);
            zero_tail(dst + kTileBytes, kStep, tail, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->full[r.s]);
        }
        if (++step == first + per_head) {
            step = first;
            ++head;
        }
    }
    // Every copy lands before the CTA may exit.
    if (lane == 0)
        for (int s = 0; s < kStages && s < it; ++s) drain_bar(&b->full[s], ((it - 1 - s) / kStages) & 1u);
}

__global__ void __launch_bounds__(kThreads, 1) attn_bwd_kernel(const __grid_constant__ Maps m, const BwdArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* b = reinterpret_cast<Bars*>(smem + kOffBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // Head-major order in both parts, so that the CTAs that run side by side share their streamed tiles
    // through L2; under a causal mask the longest of a head come first.
    const bool keys = (int)blockIdx.x < a.key_ctas;
    const int id = keys ? blockIdx.x : blockIdx.x - a.key_ctas;
    const int blocks = keys ? a.key_blocks : a.query_blocks, heads = keys ? a.Hk : a.H;
    const int batch = id / blocks / heads, head = id / blocks % heads;
    const int row0 = (keys ? id % blocks : blocks - 1 - id % blocks) * kRows;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&b->full[s], 1);
            mbar_init(&b->empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&b->scores[s], 1);
            mbar_init(&b->grads[s], 4);
        }
        mbar_init(&b->dp_read, 4);
        mbar_init(&b->own, 1);
        mbar_init(&b->own_tmem, 8);
        mbar_init(&b->done, 1);
        mbar_init(&b->tail, 1);
        b->abort = 0;
        fence_barrier_init();
        tc::prefetch_map(&m.q);
        tc::prefetch_map(&m.k);
        tc::prefetch_map(&m.v);
        tc::prefetch_map(&m.go);
    }
    pdl_wait();
    const int len = tokens_of(a.lens, batch, a.S);
    if (row0 >= len) {  // none of the CTA's rows belongs to the sequence
        const int rows = min(kRows, a.S - row0);
        for (int i = threadIdx.x; i < rows * (kDim / 8); i += kThreads) {
            const int r = row0 + i / (kDim / 8), c = i % (kDim / 8) * 8;
            const uint4 z = make_uint4(0u, 0u, 0u, 0u);
            if (keys) {
                *reinterpret_cast<uint4*>(a.dk + offset(a.sdk, batch, head, r) + c) = z;
                *reinterpret_cast<uint4*>(a.dv + offset(a.sdv, batch, head, r) + c) = z;
            } else {
                *reinterpret_cast<uint4*>(a.dq + offset(a.sdq, batch, head, r) + c) = z;
            }
        }
        return;
    }
    // Steps of the streamed side.
    const int first = keys && a.causal ? row0 / kStep : 0;
    const int end = !keys && a.causal ? min(row0 + kRows, len) : len;
    const int per_head = (end + kStep - 1) / kStep - first;
    const int n = keys ? a.group * per_head : per_head;
    const int tail = (first + per_head) * kStep > len && len < a.S ? len - (first + per_head - 1) * kStep : 0;
    // Some row's sum has fewer than kRows terms: queries that see few keys, keys few queries see.
    const bool pair = a.causal ? (keys ? row0 + 2 * kRows > len : row0 == 0) : len < kRows;

    if (warp == kMmaWarp) {
        tc::tmem_alloc(&b->tmem_base, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = b->tmem_base;

    if (warp < 8) {
        if (keys && pair) key_warps<true>(smem, b, tmem, a, batch, head, len, row0, first, per_head, n);
        else if (keys) key_warps<false>(smem, b, tmem, a, batch, head, len, row0, first, per_head, n);
        else if (pair) query_warps<true>(b, tmem, a, batch, head, len, row0, n);
        else query_warps<false>(b, tmem, a, batch, head, len, row0, n);
    } else if (warp == kMmaWarp) {
        if (lane == 0) {
            if (keys) issue_key(smem, b, tmem, n, pair);
            else issue_query(smem, b, tmem, n, pair);
        }
    } else if (keys) {
        if (lane == 0) {
            uint8_t* own = smem + kOffOwn;
            mbar_expect_tx(&b->own, kOwnBytes);
            for (int h = 0; h < 2; ++h)
                for (int r = 0; r < 2; ++r)
                    tc::tma_load_4d(own + h * kTileBytes + r * kHalfBytes, &m.k, h * kDim / 2, row0 + r * kStep, head,
                                    batch, &b->own);
        }
        produce(&m.q, &m.go, smem, b, batch, head * a.group, first, per_head, n, tail, a.nlse2, a.ndelta, a, lane);
        if (lane == 0) drain_bar(&b->own, 0);
    } else {
        produce(&m.k, &m.v, smem, b, batch, head / a.group, 0, per_head, n, tail, nullptr, nullptr, a, lane);
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc::fence_after();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

SharedLimit g_shared;

int64_t padded(int64_t seq) { return (seq + kStep - 1) / kStep * kStep; }

}  // namespace

int attn_bwd_fault_take(unsigned int* bits) { return take_attn_fault(bits); }

int64_t attention_bwd_work_bytes(const nb200_attn_args& n) {
    return 2 * n.batch * n.heads * padded(n.seq) * (int64_t)sizeof(float);
}

int launch_attention_bwd(const nb200_attn_args& n, const nb200_attn_strides* strides, const void* q, const void* k,
                         const void* v, const void* o, const float* lse, const void* grad_o, void* dq, void* dk,
                         void* dv, void* work, cudaStream_t st) {
    const char* what = "nb200_attention_bwd";
    using B = __nv_bfloat16;
    const int64_t blocks = (n.seq + kRows - 1) / kRows, pad = padded(n.seq), rows = n.batch * n.heads * pad;
    const int64_t ctas = n.batch * (n.heads + n.kv_heads) * blocks, stat_ctas = (rows + kStatRows - 1) / kStatRows;
    if (ctas > 0x7fffffffLL || stat_ctas > 0x7fffffffLL) {
        set_error("%s: batch*heads=%lld, seq=%lld exceed the kernel's index range", what,
                  (long long)(n.batch * n.heads), (long long)n.seq);
        return NB200_ERR_CAPACITY;
    }
    Maps m;
    int rc;
    if ((rc = encode_rows(&m.q, what, "q", q, n.batch, n.heads, n.seq, strides[0], kStep)) ||
        (rc = encode_rows(&m.k, what, "k", k, n.batch, n.kv_heads, n.seq, strides[1], kStep)) ||
        (rc = encode_rows(&m.v, what, "v", v, n.batch, n.kv_heads, n.seq, strides[2], kStep)) ||
        (rc = encode_rows(&m.go, what, "grad_o", grad_o, n.batch, n.heads, n.seq, strides[4], kStep)) ||
        (rc = g_shared.raise(what, attn_bwd_kernel, kSmemBytes)))
        return rc;
    StatArgs s;
    s.o = static_cast<const B*>(o);
    s.go = static_cast<const B*>(grad_o);
    s.lse = lse;
    s.lens = n.seq_lens;
    s.so = strides[3];
    s.sgo = strides[4];
    s.rows = rows;
    s.S = (int)n.seq;
    s.Spad = (int)pad;
    s.H = (int)n.heads;
    s.nlse2 = static_cast<float*>(work);
    s.ndelta = s.nlse2 + rows;
    bwd_stats_kernel<<<(unsigned)stat_ctas, kStatThreads, 0, st>>>(s);
    BwdArgs a;
    a.S = (int)n.seq;
    a.Spad = (int)pad;
    a.H = (int)n.heads;
    a.Hk = (int)n.kv_heads;
    a.group = (int)(n.heads / n.kv_heads);
    a.key_ctas = (int)(n.batch * n.kv_heads * blocks);
    a.key_blocks = a.query_blocks = (int)blocks;
    a.causal = n.causal ? 1 : 0;
    a.scale = n.scale;
    a.sl2 = n.scale * 1.4426950408889634f;
    a.lens = n.seq_lens;
    a.q = static_cast<const B*>(q);
    a.v = static_cast<const B*>(v);
    a.go = static_cast<const B*>(grad_o);
    a.dq = static_cast<B*>(dq);
    a.dk = static_cast<B*>(dk);
    a.dv = static_cast<B*>(dv);
    a.sq = strides[0];
    a.sv = strides[2];
    a.sgo = strides[4];
    a.sdq = strides[5];
    a.sdk = strides[6];
    a.sdv = strides[7];
    a.nlse2 = s.nlse2;
    a.ndelta = s.ndelta;
    launch_pdl(attn_bwd_kernel, (unsigned)ctas, kThreads, kSmemBytes, st, m, a);
    count_launch(2);
    return finish_launch(what);
}

}  // namespace nb200
