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
// steps of 128 queries over every query head that shares it (4 products a step); a query CTA owns 128
// queries of one head and streams K and V in steps of 128 keys (3 products). Together 7 products where
// the mathematics needs 5: S and dO V^T are formed twice, but no gradient is summed across CTAs, so
// there are no atomics, no fp32 copy of dQ in memory, and the result does not depend on scheduling.
//
// Both kinds have one row (a key or a query) per TMEM lane and the same roles:
//   warps 0-3 / 4-7   columns 0-63 / 64-127 of the scores: read S and dP, form P and dS, store them as
//                     bf16 into TMEM, the A operand of the products that sum them
//   warp 8            issues the products
//   warp 9            fills the ring of streamed tiles by TMA
//
// Key CTA.  TMEM: dV 0-127, dK 128-255, S 256-383 (P over it), dP 384-511 (dS over it). K and V are in
// shared memory. Order of the products: dV(i), S(i+1), dK(i), dP(i+1); while the tensor pipe works on one
// pair the warps work on the other: P(i+1) from S(i+1) during dK(i), dP(i+1), and dS(i) during dV(i), S(i+1).
// Query CTA.  TMEM: dQ 0-127, S 128-255, dP 256-383, dS 384-447, dO 448-511 (A operand). Q is in shared
// memory. S and dP of step j+1 are issued as soon as the warps hold step j in registers, dQ(j) when dS(j)
// is stored: the exponentials of a step (1024 cycles of the special-function unit) run under the products.
//
// Where a few key CTAs would run far longer than the rest (shared heads: a key CTA streams every query head
// of its group), each is cut into `parts` CTAs of consecutive steps whose fp32 sums a third kernel adds in
// order and rounds.
//
// Measured on one B200, bf16: [8, 32, 4096, 128] 6.6 ms under continuous load, at the power cap (835 TFLOP/s of the
// mathematics' 5 products, 1168 of the 7 executed, 0.86 of the sustained cuBLAS rate); a few passes from idle take
// 5.65 ms (973, 1362 and 0.83 of the burst rate). A key step
// takes 2930 cycles for 2048 of products, bound by shared memory (256 KB of operands, 64 KB of incoming tiles and
// the statistics at 128 B a cycle); a query step 2000 for 1536, its exponentials and hand-offs about 1700. A
// CTA costs 4 to 5 us besides its steps.
//
// Every wait is bounded; one that runs out sets the attention fault bit and the CTA's abort flag, the
// roles stop at their next wait and the outputs stay unwritten.
#include <stddef.h>

#include <algorithm>

#include "attn.cuh"

namespace nb200 {
namespace {

constexpr int kRows = 128;  // rows a CTA owns (= TMEM lanes)
constexpr int kStep = 128;  // streamed rows a step
// Rings of streamed tiles, which alternate K, V (or Q, dO): what the CTA's own operands leave of the
// shared memory. A query CTA needs six: V(j+1) would otherwise wait for K(j-1), that is for dQ(j-1).
constexpr int kKeyStages = 5;
constexpr int kQueryStages = 6;
constexpr uint32_t kTileBytes = kStep * kDim * 2;  // 32 KB
constexpr uint32_t kHalfBytes = kTileBytes / 2;    // 64 columns: the TMA box
constexpr uint32_t kStatBytes = kStep * 4;         // one fp32 per streamed row
constexpr uint32_t kOffOwn = 0;  // K and V of a key CTA, Q of a query CTA; the ring follows
constexpr uint32_t kOffKeyRing = kOffOwn + 2 * kTileBytes;
constexpr uint32_t kOffQueryRing = kOffOwn + kTileBytes;
constexpr uint32_t kOffStat = kOffKeyRing + kKeyStages * kTileBytes;  // two steps of two statistics rows
static_assert(kOffQueryRing + kQueryStages * kTileBytes == kOffStat, "rings end together");
constexpr uint32_t kOffBar = kOffStat + 2 * 2 * kStatBytes;
constexpr int kMmaWarp = 8;
constexpr int kLoadWarp = 9;
constexpr int kThreads = 384;  // warps 10-11 only complete the third warpgroup for the register split
// Register split (setmaxnreg, per warpgroup), within what the block is launched with.
constexpr int kLaunchRegs = 168;
constexpr int kRegsSoftmax = 208;
constexpr int kRegsControl = 88;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsControl <= kThreads * kLaunchRegs, "register split");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kIdescScores = tc::idesc_bf16(128, kStep, false);
constexpr uint32_t kIdescGrads = tc::idesc_bf16(128, kDim, true);
constexpr uint32_t kColDV = 0, kColDK = 128, kColKeyS = 256, kColKeyDP = 384;
constexpr uint32_t kColDQ = 0, kColQueryS = 128, kColQueryDP = 256, kColDS = 384, kColDO = 448;

struct Bars {
    // one arrival a phase
    uint64_t full[kQueryStages];
    uint64_t empty[kQueryStages];
    uint64_t s_full;        // S is in TMEM (a query CTA: S and dP)
    uint64_t dp_full;       // dP is in TMEM (key CTA)
    uint64_t ds_free;       // a query CTA's dS has been consumed
    uint64_t stat_full[2];  // statistics of a key CTA's step
    uint64_t own;           // the CTA's own operands in shared memory
    uint64_t done;
    uint64_t tail;          // a streamed tile with masked rows, before it is published
    // one arrival from each of four warps
    uint64_t p_full[2];     // P of a column half is in TMEM
    uint64_t ds_full[2];    // dS of a column half
    // one arrival from each of eight warps
    uint64_t read;          // a query CTA's S and dP are in registers
    uint64_t stat_empty[2];
    uint64_t own_tmem;      // the own operand in TMEM
    uint32_t tmem_base;
    int abort;
};
constexpr int kFourArrivals = offsetof(Bars, p_full) / 8, kEightArrivals = offsetof(Bars, read) / 8;
constexpr int kBarriers = offsetof(Bars, tmem_base) / 8;
static_assert(kBarriers <= 32, "one lane sets up one barrier");
constexpr uint32_t kSmemBytes = kOffBar + sizeof(Bars);
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

struct BwdArgs {
    int S, Spad, H, Hk, group, parts, key_ctas, blocks, causal;
    float scale, sl2;
    const int* lens;
    const __nv_bfloat16* go;
    __nv_bfloat16 *dq, *dk, *dv;
    nb200_attn_strides sgo, sdq, sdk, sdv;
    const float* nlse2;   // [batch, heads, Spad]: -lse log2(e), -inf where the row sees nothing
    const float* ndelta;  // [batch, heads, Spad]: -delta
    float *part_k, *part_v;  // [parts, batch, kv_heads, S, 128], with parts > 1
    int64_t part_rows;       // batch * kv_heads * S
};

struct Maps {
    CUtensorMap q, k, v, go;   // boxes of kStep rows
    CUtensorMap dq, dk, dv;    // boxes of 32 rows: what one warp stores
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
// Scores: 128 rows x 128 streamed rows over the head dimension, eight K = 16 steps of 32 bytes inside a
// half's 128-byte rows. Both operands in shared memory, or A in TMEM (8 columns a step).
__device__ __forceinline__ void scores_ss(uint32_t d, uint64_t a, uint64_t b) {
    constexpr uint32_t h = kHalfBytes >> 4;
    tc::mma_ss_at<0>(d, a, b, kIdescScores, 0u);
    tc::mma_ss_at<2>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<4>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<6>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<h + 0>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<h + 2>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<h + 4>(d, a, b, kIdescScores, 1u);
    tc::mma_ss_at<h + 6>(d, a, b, kIdescScores, 1u);
}
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
// Half of a gradient product: 128 rows x 128 head columns (+)= A[128, 64] (bf16 in TMEM) * 64 rows of a
// streamed tile, read MN-major: 16 streamed rows = 2048 bytes a K = 16 step.
__device__ __forceinline__ void grads_ts(uint32_t d, uint32_t a, uint64_t tile, int half, uint32_t acc) {
    const uint64_t b = tile + half * 512;
    tc::mma_ts_at<0, 0>(d, a, b, kIdescGrads, acc);
    tc::mma_ts_at<8, 128>(d, a, b, kIdescGrads, 1u);
    tc::mma_ts_at<16, 256>(d, a, b, kIdescGrads, 1u);
    tc::mma_ts_at<24, 384>(d, a, b, kIdescGrads, 1u);
}

// Descriptors of the ring's tiles, as K-major and as MN-major B operands (the second 64 head columns one
// half further).
struct RingDesc {
    uint64_t k0, mn0;
    __device__ __forceinline__ explicit RingDesc(uint8_t* ring)
        : k0(tc::sw128_desc(smem_u32(ring), 16, 1024)), mn0(tc::sw128_desc(smem_u32(ring), kHalfBytes, 1024)) {}
    __device__ __forceinline__ uint64_t k(int s) const { return k0 + ((s * kTileBytes) >> 4); }
    __device__ __forceinline__ uint64_t mn(int s) const { return mn0 + ((s * kTileBytes) >> 4); }
};

// Waits for both column halves of an operand as they are stored and issues their half products.
__device__ __forceinline__ bool grads(uint64_t* ready, uint32_t parity, uint32_t d, uint32_t a, uint32_t half_cols,
                                      uint32_t lo, uint64_t tile, bool acc, bool pair, volatile int* abort) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (!wait_bar(&ready[h], parity, abort)) return false;
        tc::fence_after();
        grads_ts(d, a + h * half_cols, tile, h, acc || h ? 1u : 0u);
        if (pair) grads_ts(d, lo + h * 64, tile, h, 1u);
    }
    return true;
}

__device__ __forceinline__ void issue_query(uint8_t* smem, Bars* b, uint32_t tmem, int n, bool pair) {
    volatile int* abort = &b->abort;
    const RingDesc rd(smem + kOffQueryRing);
    const uint64_t own = tc::sw128_desc(smem_u32(smem + kOffOwn), 16, 1024);
    Ring<kQueryStages> k, v, back;  // next K and V tile for S and dP; next K tile for dQ
    v.next();
    auto scores = [&](bool first) {
        if (!wait_bar(&b->full[k.s], k.ph, abort)) return false;
        tc::fence_after();
        scores_ss(tmem + kColQueryS, own, rd.k(k.s));
        if (first && !wait_bar(&b->own_tmem, 0, abort)) return false;
        if (!wait_bar(&b->full[v.s], v.ph, abort)) return false;
        tc::fence_after();
        scores_ts(tmem + kColQueryDP, tmem + kColDO, rd.k(v.s));
        tc::commit(&b->s_full);
        tc::commit(&b->empty[v.s]);
        k.next(), k.next(), v.next(), v.next();
        return true;
    };
    bool ok = wait_bar(&b->own, 0, abort) && scores(true);
    for (int j = 0; ok && j < n; ++j) {
        const uint32_t ph = j & 1u;
        if (j + 1 < n && !(ok = wait_bar(&b->read, ph, abort) && scores(false))) break;
        if (!(ok = grads(b->ds_full, ph, tmem + kColDQ, tmem + kColDS, 32, tmem + kColQueryS, rd.mn(back.s), j > 0,
                         pair, abort)))
            break;
        tc::commit(&b->ds_free);
        tc::commit(&b->empty[back.s]);
        back.next(), back.next();
    }
    tc::commit(&b->done);
    drain_bar(&b->done, 0);
}

__device__ __forceinline__ void issue_key(uint8_t* smem, Bars* b, uint32_t tmem, int n, bool pair) {
    volatile int* abort = &b->abort;
    const RingDesc rd(smem + kOffKeyRing);
    const uint64_t own = tc::sw128_desc(smem_u32(smem + kOffOwn), 16, 1024);
    Ring<kKeyStages> q, go;  // the tiles of this step; S and dP of the next step run one step ahead
    go.next();
    auto scores = [&](const Ring<kKeyStages>& r, uint64_t a, uint32_t d, uint64_t* bar) {
        if (!wait_bar(&b->full[r.s], r.ph, abort)) return false;
        tc::fence_after();
        scores_ss(d, a, rd.k(r.s));
        tc::commit(bar);
        return true;
    };
    const uint32_t s = tmem + kColKeyS, dp = tmem + kColKeyDP;
    const uint64_t own_v = own + (kTileBytes >> 4);
    bool ok = wait_bar(&b->own, 0, abort) && scores(q, own, s, &b->s_full) && scores(go, own_v, dp, &b->dp_full);
    for (int i = 0; ok && i < n; ++i) {
        const uint32_t ph = i & 1u;
        const bool more = i + 1 < n;
        Ring<kKeyStages> q1 = q, go1 = go;
        q1.next(), q1.next(), go1.next(), go1.next();
        if (!(ok = grads(b->p_full, ph, tmem + kColDV, s, 64, s + 32, rd.mn(go.s), i > 0, pair, abort))) break;
        tc::commit(&b->empty[go.s]);
        if (more && !(ok = scores(q1, own, s, &b->s_full))) break;
        if (!(ok = grads(b->ds_full, ph, tmem + kColDK, dp, 64, dp + 32, rd.mn(q.s), i > 0, pair, abort))) break;
        tc::commit(&b->empty[q.s]);
        if (more && !(ok = scores(go1, own_v, dp, &b->dp_full))) break;
        q = q1;
        go = go1;
    }
    tc::commit(&b->done);
    drain_bar(&b->done, 0);
}

// ------------------------------------------------------------------ the CTA's own operands
// What a softmax thread of a query CTA fetches for itself, on its way while the CTA sets up: 64 columns of its
// row of dO (zeros without a row) and, once the kernel before is through, the row's statistics.
struct QueryRow {
    uint32_t go[32];
    float nl, nd;
    __device__ __forceinline__ void load(const BwdArgs& a, int batch, int head, int len, int q0) {
        const int warp = threadIdx.x >> 5, row = q0 + (warp & 3) * 32 + (threadIdx.x & 31);
        const bool live = row < len;
        const __nv_bfloat16* src = a.go + offset(a.sgo, batch, head, row) + 64 * (warp >> 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint4 u = live ? ld_keep(src + 8 * i) : make_uint4(0u, 0u, 0u, 0u);
            go[4 * i] = u.x, go[4 * i + 1] = u.y, go[4 * i + 2] = u.z, go[4 * i + 3] = u.w;
        }
        pdl_wait();
        const int64_t stat = ((int64_t)batch * a.H + head) * a.Spad + row;
        nl = live ? a.nlse2[stat] : -NB200_INF;
        nd = live ? a.ndelta[stat] : 0.f;
    }
};

// 64 accumulator columns of this lane's row, times `scale`, as bf16 into row r of half `h` of a staged tile, in the
// swizzle the tensor maps expect (zeros if the row is masked).
__device__ __forceinline__ void stage_half(uint32_t col, uint8_t* tile, int h, int r, bool live, float scale) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        uint32_t v[32];
        tc::tmem_ld32(col + 32 * c, v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = live ? tc::pack_bf16(__uint_as_float(v[8 * i + 2 * e]) * scale,
                                            __uint_as_float(v[8 * i + 2 * e + 1]) * scale)
                            : 0u;
            *reinterpret_cast<uint4*>(tile + h * kHalfBytes + r * 128 + (((4 * c + i) ^ (r & 7)) << 4)) =
                make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}
// Stores halves h0 .. h1 - 1 of this warp's 32 staged rows; rows past the tensor are not written.
__device__ __forceinline__ void store_rows(const CUtensorMap* m, const uint8_t* tile, int h0, int h1, int quarter,
                                           int row, int seq, int head, int batch, int lane) {
    fence_proxy_async();
    __syncwarp();
    if (lane == 0 && row < seq) {
        for (int h = h0; h < h1; ++h)
            tc::tma_store_4d(m, tile + h * kHalfBytes + quarter * 32 * 128, h * kDim / 2, row, head, batch);
        tc::bulk_commit();
        tc::bulk_wait_read();
    }
    __syncwarp();
}

// The 128 accumulator columns of this lane's row as fp32 (nothing without a row).
__device__ __forceinline__ void write_row_f32(uint32_t col, float* row) {
#pragma unroll
    for (int c = 0; c < kDim / 32; ++c) {
        uint32_t v[32];
        __syncwarp();
        tc::tmem_ld32(col + 32 * c, v);
        if (!row) continue;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<uint4*>(row + 32 * c + 4 * i) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
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
__device__ __forceinline__ void query_warps(const Maps& m, uint8_t* smem, Bars* b, uint32_t tmem, const BwdArgs& a,
                                            const QueryRow& own, int batch, int head, int len, int q0, int n) {
    volatile int* abort = &b->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const int row = q0 + (warp & 3) * 32 + lane;
    const bool live = row < len;
    const uint32_t t = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    __syncwarp();
    tc::tmem_st32(t + kColDO + 32 * half, own.go);
    tc::tmem_wait_st();
    publish(&b->own_tmem, lane);
    const uint64_t nl2 = f2(own.nl, own.nl), nd2 = f2(own.nd, own.nd), sl2 = f2(a.sl2, a.sl2);
    const int lim = (a.causal ? min(row, len - 1) : len - 1) - 64 * half;  // last key this row sees, from column 0 on
    const uint32_t tS = t + kColQueryS + 64 * half, tDS = t + kColDS + 32 * half;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
        if (!(ok = __all_sync(0xffffffffu, wait_bar(&b->s_full, j & 1u, abort)))) break;
        tc::fence_after();
        uint32_t s[64], d[64];
        tc::tmem_ld64(tS, s);
        tc::tmem_ld64(tS + (kColQueryDP - kColQueryS), d);
        publish(&b->read, lane);
        const int room = lim - j * kStep;  // columns past it are masked
        if (__any_sync(0xffffffffu, room < 63)) {
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
        if (j > 0 && !(ok = __all_sync(0xffffffffu, wait_bar(&b->ds_free, (j - 1) & 1u, abort)))) break;
        tc::tmem_st32(tDS, w);
        // Remainders go over S: a CTA that has them runs one step, so no further S is on its way.
        if constexpr (kPair) tc::tmem_st32(tS, lo);
        tc::tmem_wait_st();
        publish(&b->ds_full[half], lane);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_bar(&b->done, 0, abort));
    if (!ok) return;
    tc::fence_after();
    // Every streamed tile has been consumed: the ring's first tile stages dQ.
    uint8_t* tile = smem + kOffQueryRing;
    stage_half(t + kColDQ + 64 * half, tile, half, row - q0, live, a.scale);
    store_rows(&m.dq, tile, half, half + 1, warp & 3, q0 + (warp & 3) * 32, a.S, head, batch, lane);
}

template <bool kPair>
__device__ __forceinline__ void key_warps(const Maps& m, uint8_t* smem, Bars* b, uint32_t tmem, const BwdArgs& a, int batch, int head,
                                          int len, int k0, int first, int per_head, int skip, int n, int part) {
    volatile int* abort = &b->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = warp >> 2;
    const int row = k0 + (warp & 3) * 32 + lane;
    const bool live = row < len;
    const uint32_t t = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint64_t sl2 = f2(a.sl2, a.sl2);
    const uint32_t tS = t + kColKeyS + 64 * half, tDP = t + kColKeyDP + 64 * half;
    bool ok = true;
    for (int i = 0, step = first + skip % per_head; i < n; ++i) {
        const uint32_t ph = i & 1u;
        ok = wait_bar(&b->s_full, ph, abort) && wait_bar(&b->stat_full[ph], (i >> 1) & 1u, abort);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc::fence_after();
        const float4* nl = reinterpret_cast<const float4*>(smem + kOffStat + ph * 2 * kStatBytes) + 16 * half;
        const float4* nd = nl + kStep / 4;
        uint32_t s[64], w[32], lo[32];
        tc::tmem_ld64(tS, s);
        const int hidden = a.causal ? row - step * kStep - 64 * half : 0;  // columns before it are masked
        if (__any_sync(0xffffffffu, hidden > 0)) {
#pragma unroll
            for (int c = 0; c < 64; ++c)
                if (c < hidden) s[c] = __float_as_uint(-NB200_INF);
        }
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
            const float4 l4 = nl[c / 2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = 2 * (c + e);
                const uint64_t x = fma2(f2(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), sl2,
                                        e ? f2(l4.z, l4.w) : f2(l4.x, l4.y));
                const uint64_t p = f2(ex2_ftz(f2lo(x)), ex2_ftz(f2hi(x)));
                s[k] = __float_as_uint(f2lo(p));
                s[k + 1] = __float_as_uint(f2hi(p));
                round_pair<kPair>(p, w[c + e], lo[c + e]);
            }
        }
        tc::tmem_st32(tS, w);
        if constexpr (kPair) tc::tmem_st32(tS + 32, lo);
        tc::tmem_wait_st();
        publish(&b->p_full[half], lane);

        if (!(ok = __all_sync(0xffffffffu, wait_bar(&b->dp_full, ph, abort)))) break;
        tc::fence_after();
        uint32_t d[64];
        tc::tmem_ld64(tDP, d);
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
            const float4 d4 = nd[c / 2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int k = 2 * (c + e);
                const uint64_t p = f2(__uint_as_float(s[k]), __uint_as_float(s[k + 1]));
                const uint64_t g = mul2(p, add2(f2(__uint_as_float(d[k]), __uint_as_float(d[k + 1])),
                                                e ? f2(d4.z, d4.w) : f2(d4.x, d4.y)));
                round_pair<kPair>(g, w[c + e], lo[c + e]);
            }
        }
        tc::tmem_st32(tDP, w);
        if constexpr (kPair) tc::tmem_st32(tDP + 32, lo);
        tc::tmem_wait_st();
        publish(&b->ds_full[half], lane);
        if (lane == 0) mbar_arrive(&b->stat_empty[ph]);
        if (++step == first + per_head) step = first;
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_bar(&b->done, 0, abort));
    if (!ok) return;
    tc::fence_after();
    if (a.parts > 1) {
        const int64_t at = part * a.part_rows + ((int64_t)batch * a.Hk + head) * a.S + row;
        write_row_f32(t + (half ? kColDK : kColDV), live ? (half ? a.part_k : a.part_v) + at * kDim : nullptr);
        return;
    }
    uint8_t* tile = smem + kOffKeyRing + half * kTileBytes;
    for (int h = 0; h < 2; ++h)
        stage_half(t + (half ? kColDK : kColDV) + 64 * h, tile, h, row - k0, live, half ? a.scale : 1.f);
    store_rows(half ? &m.dk : &m.dv, tile, 0, 2, warp & 3, k0 + (warp & 3) * 32, a.S, head, batch, lane);
}

// ------------------------------------------------------------------ producer (a whole warp; lane 0 issues)
__device__ __forceinline__ void load_tile(uint8_t* dst, const CUtensorMap* m, int row, int head, int batch,
                                          uint64_t* bar) {
    tc::tma_load_4d(dst, m, 0, row, head, batch, bar);
    tc::tma_load_4d(dst + kHalfBytes, m, kDim / 2, row, head, batch, bar);
}

// Streams n steps of two tiles from step `skip` on of steps first .. first + per_head - 1 of heads head0, head0 + 1,
// ... Rows past the sequence in a head's last step are zeroed before the tile is published (`tail` rows remain;
// 0: none to zero): they enter sums over the streamed rows, where a coefficient of 0 times an infinity or NaN
// would still poison the result. A key CTA's steps come with their rows' statistics.
template <bool kKeys>
struct Producer {
    static constexpr int kStages = kKeys ? kKeyStages : kQueryStages;
    const CUtensorMap *mx, *my;
    uint8_t* smem;
    Bars* b;
    int batch, first, per_head, tiles, tail;
    const BwdArgs& a;
    int head, step, it = 0;
    uint32_t tail_ph = 0;
    bool ok = true, left = false;
    Ring<kStages> r;

    __device__ __forceinline__ Producer(const CUtensorMap* mx_, const CUtensorMap* my_, uint8_t* smem_, Bars* b_, int batch_,
                                        int head0, int first_, int per_head_, int skip, int n, int tail_,
                                        const BwdArgs& a_)
        : mx(mx_), my(my_), smem(smem_), b(b_), batch(batch_), first(first_), per_head(per_head_), tiles(2 * n),
          tail(tail_), a(a_), head(head0 + skip / per_head_), step(first_ + skip % per_head_) {}

    // Issues tiles up to number `end`; ahead of the CTA's first barrier (`early`) only those nothing waits for.
    __device__ __forceinline__ void run(int end, bool early, int lane) {
        volatile int* abort = &b->abort;
        for (; ok && it < end; ++it, r.next()) {
            const int i = it >> 1;
            const bool second = it & 1, cut = tail && step == first + per_head - 1;
            if (early && cut) return;
            ok = lane != 0 || wait_bar(&b->empty[r.s], r.ph ^ 1u, abort);
            if (kKeys && ok && lane == 0 && !second) ok = wait_bar(&b->stat_empty[i & 1], ((i >> 1) & 1u) ^ 1u, abort);
            if (!(ok = __all_sync(0xffffffffu, ok))) return;
            uint8_t* dst = smem + (kKeys ? kOffKeyRing : kOffQueryRing) + r.s * kTileBytes;
            if (lane == 0) {
                uint64_t* bar = cut ? &b->tail : &b->full[r.s];
                mbar_expect_tx(bar, kTileBytes);
                load_tile(dst, second ? my : mx, step * kStep, head, batch, bar);
                if (kKeys && !second) {
                    const int64_t at = ((int64_t)batch * a.H + head) * a.Spad + step * kStep;
                    uint8_t* to = smem + kOffStat + (i & 1) * 2 * kStatBytes;
                    mbar_expect_tx(&b->stat_full[i & 1], 2 * kStatBytes);
                    bulk_load(to, a.nlse2 + at, kStatBytes, &b->stat_full[i & 1]);
                    bulk_load(to + kStatBytes, a.ndelta + at, kStatBytes, &b->stat_full[i & 1]);
                }
            }
            if (cut) {
                if (!(ok = __all_sync(0xffffffffu, wait_bar(&b->tail, tail_ph, abort)))) {
                    if (lane == 0) drain_bar(&b->tail, tail_ph);
                    left = !second;  // the statistics came with this tile
                    return;
                }
                tail_ph ^= 1u;
                zero_tail(dst, kStep, tail, lane);
                __syncwarp();
                if (lane == 0) mbar_arrive(&b->full[r.s]);
            }
            if (second && ++step == first + per_head) {
                step = first;
                ++head;
            }
        }
    }
    // Every copy lands before the CTA may exit.
    __device__ __forceinline__ void drain(int lane) {
        if (lane != 0) return;
        for (int s = 0; s < kStages && s < it; ++s) drain_bar(&b->full[s], ((it - 1 - s) / kStages) & 1u);
        const int steps = (it + 1) / 2 + (left ? 1 : 0);
        for (int s = 0; kKeys && s < 2 && s < steps; ++s) drain_bar(&b->stat_full[s], ((steps - 1 - s) / 2) & 1u);
        drain_bar(&b->own, 0);
    }
};

// A whole warp: one lane per barrier.
__device__ __forceinline__ void init_barriers(Bars* b, bool aligned, int lane) {
    if (lane < kBarriers)
        mbar_init(reinterpret_cast<uint64_t*>(b) + lane, lane < kFourArrivals ? 1 : lane < kEightArrivals ? 4 : 8);
    if (lane == 0) {
        b->abort = !aligned;
        if (!aligned) atomicOr(&g_attn_fault, 2u);
    }
    fence_barrier_init();
    fence_proxy_async();
    __syncwarp();
}

// One barrier for the whole CTA, met by its roles at different places.
__device__ __forceinline__ void cta_sync() { asm volatile("bar.sync 0;" ::: "memory"); }

__global__ void __launch_bounds__(kThreads, 1) attn_bwd_kernel(const __grid_constant__ Maps m, const BwdArgs a) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Bars* b = reinterpret_cast<Bars*>(smem + kOffBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // Head-major order in both parts, so that the CTAs that run side by side share their streamed tiles
    // through L2; under a causal mask the longest of a head come first.
    const bool keys = (int)blockIdx.x < a.key_ctas;
    const unsigned part = keys ? blockIdx.x % (unsigned)a.parts : 0u;
    const unsigned id = keys ? blockIdx.x / (unsigned)a.parts : blockIdx.x - a.key_ctas;
    const unsigned bh = id / (unsigned)a.blocks, block = id - bh * a.blocks, heads = keys ? a.Hk : a.H;
    const int batch = (int)(bh / heads), head = (int)(bh - batch * heads);
    const int row0 = (int)(keys ? block : a.blocks - 1 - block) * kRows;

    // Only the statistics come from the kernel before this one: everything else may be read while that one drains.
    const int len = tokens_of(a.lens, batch, a.S);
    if (row0 >= len) {  // none of the CTA's rows belongs to the sequence
        pdl_wait();  // so that this grid never ends before the one ahead of it
        if (keys && a.parts > 1) return;
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
    const int all = keys ? a.group * per_head : per_head;
    const bool cut = keys && a.parts > 1;
    const int skip = cut ? (int)((int64_t)all * part / a.parts) : 0;
    const int n = cut ? (int)((int64_t)all * (part + 1) / a.parts) - skip : all;
    if (n == 0) {  // a part without steps: its sums are zero
        pdl_wait();
        for (int i = threadIdx.x; i < min(kRows, len - row0) * (kDim / 4); i += kThreads) {
            const int64_t at = (part * a.part_rows + ((int64_t)batch * a.Hk + head) * a.S + row0) * kDim + 4 * i;
            *reinterpret_cast<uint4*>(a.part_k + at) = *reinterpret_cast<uint4*>(a.part_v + at) =
                make_uint4(0u, 0u, 0u, 0u);
        }
        return;
    }
    const int tail = (first + per_head) * kStep > len && len < a.S ? len - (first + per_head - 1) * kStep : 0;
    // Some row's sum has fewer than kRows terms: queries that see few keys, keys few queries see.
    const bool pair = a.causal ? (keys ? row0 + 2 * kRows > len : row0 == 0) : len < kRows;

    // The control warpgroup gives its registers up before any softmax warp asks for them.
    if (warp >= kMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));

    // The producer sets up the barriers and sends for the first tiles before the CTA's first barrier; the tiles'
    // way to shared memory (1 to 2 us) then overlaps the allocation of the tensor memory.
    auto produce = [&](auto& p) {
        init_barriers(b, (smem_u32(smem) & 1023u) == 0, lane);  // the swizzled tiles need the alignment
        const bool issue = !b->abort;  // nobody else writes it before the CTA's first barrier
        if (lane == 0 && issue) {
            uint8_t* own = smem + kOffOwn;
            mbar_expect_tx(&b->own, keys ? 2 * kTileBytes : kTileBytes);
            load_tile(own, keys ? &m.k : &m.q, row0, head, batch, &b->own);
            if (keys) load_tile(own + kTileBytes, &m.v, row0, head, batch, &b->own);
        }
        __syncwarp();
        if (keys) pdl_wait();
        if (issue) p.run(2, true, lane);  // the first step
        __syncwarp();
        cta_sync();
        if (issue) {
            p.run(p.tiles, false, lane);
            p.drain(lane);
        }
    };
    if (warp == kLoadWarp) {
        if (keys) {
            Producer<true> p(&m.q, &m.go, smem, b, batch, head * a.group, first, per_head, skip, n, tail, a);
            produce(p);
        } else {
            Producer<false> p(&m.k, &m.v, smem, b, batch, head / a.group, 0, per_head, 0, n, tail, a);
            produce(p);
        }
        __syncwarp();
    } else {
        if (warp == kMmaWarp) {
            tc::tmem_alloc(&b->tmem_base, kTmemCols);
            tc::tmem_relinquish();
        }
        QueryRow own;
        if (warp < 8 && !keys) own.load(a, batch, head, len, row0);
        tc::fence_before();
        cta_sync();
        tc::fence_after();
        const uint32_t tmem = b->tmem_base;
        if (b->abort) {
            // nothing was issued
        } else if (warp < 8) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
            if (keys && pair) key_warps<true>(m, smem, b, tmem, a, batch, head, len, row0, first, per_head, skip, n, part);
            else if (keys) key_warps<false>(m, smem, b, tmem, a, batch, head, len, row0, first, per_head, skip, n, part);
            else if (pair) query_warps<true>(m, smem, b, tmem, a, own, batch, head, len, row0, n);
            else query_warps<false>(m, smem, b, tmem, a, own, batch, head, len, row0, n);
        } else if (warp == kMmaWarp) {
            if (tc::elect_one()) {
                if (keys) issue_key(smem, b, tmem, n, pair);
                else issue_query(smem, b, tmem, n, pair);
            }
            __syncwarp();
        }
    }
    tc::fence_before();
    cta_sync();
    if (warp == kMmaWarp) {
        tc::fence_after();
        tc::tmem_dealloc(b->tmem_base, kTmemCols);
    }
}

// dK and dV from the parts' sums, in part order; a warp per row, four columns a lane.
constexpr int kJoinRows = 8;
__global__ void __launch_bounds__(32 * kJoinRows) bwd_join_kernel(BwdArgs a) {
    pdl_wait();
    const int64_t row = (int64_t)blockIdx.x * kJoinRows + (threadIdx.x >> 5);
    if (row >= a.part_rows) return;
    const int lane = threadIdx.x & 31, i = (int)(row % a.S), head = (int)(row / a.S % a.Hk);
    const int batch = (int)(row / a.S / a.Hk);
    float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
    if (i < tokens_of(a.lens, batch, a.S))
        for (int p = 0; p < a.parts; ++p) {
            const int64_t at = ((p * a.part_rows + row) * kDim) / 4 + lane;
            const float4 x = reinterpret_cast<const float4*>(a.part_k)[at], y = reinterpret_cast<const float4*>(a.part_v)[at];
            k.x += x.x, k.y += x.y, k.z += x.z, k.w += x.w;
            v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
        }
    *reinterpret_cast<uint2*>(a.dk + offset(a.sdk, batch, head, i) + 4 * lane) =
        make_uint2(tc::pack_bf16(k.x * a.scale, k.y * a.scale), tc::pack_bf16(k.z * a.scale, k.w * a.scale));
    *reinterpret_cast<uint2*>(a.dv + offset(a.sdv, batch, head, i) + 4 * lane) =
        make_uint2(tc::pack_bf16(v.x, v.y), tc::pack_bf16(v.z, v.w));
}

SharedLimit g_shared;

int64_t padded(int64_t seq) { return (seq + kStep - 1) / kStep * kStep; }

// CTAs a key block is cut into, so that the longest runs about as long as an SM's share of all the work (within a
// quarter of it), and no fewer than 4 steps. Units of 0.57 us: a step of a key CTA takes 3, one of a query CTA 2, and every CTA about
// 9 or 8 besides (set-up, the way of the first tiles, the epilogue). bf16 causal [1, 32 heads on 1, 4096, 128]
// 1.59 ms uncut, 0.41 ms with 4 parts; [1, 8 on 1, 2048, 128] 207 and 62 us (76 us with
// 21 parts); not causal [1, 8 on 1, 8192, 128] 865 and 691 us (2 parts).
int parts_of(const nb200_attn_args& n) {
    const int64_t blocks = (n.seq + kRows - 1) / kRows, group = n.heads / n.kv_heads;
    const int64_t pairs = n.causal ? blocks * (blocks + 1) / 2 : blocks * blocks;  // (block, step) of one head
    const int64_t work = n.batch * (n.heads * (5 * pairs + 8 * blocks) + 9 * n.kv_heads * blocks);
    const int64_t share = std::max<int64_t>(work / sm_count(), 1), longest = 3 * group * blocks;
    return (int)std::max<int64_t>(1, std::min(group * blocks / 4, (4 * longest + 5 * share - 1) / (5 * share)));
}

}  // namespace

int attn_bwd_fault_take(unsigned int* bits) { return take_attn_fault(bits); }

int64_t attention_bwd_work_bytes(const nb200_attn_args& n) {
    const int64_t parts = parts_of(n);
    return 2 * (int64_t)sizeof(float) *
           (n.batch * n.heads * padded(n.seq) + (parts > 1 ? parts * n.batch * n.kv_heads * n.seq * kDim : 0));
}

int launch_attention_bwd(const nb200_attn_args& n, const nb200_attn_strides* strides, const void* q, const void* k,
                         const void* v, const void* o, const float* lse, const void* grad_o, void* dq, void* dk,
                         void* dv, void* work, cudaStream_t st) {
    const char* what = "nb200_attention_bwd";
    using B = __nv_bfloat16;
    const int64_t blocks = (n.seq + kRows - 1) / kRows, pad = padded(n.seq), rows = n.batch * n.heads * pad;
    const int64_t parts = parts_of(n), part_rows = n.batch * n.kv_heads * n.seq;
    const int64_t ctas = n.batch * (n.heads + n.kv_heads * parts) * blocks, stat_ctas = (rows + kStatRows - 1) / kStatRows;
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
        (rc = encode_rows(&m.dq, what, "dq", dq, n.batch, n.heads, n.seq, strides[5], 32)) ||
        (rc = encode_rows(&m.dk, what, "dk", dk, n.batch, n.kv_heads, n.seq, strides[6], 32)) ||
        (rc = encode_rows(&m.dv, what, "dv", dv, n.batch, n.kv_heads, n.seq, strides[7], 32)) ||
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
    a.parts = (int)parts;
    a.key_ctas = (int)(n.batch * n.kv_heads * blocks * parts);
    a.part_k = s.ndelta + rows;
    a.part_v = a.part_k + parts * part_rows * kDim;
    a.part_rows = part_rows;
    a.blocks = (int)blocks;
    a.causal = n.causal ? 1 : 0;
    a.scale = n.scale;
    a.sl2 = n.scale * 1.4426950408889634f;
    a.lens = n.seq_lens;
    a.go = static_cast<const B*>(grad_o);
    a.dq = static_cast<B*>(dq);
    a.dk = static_cast<B*>(dk);
    a.dv = static_cast<B*>(dv);
    a.sgo = strides[4];
    a.sdq = strides[5];
    a.sdk = strides[6];
    a.sdv = strides[7];
    a.nlse2 = s.nlse2;
    a.ndelta = s.ndelta;
    launch_pdl(attn_bwd_kernel, (unsigned)ctas, kThreads, kSmemBytes, st, m, a);
    count_launch(2);
    if (parts > 1) {
        launch_pdl(bwd_join_kernel, (unsigned)((part_rows + kJoinRows - 1) / kJoinRows), 32 * kJoinRows, 0, st, a);
        count_launch();
    }
    return finish_launch(what);
}

}  // namespace nb200
