// Fused single-pass attention forward, O = softmax(scale * Q K^T [+ masks]) V, bf16 in and out, fp32
// scores and online max/sum repair, on the sm_100a tensor cores. Query heads may share key/value
// heads; a batch element may hold fewer tokens than the tensors (the rest is masked).
//
// One CTA owns 256 query rows of one (batch, head): two query tiles of 128 rows, one tensor-memory
// lane per row. The K/V sequence streams through a ring of shared-memory stages filled by
// tensor-map (TMA) loads; one thread issues the tcgen05 MMAs; two softmax warpgroups, one per
// query tile, hold one query row per thread.
//
//   warp 9      producer: Q tiles once, then K_0, V_0, K_1, V_1, ... into the stage ring
//   warp 8      MMA: S_t = Q_t K_j^T (shared x shared -> TMEM, fp32)
//                    O_t += P_t V_j    (P from TMEM, V from shared -> TMEM, fp32)
//   warps 0-7   softmax for tile t = warp / 4: read S_t, update the running max (log2 domain),
//               rescale O_t in TMEM when the max grew by more than 2^8, write P_t = 2^(s - m)
//               as bf16 into the upper half of S_t's columns, accumulate the row sum;
//               at the end O_t / l -> bf16 -> shared -> TMA store, and the row's log-sum-exp.
//
// TMEM (512 columns x 128 lanes of 32 bits): S_0 [0,128), S_1 [128,256), O_0 [256,384),
// O_1 [384,512); P_t occupies columns [64,128) of S_t.
//
// MMA issue order per key tile j: PV_0(j), S_0(j+1), PV_1(j), S_1(j+1). tcgen05.commit arrives
// only when every earlier MMA of the issuing thread has finished, so the arrival of S_t(j+1)
// also means PV_t(j) is complete: the softmax warps may rescale O_t between reading S_t(j+1) and
// publishing P_t(j+1) without a separate barrier. S_t(j+1) overwrites the columns PV_t(j) reads
// P_t(j) from; the tensor pipe executes one thread's MMAs in issue order. Under a causal mask
// query tile 0 stops one key tile early: its rows end where tile 1's begin, so the unit's last key
// tile lies entirely above tile 0's diagonal.
//
// Every wait is bounded (about a second of SM clock). A wait that runs out sets bit 1 of the
// attention fault word and the CTA's abort flag; the other roles stop at their next wait, the
// producer waits for the copies it issued, the MMA thread waits for its MMAs, and the CTA frees
// its tensor memory and exits with the output unwritten.
#include "attn.cuh"

namespace nb200 {
namespace {

constexpr int kRows = 128;   // query rows per tile (= TMEM lanes)
constexpr int kQTiles = 2;   // query tiles per CTA
constexpr int kKeys = 128;   // keys per K/V tile
constexpr int kStages = 5;   // K/V ring stages; each holds one K or one V tile
constexpr uint32_t kTileBytes = kRows * kDim * 2;  // 32 KB per Q, K or V tile
constexpr uint32_t kHalfBytes = kTileBytes / 2;    // one 64-column half: the TMA box
constexpr int kMmaWarp = 8;
constexpr int kLoadWarp = 9;
constexpr int kThreads = 384;  // warps 10-11 only complete the third warpgroup for the register split
// Register split (setmaxnreg, per warpgroup): the softmax warpgroups hold a 128-column score row
// per thread; the MMA/producer warpgroup needs little. The sum stays within what the block is
// launched with (kThreads x kLaunchRegs), so the increase never waits on registers that do not exist.
constexpr int kLaunchRegs = 168;
constexpr int kRegsSoftmax = 216;
constexpr int kRegsControl = 72;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsControl <= kThreads * kLaunchRegs, "register split");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColS0 = 0, kColO0 = 256;  // tile t: S at kColS0 + 128 t, O at kColO0 + 128 t
constexpr uint32_t kColP = 64;                // P inside S's columns
// P is published in kPParts parts of 128 / kPParts keys; the MMA thread issues each part's P V
// steps as soon as that part is in TMEM. Two parts measured fastest (interleaved A/B on one box,
// non-causal: 2 parts 1059-1222, 4 parts 1001-1096, 8 parts 857-915 TFLOP/s): every further
// hand-off (store wait, fence, arrival, one more wait in the MMA thread) costs more than the extra
// overlap of the P V MMAs with the exponentials gains.
#ifndef NB200_ATTN_PPARTS
#define NB200_ATTN_PPARTS 2
#endif
constexpr int kPParts = NB200_ATTN_PPARTS;
constexpr int kPairsPerPart = 64 / kPParts;  // TMEM columns of P per part (two keys per column)
constexpr int kStepsPerPart = 8 / kPParts;   // K=16 P V MMA steps per part
static_assert(kPParts == 2 || kPParts == 4 || kPParts == 8, "P parts");
constexpr float kRescaleSlack = 8.f;          // keep a stale max while the new one is < 2^8 above it
constexpr uint32_t kIdescQK = tc::idesc_bf16(128, 128, false);
constexpr uint32_t kIdescPV = tc::idesc_bf16(128, 128, true);

// Shared-memory layout (offsets from a 1024-byte aligned base).
constexpr uint32_t kOffQ = 0;                                // kQTiles tiles
constexpr uint32_t kOffKV = kOffQ + kQTiles * kTileBytes;    // kStages tiles
constexpr uint32_t kOffBar = kOffKV + kStages * kTileBytes;  // mbarriers
struct Bars {
    uint64_t q_full[kQTiles];
    uint64_t kv_full[kStages];
    uint64_t kv_empty[kStages];
    uint64_t s_full[kQTiles];
    uint64_t p_full[kQTiles][kPParts];  // per part of P (128 / kPParts keys each)
    uint64_t o_final;
    uint64_t tail;  // the last V tile's copy, when rows of it are masked before it is published
    uint32_t tmem_base;
    int abort;
};
constexpr uint32_t kSmemBytes = kOffBar + sizeof(Bars) + 1024;  // + alignment slack

struct AttnArgs {
    int S;        // sequence length (queries = keys)
    int H;        // query heads
    int group;    // query heads that share a key/value head
    const int* lens;  // tokens of each batch element, nullable
    int64_t ob, oh, os;  // strides of o
    __nv_bfloat16* o;
    int nqb;      // query blocks of kQTiles * kRows rows per (batch, head)
    int causal;
    float sl2;    // scale * log2(e)
    float* lse;   // [BH, S] natural log-sum-exp, nullable
};

// P for part qp of this row's keys: p = 2^(s * sl2 - m) on the special-function unit,
// rounded to bf16 into TMEM (one column per key pair, the lower key in the low half), fp32 p added
// to the row sums. (Computing a share of the exponentials with an FMA-pipe polynomial instead was
// measured slower at every share tried, 2/8 to 5/8 of the pairs: the softmax warps run out of
// issue slots before the special-function unit saturates.)
template <int kPairs = kPairsPerPart>
__device__ __forceinline__ void p_part(const float* s, int qp, uint64_t sl2, uint64_t nm, uint64_t& acc0,
                                       uint64_t& acc1, uint32_t tP) {
    uint32_t pk[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
        const int pi = kPairs * qp + i;
        const uint64_t x = fma2(f2(s[2 * pi], s[2 * pi + 1]), sl2, nm);
        const uint64_t p = f2(ex2_ftz(f2lo(x)), ex2_ftz(f2hi(x)));
        if (i & 1)
            acc1 = add2(acc1, p);
        else
            acc0 = add2(acc0, p);
        pk[i] = tc::pack_bf16(f2lo(p), f2hi(p));
    }
    const uint32_t col = tP + kPairs * qp;
    if constexpr (kPairs == 32) {
        tc::tmem_st16(col, pk);
        tc::tmem_st16(col + 16, pk + 16);
    } else if constexpr (kPairs == 16) {
        tc::tmem_st16(col, pk);
    } else {
        tc::tmem_st8(col, pk);
    }
}

// The whole warp calls it; lane 0 issues. With tail > 0 only that many rows of the last V tile belong
// to the sequence: what lies past them is zeroed before the tile is published, because a masked
// probability of 0 times an infinity or NaN there would still poison the product.
__device__ __forceinline__ void producer(const CUtensorMap* mq, const CUtensorMap* mk, const CUtensorMap* mv,
                                         uint8_t* smem, Bars* b, int head, int kv_head, int batch, int q0, int n,
                                         int tail, int lane) {
    volatile int* abort = &b->abort;
    if (lane == 0) {
        tc::prefetch_map(mq);
        tc::prefetch_map(mk);
        tc::prefetch_map(mv);
        for (int t = 0; t < kQTiles; ++t) {
            uint8_t* dst = smem + kOffQ + t * kTileBytes;
            mbar_expect_tx(&b->q_full[t], kTileBytes);
            tc::tma_load_4d(dst, mq, 0, q0 + t * kRows, head, batch, &b->q_full[t]);
            tc::tma_load_4d(dst + kHalfBytes, mq, kDim / 2, q0 + t * kRows, head, batch, &b->q_full[t]);
        }
    }
    auto load = [&](int it, int s, uint64_t* bar) {
        uint8_t* dst = smem + kOffKV + s * kTileBytes;
        const CUtensorMap* m = (it & 1) ? mv : mk;
        const int row = (it >> 1) * kKeys;
        mbar_expect_tx(bar, kTileBytes);
        tc::tma_load_4d(dst, m, 0, row, kv_head, batch, bar);
        tc::tma_load_4d(dst + kHalfBytes, m, kDim / 2, row, kv_head, batch, bar);
    };
    int it = 0;
    Ring<kStages> r;
    bool ok = true;
    for (const int whole = tail ? 2 * n - 1 : 2 * n; it < whole; ++it, r.next()) {
        ok = lane != 0 || wait_bar(&b->kv_empty[r.s], r.ph ^ 1u, abort);
        if (!ok) break;
        if (lane == 0) load(it, r.s, &b->kv_full[r.s]);
    }
    ok = __all_sync(0xffffffffu, ok);
    if (tail && ok) {
        ok = lane != 0 || wait_bar(&b->kv_empty[r.s], r.ph ^ 1u, abort);
        if (lane == 0 && ok) load(it, r.s, &b->tail);
        const bool sent = __all_sync(0xffffffffu, ok);
        ok = sent && __all_sync(0xffffffffu, wait_bar(&b->tail, 0, abort));
        if (sent && !ok && lane == 0) drain_bar(&b->tail, 0);
        if (ok) {
            zero_tail(smem + kOffKV + r.s * kTileBytes, kKeys, tail, lane);
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->kv_full[r.s]);
            ++it;
        }
    }
    // Every copy issued into this CTA's shared memory lands before the CTA may exit: wait for the
    // last phase filled in each stage (`it` tiles were issued, stage s got those with index = s
    // mod kStages).
    if (lane == 0) {
        for (int t = 0; t < kQTiles; ++t) drain_bar(&b->q_full[t], 0);
        for (int s = 0; s < kStages && s < it; ++s) drain_bar(&b->kv_full[s], ((it - 1 - s) / kStages) & 1u);
    }
}

// n K/V tiles in the unit; query tile 0 uses the first n0 of them (n0 = n, or n - 1 under a causal
// mask, where tile 0's rows end 128 keys before tile 1's).
__device__ __forceinline__ void mma_issuer(uint8_t* smem, Bars* b, uint32_t tmem, int n0, int n) {
    volatile int* abort = &b->abort;
    // Descriptors are built once; an operand step only adds its byte offset / 16 to the start-
    // address field (bits 0-13, which cannot carry: shared addresses stay below 2^18 bytes).
    const uint64_t q_desc = tc::sw128_desc(smem_u32(smem + kOffQ), 16, 1024);
    const uint64_t k_desc = tc::sw128_desc(smem_u32(smem + kOffKV), 16, 1024);
    const uint64_t v_desc = tc::sw128_desc(smem_u32(smem + kOffKV), kHalfBytes, 1024);
    // S_t = Q_t K^T: eight K=16 steps along the head dimension; 32 bytes per step inside a
    // 128-byte swizzled row, the second 64 columns in the other half tile.
    auto qk = [&](int t, int s) {
        const uint64_t qa = q_desc + ((t * kTileBytes) >> 4), ka = k_desc + ((s * kTileBytes) >> 4);
        const uint32_t d = tmem + kColS0 + 128 * t;
        constexpr uint32_t h = kHalfBytes >> 4;  // second 64 head columns
        tc::mma_ss_at<0>(d, qa, ka, kIdescQK, 0u);
        tc::mma_ss_at<2>(d, qa, ka, kIdescQK, 1u);
        tc::mma_ss_at<4>(d, qa, ka, kIdescQK, 1u);
        tc::mma_ss_at<6>(d, qa, ka, kIdescQK, 1u);
        tc::mma_ss_at<h + 0>(d, qa, ka, kIdescQK, 1u);
        tc::mma_ss_at<h + 2>(d, qa, ka, kIdescQK, 1u);
        tc::mma_ss_at<h + 4>(d, qa, ka, kIdescQK, 1u);
        tc::mma_ss_at<h + 6>(d, qa, ka, kIdescQK, 1u);
    };
    // O_t += P_t V: eight K=16 steps along the keys; P from TMEM (8 columns per step), V as an
    // MN-major operand (head dimension contiguous, 16 key rows = 2048 bytes per step, the second
    // 64 head columns 16 KB further).
    // One K=16 step k of O_t += P_t V (compile-time k after unrolling).
    auto pv_step = [&](int k, uint32_t d, uint32_t pa, uint64_t va, uint32_t acc) {
        switch (k) {
            case 0: tc::mma_ts_at<0, 0>(d, pa, va, kIdescPV, acc); break;
            case 1: tc::mma_ts_at<8, 128>(d, pa, va, kIdescPV, acc); break;
            case 2: tc::mma_ts_at<16, 256>(d, pa, va, kIdescPV, acc); break;
            case 3: tc::mma_ts_at<24, 384>(d, pa, va, kIdescPV, acc); break;
            case 4: tc::mma_ts_at<32, 512>(d, pa, va, kIdescPV, acc); break;
            case 5: tc::mma_ts_at<40, 640>(d, pa, va, kIdescPV, acc); break;
            case 6: tc::mma_ts_at<48, 768>(d, pa, va, kIdescPV, acc); break;
            default: tc::mma_ts_at<56, 896>(d, pa, va, kIdescPV, acc); break;
        }
    };
    // Issued part by part, each as soon as the softmax warps publish that part of P.
    auto pv_tile = [&](int t, int s, bool acc, uint32_t parity) {
        const uint64_t va = v_desc + ((s * kTileBytes) >> 4);
        const uint32_t d = tmem + kColO0 + 128 * t, pa = tmem + kColS0 + 128 * t + kColP;
#pragma unroll
        for (int qp = 0; qp < kPParts; ++qp) {
            if (!wait_bar(&b->p_full[t][qp], parity, abort)) return false;
            tc::fence_after();
#pragma unroll
            for (int kk = 0; kk < kStepsPerPart; ++kk) {
                const int k = qp * kStepsPerPart + kk;
                pv_step(k, d, pa, va, (acc || k > 0) ? 1u : 0u);
            }
        }
        return true;
    };
    // kr: the next K tile's stage, vr: the next V tile's stage (tiles alternate K_0, V_0, K_1, ...).
    Ring<kStages> kr, vr;
    vr.next();
    bool ok = wait_bar(&b->q_full[0], 0, abort) && wait_bar(&b->q_full[1], 0, abort) &&
              wait_bar(&b->kv_full[kr.s], kr.ph, abort);
    if (ok) {
        tc::fence_after();
        qk(0, kr.s);
        tc::commit(&b->s_full[0]);
        qk(1, kr.s);
        tc::commit(&b->s_full[1]);
        tc::commit(&b->kv_empty[kr.s]);
        kr.next();
        kr.next();
    }
    for (int j = 0; ok && j < n; ++j) {
        const bool more = j + 1 < n;
        if (!(ok = wait_bar(&b->kv_full[vr.s], vr.ph, abort))) break;
        if (j < n0 && !(ok = pv_tile(0, vr.s, j > 0, j & 1u))) break;
        if (more) {
            if (!(ok = wait_bar(&b->kv_full[kr.s], kr.ph, abort))) break;
            tc::fence_after();
            if (j + 1 < n0) {
                qk(0, kr.s);
                tc::commit(&b->s_full[0]);
            }
        }
        if (!(ok = pv_tile(1, vr.s, j > 0, j & 1u))) break;
        tc::commit(&b->kv_empty[vr.s]);
        vr.next();
        vr.next();
        if (more) {
            qk(1, kr.s);
            tc::commit(&b->s_full[1]);
            tc::commit(&b->kv_empty[kr.s]);
            kr.next();
            kr.next();
        }
    }
    // Arrives when every MMA above has finished (at once if none was issued).
    tc::commit(&b->o_final);
    drain_bar(&b->o_final, 0);
}

__device__ __forceinline__ void softmax_tile(const CUtensorMap* mo, uint8_t* smem, Bars* b, uint32_t tmem,
                                             const AttnArgs& a, int head, int batch, int len, int q0, int n) {
    volatile int* abort = &b->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = warp >> 2, wq = warp & 3;
    const int r = wq * 32 + lane;  // row inside the tile = TMEM lane
    const int qrow = q0 + t * kRows + r;
    const int lim = a.causal ? min(qrow, len - 1) : len - 1;  // last key this row attends to
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lanes + kColS0 + 128 * t;
    const uint32_t tP = tS + kColP;
    const uint32_t tO = tmem + lanes + kColO0 + 128 * t;
    const float sl2 = a.sl2;
    float m = -NB200_INF, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; ++j) {
        // All lanes take the same branch: the TMEM accesses below are warp-collective.
        if (!(ok = __all_sync(0xffffffffu, wait_bar(&b->s_full[t], j & 1u, abort)))) break;
        tc::fence_after();
        uint32_t u[128];
        tc::tmem_ld128(tS, u);
        float s[128];
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = __uint_as_float(u[c]);
        const int kb = j * kKeys;
        // Warp-uniform: the tile holds a key past some row's last (causal diagonal, ragged end).
        const bool masked = __any_sync(0xffffffffu, kb + kKeys - 1 > lim);
        if (masked) {
#pragma unroll
            for (int c = 0; c < 128; ++c)
                if (kb + c > lim) s[c] = -NB200_INF;
        }
        float a0 = s[0], a1 = s[1], a2 = s[2], a3 = s[3];
#pragma unroll
        for (int c = 4; c < 124; c += 8) {
            a0 = max3(a0, s[c], s[c + 1]);
            a1 = max3(a1, s[c + 2], s[c + 3]);
            a2 = max3(a2, s[c + 4], s[c + 5]);
            a3 = max3(a3, s[c + 6], s[c + 7]);
        }
        a0 = max3(a0, s[124], s[125]);
        a1 = max3(a1, s[126], s[127]);
        const float mnew = fmaxf(m, fmaxf(max3(a0, a1, a2), a3) * sl2);
        const bool grow = mnew > m + kRescaleSlack;
        if (__any_sync(0xffffffffu, grow)) {
            // Move the whole warp to the new maxima; rows whose max did not move keep factor 1.
            const float f = (mnew == m) ? 1.f : ex2(m - mnew);
            if (j > 0) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tc::tmem_ld32(tO + 32 * c, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                    tc::tmem_st32(tO + 32 * c, v);
                }
            }
            l *= f;
            m = mnew;
        }
        const uint64_t sl2x2 = f2(sl2, sl2), nm = f2(-m, -m);
        uint64_t acc0 = 0, acc1 = 0;  // packed fp32 partial row sums (+0.0 bit patterns)
#pragma unroll
        for (int qp = 0; qp < kPParts; ++qp) {
            p_part(s, qp, sl2x2, nm, acc0, acc1, tP);
            tc::tmem_wait_st();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b->p_full[t][qp]);
        }
        const uint64_t acc = add2(acc0, acc1);
        l += f2lo(acc) + f2hi(acc);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_bar(&b->o_final, 0, abort));
    if (!ok) return;
    tc::fence_after();
    // Epilogue: O / l in bf16, written into this tile's (now idle) Q buffer in the swizzled layout
    // the O tensor map expects, then one TMA store per warp for its 32 rows.
    uint8_t* stage = smem + kOffQ + t * kTileBytes;
    const float inv = 1.f / l;
    const bool live = qrow < len;  // rows past the sequence read out as zero, whatever q held there
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        tc::tmem_ld32(tO + 32 * c, v);
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            pk[i] = live ? tc::pack_bf16(__uint_as_float(v[2 * i]) * inv, __uint_as_float(v[2 * i + 1]) * inv) : 0u;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int ch = 4 * c + q;  // 16-byte chunk of the 256-byte row
            uint8_t* dst = stage + (ch >> 3) * kHalfBytes + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
            *reinterpret_cast<uint4*>(dst) = make_uint4(pk[4 * q], pk[4 * q + 1], pk[4 * q + 2], pk[4 * q + 3]);
        }
    }
    if (a.lse && qrow < a.S)
        a.lse[((size_t)batch * a.H + head) * a.S + qrow] = live ? (m + log2f(l)) * 0.69314718055994531f : -NB200_INF;
    fence_proxy_async();
    __syncwarp();
    const int row0 = q0 + t * kRows + wq * 32;
    if (lane == 0 && row0 < a.S) {
        tc::tma_store_4d(mo, stage + wq * 32 * 128, 0, row0, head, batch);
        tc::tma_store_4d(mo, stage + kHalfBytes + wq * 32 * 128, kDim / 2, row0, head, batch);
        tc::bulk_commit();
        tc::bulk_wait_read();
    }
    __syncwarp();
}

__global__ void __launch_bounds__(kThreads, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                    const __grid_constant__ CUtensorMap mv, const __grid_constant__ CUtensorMap mo, AttnArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* b = reinterpret_cast<Bars*>(smem + kOffBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // Head-major order: the query blocks of one (batch, head) run side by side and share its K/V
    // through L2, so each head's K/V is read from HBM about once. Within a head the longest causal
    // blocks go first.
    const int bh = (int)(blockIdx.x / (unsigned)a.nqb);
    const int qb = a.nqb - 1 - (int)(blockIdx.x % (unsigned)a.nqb);
    const int q0 = qb * kQTiles * kRows;
    const int batch = bh / a.H, head = bh % a.H;
    const int len = tokens_of(a.lens, batch, a.S);
    if (q0 >= len) {  // no query of this block belongs to the sequence
        const int rows = min(kQTiles * kRows, a.S - q0);
        for (int i = threadIdx.x; i < rows * (kDim / 8); i += kThreads)
            *reinterpret_cast<uint4*>(a.o + batch * a.ob + head * a.oh + (q0 + i / (kDim / 8)) * a.os +
                                      i % (kDim / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
        if (a.lse)
            for (int i = threadIdx.x; i < rows; i += kThreads) a.lse[(size_t)bh * a.S + q0 + i] = -NB200_INF;
        return;
    }
    const int kv_end = a.causal ? min(q0 + kQTiles * kRows, len) : len;
    const int n = (kv_end + kKeys - 1) / kKeys;
    // Query tile 0 of a causal unit ends 128 rows earlier: its last K/V tile would be fully masked.
    const int n0 = a.causal ? (min(q0 + kRows, len) + kKeys - 1) / kKeys : n;
    // Rows of the last V tile inside the sequence, when the tensor holds more rows past them.
    const int tail = n * kKeys > len && len < a.S ? len - (n - 1) * kKeys : 0;

    if (threadIdx.x == 0) {
        for (int t = 0; t < kQTiles; ++t) {
            mbar_init(&b->q_full[t], 1);
            mbar_init(&b->s_full[t], 1);
            for (int qp = 0; qp < kPParts; ++qp) mbar_init(&b->p_full[t][qp], 4);  // one arrival per softmax warp
        }
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&b->kv_full[s], 1);
            mbar_init(&b->kv_empty[s], 1);
        }
        mbar_init(&b->o_final, 1);
        mbar_init(&b->tail, 1);
        b->abort = 0;
        fence_barrier_init();
    }
    if (warp == kMmaWarp) {
        tc::tmem_alloc(&b->tmem_base, kTmemCols);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = b->tmem_base;

    // Each role runs to the end of the kernel in its own branch (the register budget differs per
    // branch); both end at barrier 0, after which the MMA warp frees the tensor memory.
    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        softmax_tile(&mo, smem, b, tmem, a, head, batch, len, q0, warp < 4 ? n0 : n);
        tc::fence_before();
        asm volatile("bar.sync 0;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if (warp == kLoadWarp) {
            producer(&mq, &mk, &mv, smem, b, head, head / a.group, batch, q0, n, tail, lane);
            __syncwarp();
        } else if (warp == kMmaWarp) {
            if (tc::elect_one()) mma_issuer(smem, b, tmem, n0, n);
            __syncwarp();
        }
        tc::fence_before();
        asm volatile("bar.sync 0;" ::: "memory");
        if (warp == kMmaWarp) {
            tc::fence_after();
            tc::tmem_dealloc(tmem, kTmemCols);
        }
    }
}

// ------------------------------------------------------------------ host side
PFN_cuTensorMapEncodeTiled_v12000 g_encode = nullptr;
std::once_flag g_encode_once;
SharedLimit g_shared;

}  // namespace

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder(const char* what) {
    std::call_once(g_encode_once, [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            g_encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
        cudaGetLastError();
    });
    if (!g_encode) set_error("%s: the driver does not provide cuTensorMapEncodeTiled", what);
    return g_encode;
}

int attn_fault_take(unsigned int* bits) { return take_attn_fault(bits); }

int launch_attention(const nb200_attn_args& n, const nb200_attn_strides* strides, const void* q, const void* k,
                     const void* v, void* o, float* lse, cudaStream_t st) {
    const char* what = "nb200_attention";
    const int64_t nqb = (n.seq + kQTiles * kRows - 1) / (kQTiles * kRows);
    if (n.batch * n.heads * nqb > 0x7fffffffLL) {
        set_error("%s: batch*heads=%lld, seq=%lld exceed the kernel's index range", what,
                  (long long)(n.batch * n.heads), (long long)n.seq);
        return NB200_ERR_CAPACITY;
    }
    CUtensorMap mq, mk, mv, mo;
    int rc;
    if ((rc = encode_rows(&mq, what, "q", q, n.batch, n.heads, n.seq, strides[0], kRows)) ||
        (rc = encode_rows(&mk, what, "k", k, n.batch, n.kv_heads, n.seq, strides[1], kKeys)) ||
        (rc = encode_rows(&mv, what, "v", v, n.batch, n.kv_heads, n.seq, strides[2], kKeys)) ||
        (rc = encode_rows(&mo, what, "o", o, n.batch, n.heads, n.seq, strides[3], 32)))
        return rc;
    if ((rc = g_shared.raise(what, attn_fwd_kernel, kSmemBytes))) return rc;
    AttnArgs a;
    a.S = (int)n.seq;
    a.H = (int)n.heads;
    a.group = (int)(n.heads / n.kv_heads);
    a.lens = n.seq_lens;
    a.ob = strides[3].batch;
    a.oh = strides[3].head;
    a.os = strides[3].seq;
    a.o = static_cast<__nv_bfloat16*>(o);
    a.nqb = (int)nqb;
    a.causal = n.causal ? 1 : 0;
    a.sl2 = n.scale * 1.4426950408889634f;
    a.lse = lse;
    attn_fwd_kernel<<<(unsigned)(n.batch * n.heads * nqb), kThreads, kSmemBytes, st>>>(mq, mk, mv, mo, a);
    count_launch();
    return finish_launch("nb200_attention");
}

}  // namespace nb200
