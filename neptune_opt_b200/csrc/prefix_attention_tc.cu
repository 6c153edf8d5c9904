// The shared prefix on the tensor cores: softmax(scale Q K^T) V of many query rows against a range of the
// prefix's keys, with the range's maximum and sum (one part of prefix_attention.cu).
//
// One CTA owns up to 256 query rows of one key/value head, gathered from all sequences, and a range of 128-key
// tiles. Two softmax warpgroups each own a stream: a 128-row query tile with its scores and output in tensor
// memory, one row per thread. With more than 128 rows the streams are two query tiles that share every K/V
// tile; with fewer they are the same query tile on alternate K/V tiles, and their results are merged at the
// end, so that both warpgroups work whatever the number of rows.
//
//   warp 9      producer: K and V tiles through a ring of stages (TMA), in the order in which they are used
//   warp 8      MMA: S_t = Q K^T (shared x shared -> TMEM, fp32), O_t += P_t V (P from TMEM, V from shared)
//   warps 0-7   softmax of stream t = warp / 4: scores, running maximum, rescale O_t when the
//               maximum grew by more than 2^8, P_t in the inputs' type into the upper half of S_t's columns
//
// TMEM (512 columns x 128 lanes): S_0 [0, 128), S_1 [128, 256), O_0 [256, 256 + D), O_1 [384, 384 + D).
// tcgen05.commit arrives once all earlier MMAs of the issuing thread are done, so the arrival of S_t's next
// scores also says that the last P_t V is complete, and O_t may be rescaled. S_t's next scores overwrite the
// columns the last P_t was read from: one thread's MMAs execute in issue order.
//
// Every wait is bounded; one that runs out sets bit 1 of the fault word and the CTA's abort flag, the producer
// waits for its copies, the MMA thread for its products, and the CTA frees its tensor memory and ends with NaN in its
// part's sums.
#include <algorithm>

#include "attn.cuh"
#include "prefix_attention.cuh"

namespace nb200 {
namespace prefix {
namespace {

constexpr int kRows = 128;  // query rows per tile (= TMEM lanes)
constexpr int kKeys = 128;  // keys per K/V tile
constexpr int kMmaWarp = 8, kLoadWarp = 9;
constexpr int kThreads = 384;  // warps 10-11 only complete the third warpgroup for the register split
constexpr int kLaunchRegs = 168, kRegsSoftmax = 216, kRegsControl = 72;
static_assert(2 * 128 * kRegsSoftmax + 128 * kRegsControl <= kThreads * kLaunchRegs, "register split");
constexpr uint32_t kTmemCols = 512, kColS = 0, kColO = 256, kColP = 64;

template <int D> struct Shape {
    static constexpr uint32_t kTile = kKeys * D * 2;             // a Q, K or V tile
    static constexpr uint32_t kHalf = kKeys * 128;               // 64 of its columns: a TMA box
    static constexpr int kHalves = D / 64;
    static constexpr int kStages = D == 128 ? 5 : 8;
    static constexpr uint32_t kOffKV = 2 * kTile;                // behind the two query tiles
    static constexpr uint32_t kOffBar = kOffKV + kStages * kTile;
};

struct Bars {
    uint64_t q_full;
    uint64_t kv_full[8], kv_empty[8];
    uint64_t s_full[2], p_full[2][2];  // P is published in two halves of 64 keys
    uint64_t o_final;
    uint32_t tmem_base;
    int abort;
    float m[kRows], l[kRows];  // of stream 1, for the merge
};
template <int D> constexpr uint32_t kSmem = Shape<D>::kOffBar + sizeof(Bars) + 1024;  // + alignment slack

template <typename T> constexpr uint32_t idesc(uint32_t n, bool b_mn_major) {
    const uint32_t bf16 = tc::idesc_bf16(128, n, b_mn_major);
    return std::is_same<T, __half>::value ? bf16 & ~((1u << 7) | (1u << 10)) : bf16;  // a and b format F16 = 0
}

template <typename T>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    if constexpr (std::is_same<T, __half>::value) {
        uint32_t r;
        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        return r;
    } else {
        return tc::pack_bf16(lo, hi);
    }
}

// What a CTA does: `pair` streams share n tiles, or the streams take tiles 0, 2, .. and 1, 3, .. of them.
struct Unit {
    int head, row0, nrows, tile0, n;
    bool pair;
    __device__ __forceinline__ int tiles_of(int t) const { return pair ? n : (n + 1 - t) / 2; }
};

// K_0 (and K_1 where the streams alternate), then V_j followed by the next K that a stream waits for.
template <int D>
__device__ __forceinline__ void producer(const CUtensorMap* mk, const CUtensorMap* mv, uint8_t* smem, Bars* b,
                                         const Unit& u) {
    using S = Shape<D>;
    volatile int* abort = &b->abort;
    tc::prefetch_map(mk);
    tc::prefetch_map(mv);
    Ring<S::kStages> r;
    int issued = 0;
    auto load = [&](const CUtensorMap* m, int j) {
        if (!wait_bar(&b->kv_empty[r.s], r.ph ^ 1u, abort)) return false;
        uint8_t* dst = smem + S::kOffKV + r.s * S::kTile;
        mbar_expect_tx(&b->kv_full[r.s], S::kTile);
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
            tc::tma_load_4d(dst + h * S::kHalf, m, 64 * h, (u.tile0 + j) * kKeys, u.head, 0, &b->kv_full[r.s]);
        r.next();
        ++issued;
        return true;
    };
    const int ahead = u.pair ? 1 : 2;
    bool ok = true;
    for (int j = 0; ok && j < ahead && j < u.n; ++j) ok = load(mk, j);
    for (int j = 0; ok && j < u.n; ++j) {
        ok = load(mv, j);
        if (ok && j + ahead < u.n) ok = load(mk, j + ahead);
    }
    // Every copy lands before the CTA may exit: the last fill of each stage.
    for (int s = 0; s < S::kStages && s < issued; ++s) drain_bar(&b->kv_full[s], ((issued - 1 - s) / S::kStages) & 1u);
}

template <typename T, int D>
__device__ __forceinline__ void mma_issuer(uint8_t* smem, Bars* b, uint32_t tmem, const Unit& u) {
    using S = Shape<D>;
    constexpr uint32_t kQK = idesc<T>(128, false), kPV = idesc<T>(D, true);
    volatile int* abort = &b->abort;
    // Descriptors are built once; a step adds its byte offset / 16 to the start-address field.
    const uint64_t q_desc = tc::sw128_desc(smem_u32(smem), 16, 1024);
    const uint64_t k_desc = tc::sw128_desc(smem_u32(smem + S::kOffKV), 16, 1024);
    const uint64_t v_desc = tc::sw128_desc(smem_u32(smem + S::kOffKV), S::kHalf, 1024);
    Ring<S::kStages> r;
    // S_t = Q K^T: K=16 steps along the head dimension, 32 bytes each inside a 128-byte swizzled row.
    auto scores = [&](int t) {
        const uint64_t qa = q_desc + ((u.pair ? t * S::kTile : 0u) >> 4), ka = k_desc + ((r.s * S::kTile) >> 4);
        const uint32_t d = tmem + kColS + 128 * t;
        tc::mma_ss_at<0>(d, qa, ka, kQK, 0u);
        tc::mma_ss_at<2>(d, qa, ka, kQK, 1u);
        tc::mma_ss_at<4>(d, qa, ka, kQK, 1u);
        tc::mma_ss_at<6>(d, qa, ka, kQK, 1u);
        if constexpr (D == 128) {
            constexpr uint32_t h = S::kHalf >> 4;  // second 64 head columns
            tc::mma_ss_at<h + 0>(d, qa, ka, kQK, 1u);
            tc::mma_ss_at<h + 2>(d, qa, ka, kQK, 1u);
            tc::mma_ss_at<h + 4>(d, qa, ka, kQK, 1u);
            tc::mma_ss_at<h + 6>(d, qa, ka, kQK, 1u);
        }
        tc::commit(&b->s_full[t]);
    };
    // O_t += P_t V: K=16 steps along the keys (8 TMEM columns of P, 16 rows of V), half by half as P comes.
    auto values = [&](int t, int i) {
        const uint64_t va = v_desc + ((r.s * S::kTile) >> 4);
        const uint32_t d = tmem + kColO + 128 * t, pa = tmem + kColS + 128 * t + kColP;
        if (!wait_bar(&b->p_full[t][0], i & 1u, abort)) return false;
        tc::fence_after();
        tc::mma_ts_at<0, 0>(d, pa, va, kPV, i > 0);
        tc::mma_ts_at<8, 128>(d, pa, va, kPV, 1u);
        tc::mma_ts_at<16, 256>(d, pa, va, kPV, 1u);
        tc::mma_ts_at<24, 384>(d, pa, va, kPV, 1u);
        if (!wait_bar(&b->p_full[t][1], i & 1u, abort)) return false;
        tc::fence_after();
        tc::mma_ts_at<32, 512>(d, pa, va, kPV, 1u);
        tc::mma_ts_at<40, 640>(d, pa, va, kPV, 1u);
        tc::mma_ts_at<48, 768>(d, pa, va, kPV, 1u);
        tc::mma_ts_at<56, 896>(d, pa, va, kPV, 1u);
        return true;
    };
    auto arrived = [&] {
        const bool ok = wait_bar(&b->kv_full[r.s], r.ph, abort);
        tc::fence_after();
        return ok;
    };
    auto release = [&] {
        tc::commit(&b->kv_empty[r.s]);
        r.next();
    };
    bool ok = wait_bar(&b->q_full, 0, abort);
    if (!ok) {
    } else if (u.pair) {
        if ((ok = arrived())) {
            scores(0);
            scores(1);
            release();
        }
        for (int j = 0; ok && j < u.n; ++j) {
            // The stage of V_j, and behind it that of K_{j+1}.
            if (!(ok = arrived() && values(0, j))) break;
            const bool more = j + 1 < u.n;
            const Ring<S::kStages> vr = r;
            if (more) {
                r.next();
                if (!(ok = arrived())) break;
                scores(0);
            }
            const Ring<S::kStages> kr = r;
            r = vr;
            if (!(ok = values(1, j))) break;
            release();
            if (more) {
                r = kr;
                scores(1);
                release();
            }
        }
    } else {
        for (int j = 0; ok && j < 2 && j < u.n; ++j)
            if ((ok = arrived())) {
                scores(j);
                release();
            }
        for (int j = 0; ok && j < u.n; ++j) {
            if (!(ok = arrived() && values(j & 1, j >> 1))) break;
            release();
            if (j + 2 < u.n) {
                if (!(ok = arrived())) break;
                scores(j & 1);
                release();
            }
        }
    }
    // Arrives when every MMA above has finished (at once if none was issued).
    tc::commit(&b->o_final);
    drain_bar(&b->o_final, 0);
}

// While |m sl2| is at most kFar the exponent takes one multiply-add here, 2^(s sl2 - m sl2), from which the rounding of m sl2
// takes 2^-16 at most; a warp with a row that is farther from 0 subtracts first. (Subtracting always spills, and takes 80 us
// for 77 over 16384 keys and 1024 rows a head.)
constexpr float kFar = 256.f;
__device__ __forceinline__ bool is_far(float m, float sl2) { return m != -NB200_INF && fabsf(m * sl2) > kFar; }

// Half qp of P for this row: p = 2^(s sl2 + nm), FAR: 2^((s - m) sl2 + nm), rounded into TMEM, its fp32 value added to the
// row sums.
template <typename T, bool FAR>
__device__ __forceinline__ void p_half(const float* s, int qp, uint64_t minus_m, uint64_t sl2, uint64_t nm, uint64_t& acc0,
                                       uint64_t& acc1, uint32_t tP) {
    uint32_t pk[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int pi = 32 * qp + i;
        uint64_t x = f2(s[2 * pi], s[2 * pi + 1]);
        if constexpr (FAR) x = add2(x, minus_m);
        x = fma2(x, sl2, nm);
        const uint64_t p = f2(ex2_ftz(f2lo(x)), ex2_ftz(f2hi(x)));
        if (i & 1) acc1 = add2(acc1, p);
        else acc0 = add2(acc0, p);
        pk[i] = pack<T>(f2lo(p), f2hi(p));
    }
    tc::tmem_st16(tP + 32 * qp, pk);
    tc::tmem_st16(tP + 32 * qp + 16, pk + 16);
}

template <typename T, int D>
__device__ __forceinline__ void softmax_stream(uint8_t* smem, Bars* b, uint32_t tmem, const TensorPart& a, const Unit& u,
                                               int split) {
    volatile int* abort = &b->abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = warp >> 2, wq = warp & 3;
    const int r = wq * 32 + lane;  // row inside the tile = TMEM lane
    const uint32_t lanes = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lanes + kColS + 128 * t, tP = tS + kColP, tO = tmem + lanes + kColO + 128 * t;
    const float sl2 = a.sl2;
    const int n = u.tiles_of(t);
    float m = -NB200_INF, l = 0.f, add = kLift<T>;  // add: what the exponent gets beside s sl2
    bool ok = true, far = false;  // far: a maximum of the warp is
    for (int i = 0; i < n; ++i) {
        // All lanes take the same branch: the TMEM accesses below are warp-collective.
        if (!(ok = __all_sync(0xffffffffu, wait_bar(&b->s_full[t], i & 1u, abort)))) break;
        tc::fence_after();
        uint32_t v[128];
        tc::tmem_ld128(tS, v);
        float s[128];
#pragma unroll
        for (int c = 0; c < 128; ++c) s[c] = __uint_as_float(v[c]);
        const int kb = (u.tile0 + (u.pair ? i : 2 * i + t)) * kKeys;
        if (kb + kKeys > a.keys) {  // the prefix ends inside the tile
#pragma unroll
            for (int c = 0; c < 128; ++c)
                if (kb + c >= a.keys) s[c] = -NB200_INF;
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
        const float mnew = fmaxf(m, fmaxf(max3(a0, a1, a2), a3));
        if (__any_sync(0xffffffffu, mnew > m + a.slack)) {
            // Move the whole warp to the new maxima; rows whose maximum did not move keep factor 1.
            const float f = mnew == m ? 1.f : ex2((m - mnew) * sl2);
            if (i > 0) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tc::tmem_ld32(tO + 32 * c, o);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                    tc::tmem_st32(tO + 32 * c, o);
                }
            }
            l *= f;
            m = mnew;
            add = kLift<T> - (m == -NB200_INF ? 0.f : m * sl2);  // no score but -inf so far: all p are 0
            far = __any_sync(0xffffffffu, is_far(m, sl2));
        }
        const uint64_t sl2x2 = f2(sl2, sl2);
        uint64_t acc0 = 0, acc1 = 0;
        auto probabilities = [&](auto is) {
            constexpr bool FAR = decltype(is)::value;
            const float top = m == -NB200_INF ? 0.f : m, x = FAR ? kLift<T> : add;
#pragma unroll
            for (int qp = 0; qp < 2; ++qp) {
                p_half<T, FAR>(s, qp, f2(-top, -top), sl2x2, f2(x, x), acc0, acc1, tP);
                tc::tmem_wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&b->p_full[t][qp]);
            }
        };
        if (__builtin_expect(far, 0)) probabilities(std::true_type{});
        else probabilities(std::false_type{});
        const uint64_t acc = add2(acc0, acc1);
        l += f2lo(acc) + f2hi(acc);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_bar(&b->o_final, 0, abort));
    tc::fence_after();
    // Alternating streams meet: stream 1 leaves its sums in the idle stages, 16 bytes of a row side by side
    // over the rows. Every softmax thread comes to the barrier, aborted or not.
    float4* other = reinterpret_cast<float4*>(smem + Shape<D>::kOffKV);
    if (!u.pair) {
        if (t == 1 && n > 0 && ok) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tc::tmem_ld32(tO + 32 * c, o);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    other[(8 * c + e) * kRows + r] = make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                                                 __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
            }
        }
        if (t == 1) b->m[r] = m, b->l[r] = l;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (t == 1) return;
        if (*abort) ok = false;  // either stream
    }
    const int row = (u.pair ? t * kRows : 0) + r;
    const int64_t at = ((int64_t)split * a.kv_heads + u.head) * a.rows + u.row0 + row;
    if (!ok) {
        if (row < u.nrows) a.ml[at] = make_float2(NB200_NAN, NB200_NAN);
        return;
    }
    float f0 = 1.f, f1 = 0.f;
    const bool merge = !u.pair && u.n > 1;
    if (merge) {
        const float m1 = b->m[r], top = fmaxf(m, m1);
        f0 = weight_of(m, l, top, sl2);
        f1 = weight_of(m1, b->l[r], top, sl2);
        l = l * f0 + b->l[r] * f1;
        m = top;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    f0 *= inv, f1 *= inv;
    float4* out = reinterpret_cast<float4*>(a.o + at * D);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tc::tmem_ld32(tO + 32 * c, o);
        if (row < u.nrows) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (f0 != 0.f)
                    x = make_float4(f0 * __uint_as_float(o[4 * e]), f0 * __uint_as_float(o[4 * e + 1]),
                                    f0 * __uint_as_float(o[4 * e + 2]), f0 * __uint_as_float(o[4 * e + 3]));
                if (merge && f1 != 0.f) {
                    const float4 y = other[(8 * c + e) * kRows + r];
                    x.x += f1 * y.x, x.y += f1 * y.y, x.z += f1 * y.z, x.w += f1 * y.w;
                }
                out[8 * c + e] = x;
            }
        }
    }
    if (row < u.nrows) a.ml[at] = make_float2(m, l);
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    tensor_part_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv, const TensorPart a) {
    using S = Shape<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Bars* b = reinterpret_cast<Bars*>(smem + S::kOffBar);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // Row blocks of one range of keys run side by side and share its tiles through L2.
    const unsigned blocks = (unsigned)(a.rows + 2 * kRows - 1) / (2 * kRows);
    unsigned id = blockIdx.x;
    Unit u;
    u.row0 = (int)(id % blocks) * 2 * kRows;
    id /= blocks;
    const int split = (int)(id % (unsigned)a.splits);
    u.head = (int)(id / (unsigned)a.splits);
    u.nrows = min(2 * kRows, a.rows - u.row0);
    u.pair = u.nrows > kRows;
    // The first tiles % splits ranges have a tile more.
    const int tiles = (a.keys + kKeys - 1) / kKeys, each = tiles / a.splits, more = tiles % a.splits;
    u.tile0 = split * each + min(split, more);
    u.n = each + (split < more);

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(&b->s_full[t], 1);
            for (int qp = 0; qp < 2; ++qp) mbar_init(&b->p_full[t][qp], 4);  // one arrival per softmax warp
        }
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&b->kv_full[s], 1);
            mbar_init(&b->kv_empty[s], 1);
        }
        mbar_init(&b->q_full, 8);  // one arrival per softmax warp
        mbar_init(&b->o_final, 1);
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
    pdl_wait();
    pdl_trigger();
    // Each role runs to the end of the kernel in its own branch (the register budget differs per branch); both
    // end at barrier 0, after which the MMA warp frees the tensor memory.
    if (warp < 8) {
        // The query rows, into the 128-byte swizzled tiles that the products read, while the first K/V tiles come;
        // rows past the last are zero. All copies of a thread in flight together: one after another their latencies took 15 us.
        constexpr int kPieces = D / 8, kStep = 256 / kPieces;  // 16-byte pieces of a row; rows of one round of the threads
        const int ch = threadIdx.x % kPieces, tokens = a.query.tokens, group = a.query.group;
        int row = threadIdx.x / kPieces;
        // Row row0 + row as (sequence, head, token); a round adds kStep rows, without a division.
        int tok = (u.row0 + row) % tokens, g = (u.row0 + row) / tokens, seq = g / group;
        g %= group;
        const int add_tok = kStep % tokens, add_g = kStep / tokens % group, add_seq = kStep / tokens / group;
        for (const int rows = u.pair ? 2 * kRows : kRows; row < rows; row += kStep) {
            const bool in = row < u.nrows;
            const T* src = static_cast<const T*>(a.query.q) +
                           (in ? seq * a.query.qb + (int64_t)(u.head * group + g) * a.query.qh + tok * a.query.qt + 8 * ch : 0);
            uint8_t* dst = smem + (row / kRows) * S::kTile + (ch >> 3) * S::kHalf + (row % kRows) * 128 +
                           (((ch & 7) ^ (row & 7)) << 4);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
                         : "memory");
            tok += add_tok;
            const bool carry = tok >= tokens;
            tok -= carry ? tokens : 0;
            g += add_g + carry;
            const bool next = g >= group;
            g -= next ? group : 0;
            seq += add_seq + next;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&b->q_full);
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        softmax_stream<T, D>(smem, b, tmem, a, u, split);
        tc::fence_before();
        asm volatile("bar.sync 0;" ::: "memory");
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
        if (warp == kLoadWarp) {
            if (lane == 0) producer<D>(&mk, &mv, smem, b, u);
            __syncwarp();
        } else if (warp == kMmaWarp) {
            if (tc::elect_one()) mma_issuer<T, D>(smem, b, tmem, u);
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

SharedLimit g_shared[4];

template <typename T, int D>
int launch(const CUtensorMap& mk, const CUtensorMap& mv, const TensorPart& a, SharedLimit& limit, cudaStream_t st) {
    const char* what = "nb200_prefix_attention";
    if (const int rc = limit.raise(what, tensor_part_kernel<T, D>, kSmem<D>)) return rc;
    const int64_t grid = (int64_t)((a.rows + 2 * kRows - 1) / (2 * kRows)) * a.splits * a.kv_heads;
    launch_pdl(tensor_part_kernel<T, D>, (unsigned)grid, kThreads, kSmem<D>, st, mk, mv, a);
    count_launch();
    return finish_launch(what);
}

}  // namespace

// Ranges of keys. A CTA has an SM for itself, for about 8 us and 2 us a tile (1 us where its streams alternate). The caches'
// workers run beside it on the SMs that are left, at about 95 MB/ms each and 5800 together, and on all of them behind it.
// The number of ranges for which both end first; the fewest of those, as every range is one more part to join.
int tensor_splits(int64_t kv_heads, int64_t rows, int64_t keys, int64_t other_bytes) {
    const int64_t units = kv_heads * ((rows + 2 * kRows - 1) / (2 * kRows)), tiles = (keys + kKeys - 1) / kKeys;
    const int64_t sms = sm_count();
    const float per_tile = rows > kRows ? 2.f : 1.f, other = (float)other_bytes * 1e-3f;  // KB; KB a us below
    int64_t best = 1;
    float least = 1e30f;
    auto consider = [&](int64_t s) {
        if (s < 1 || s > tiles) return;
        const int64_t waves = (units * s + sms - 1) / sms;
        const float end = (float)waves * (8.f + per_tile * (float)((tiles + s - 1) / s));
        const float beside = std::min(95.f * (float)(sms - units * s / waves), 5800.f);
        const float cost = end + std::max(other - beside * end, 0.f) / 5800.f;
        if (cost < 0.98f * least) best = s, least = cost;
    };
    const int64_t wave = std::max<int64_t>(1, sms / units);
    for (int64_t i = 1; i <= 8; ++i) consider(wave * i / 8);
    for (int64_t waves = 2; waves <= 4; ++waves) consider(waves * sms / units);
    return (int)best;
}

int launch_tensor_part(const TensorPart& a, int dtype, int64_t head_dim, const void* k, const nb200_attn_strides& ks,
                       const void* v, const nb200_attn_strides& vs, cudaStream_t st) {
    CUtensorMap mk, mv;
    int rc;
    if ((rc = encode_keys(&mk, "prefix_k", k, dtype, head_dim, a.keys, a.kv_heads, 1, ks, kKeys)) ||
        (rc = encode_keys(&mv, "prefix_v", v, dtype, head_dim, a.keys, a.kv_heads, 1, vs, kKeys)))
        return rc;
    if (dtype == NB200_BF16)
        return head_dim == 128 ? launch<__nv_bfloat16, 128>(mk, mv, a, g_shared[0], st)
                               : launch<__nv_bfloat16, 64>(mk, mv, a, g_shared[1], st);
    return head_dim == 128 ? launch<__half, 128>(mk, mv, a, g_shared[2], st) : launch<__half, 64>(mk, mv, a, g_shared[3], st);
}

}  // namespace prefix

int prefix_fault_take(unsigned int* bits) { return take_attn_fault(bits); }

}  // namespace nb200
