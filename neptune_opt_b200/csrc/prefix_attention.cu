// Attention of a few new tokens per sequence against a prefix that all sequences of the batch share and
// each sequence's own cache:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q k_j),   j over the prefix and the sequence's own
//                                                              tokens up to the query's own position
//
// The keys are cut into parts. A part's result for a query row is its output o over its keys alone, their maximum score m
// and the sum l behind it, and parts merge exactly: with w_i = l_i exp(scale (m_i - max m)), o = sum w_i o_i / sum w_i. (The
// pair, not m + log l: beside a maximum far from 0 the logarithm would be rounded away.) So the prefix is
// read once for the query rows of all sequences, whatever their number, each own cache once for its
// sequence, and long key ranges are split until the GPU is full; one pass over the pairs joins them, in a
// fixed order.
//
// Rows. The query rows that share a key/value head are numbered r = (b G + g) T + t (G = query heads per
// key/value head, T = new tokens): a sequence's rows are neighbours, and all B G T of them meet the prefix.
//
// Three kernels: tensor_part_kernel (prefix_attention_tc.cu) for a prefix with many query rows; stream_kernel
// for the caches, and for a prefix with few rows, where the bound is the keys' bytes; join_kernel. Few keys for few
// sequences take one, solo_kernel. bf16, 32 heads on 8 of
// 128: 256 sequences behind 16384 keys with uneven caches up to 512 take 117 us a call (bytes 53, the prefix's products
// 43), 4 behind 131072 keys 96 us, 5.6 TB/s.
#include <algorithm>

#include "attn.cuh"
#include "prefix_attention.cuh"
#include "prefix_line.h"

namespace nb200 {
namespace prefix {
namespace {

constexpr int kWarps = 4;      // warps of a stream kernel's CTA, each a worker of its own
constexpr int kStages = 3;     // steps of a worker in shared memory: one in use, two in flight
// CTAs that an SM can hold: half the head dimension leaves room for twice as many.
template <int D, int NT> constexpr int kCtas = D == 64 && NT <= 2 ? 4 : 2;

// What the stream kernel's workers share out (prefix_line.h), row tiles of 8 NT query rows each, and where it goes.
struct StreamArgs : Line {
    Query query;
    int rows;       // query rows of a key/value head over all sequences
    int slot_rows;
    float scale, sl2, slack;  // sl2 = scale * log2(e); kSlack in scores
    float* o;       // [slots][slot_rows][D]
    float2* ml;     // [slots][slot_rows]
    int2* span;     // [units]: first and last worker
    bool beside;    // runs beside the kernel ahead of it, of which it needs nothing (common.cuh)
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
    static constexpr uint32_t kExponents = 0x7f807f80u;  // of a pair, all ones: infinities and NaN
    __device__ __forceinline__ static void mul(float* d, const uint32_t* a, const uint32_t* b) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    }
};
template <> struct Mma<__half> {
    static constexpr uint32_t kExponents = 0x7c007c00u;
    __device__ __forceinline__ static void mul(float* d, const uint32_t* a, const uint32_t* b) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    }
};
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {  // an 8 x 8 matrix of 16-bit values over the warp
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    tc::tma_load_4d(reinterpret_cast<void*>(__cvta_shared_to_generic(dst)), map, c0, c1, c2, c3, bar);
}

// The piece of the line that a worker takes (a whole warp calls it). Each lane sums up the places of a run of sequences;
// the run that holds the piece's first place is then walked by its lane.
__device__ __forceinline__ Cursor piece_of(const StreamArgs& a, int worker, int workers) {
    const int lane = threadIdx.x & 31;
    const int64_t each = a.units_of_a_sequence();
    const int run = (a.batch + 31) / 32, b0 = min(lane * run, a.batch), b1 = min(b0 + run, a.batch);
    int own = 0;  // places of the lane's sequences, for one unit of each
    if (a.lens) {
#pragma unroll 8
        for (int b = b0; b < b1; ++b) own += places_of(a.tokens(b));
    } else {
        own = (b1 - b0) * places_of(a.cache);
    }
    int upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    const int64_t shared = a.shared_places(), all = shared + each * __shfl_sync(0xffffffffu, upto, 31);
    const int64_t share = (all + workers - 1) / workers;
    int64_t at = worker * share;
    Cursor c;
    c.left = 0;
    if (at >= all) return c;
    c.left = (int)min(share, all - at);
    int b = -1;
    if (at >= shared) {
        at -= shared;
        const int unit_at = (int)(at / each);  // the place, counted in one unit of each sequence
        const int holder = __ffs(__ballot_sync(0xffffffffu, upto > unit_at)) - 1;
        int before = upto - own;
        b = b0;
        if (lane == holder)
            for (int p; before + (p = places_of(a.tokens(b))) <= unit_at; ++b) before += p;
        b = __shfl_sync(0xffffffffu, b, holder);
        at -= each * __shfl_sync(0xffffffffu, before, holder);
    }
    c.start(a, b, at);
    return c;
}

// What a worker keeps of a unit's query rows, its running maximum, sum and output, and what a step of 16
// keys does to it. Column tile n of a lane's accumulators: query rows 8 n + 2 (lane % 4) and the next one. SEVERAL: of new
// tokens a sequence (what only several need would cost single ones 2 to 5%).
template <typename T, int D, int NT, bool SEVERAL>
struct Rows {
    float o[NT][D / 16][4], m[NT][2], l[NT][2];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) m[n][e] = -NB200_INF, l[n][e] = 0.f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][d][e] = 0.f;
        }
    }
    // Whether the lane's part of a staged V's keys from..to holds an infinity or NaN.
    __device__ __forceinline__ static bool any_odd(uint32_t vs, int from, int to, int lane) {
        bool odd = false;
#pragma unroll 1
        for (int i = from * 8 + lane; i < (to + 1) * 8; i += 32)
#pragma unroll 1
            for (int h = 0; h < D / 64; ++h) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(vs + h * kStepKeys * 128 + i * 16));
#pragma unroll
                for (int k = 0; k < 4; ++k) odd |= __vcmpeq2(w[k] & Mma<T>::kExponents, Mma<T>::kExponents) != 0u;
            }
        return odd;
    }
    // Keys kb on, of a box at ks and vs in shared memory; `limit`: the last key a row sees, `lowest` and `highest`: the least
    // and the greatest of them.
    __device__ __forceinline__ void step(const uint32_t (*qf)[D / 16][2], uint32_t ks, uint32_t vs, int kb,
                                         const int (*limit)[2], int lowest, int highest, float sl2, float slack, int lane) {
        constexpr uint32_t kBox = kStepKeys * 128;
        // This lane's address in a box: the row it loads for ldmatrix, and the swizzle of its 16-byte pieces.
        const int k_row = lane & 15, k_piece = lane >> 4;                         // K: keys 0-15, then 8 columns on
        const int v_row = (lane >> 4) * 8 + (lane & 7), v_piece = lane >> 3 & 1;  // V, transposed: columns, then keys
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t f[4];
            ldmatrix4(f, ks + (d / 4) * kBox + k_row * 128 + (((2 * (d % 4) + k_piece) ^ (k_row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) Mma<T>::mul(s[n], f, qf[n][d]);
        }
        // s[n][e]: key lane / 4 + 8 (e / 2), query row e % 2 of the lane's two.
        if (kb + kStepKeys - 1 > lowest) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (kb + (lane >> 2) + 8 * (e / 2) > limit[n][e % 2]) s[n][e] = -NB200_INF;
        }
        bool grow = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) grow |= fmaxf(s[n][e], s[n][e + 2]) > m[n][e] + slack;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = fmaxf(s[n][e], s[n][e + 2]);
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                    const float next = fmaxf(m[n][e], top);
                    const float f = next == m[n][e] ? 1.f : ex2((m[n][e] - next) * sl2);
                    m[n][e] = next;
                    l[n][e] *= f;
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) o[n][d][e] *= f, o[n][d][e + 2] *= f;
                }
        }
        uint32_t p[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float top = m[n][e] == -NB200_INF ? 0.f : m[n][e];
                x[e] = ex2(fmaf(s[n][e] - top, sl2, kLift<T>));
                x[e + 2] = ex2(fmaf(s[n][e + 2] - top, sl2, kLift<T>));
                l[n][e] += x[e] + x[e + 2];
            }
            p[n][0] = transpose8(Elem<T>::pack_word(x[0], x[1]));
            p[n][1] = transpose8(Elem<T>::pack_word(x[2], x[3]));
        }
        auto values = [&](int d, uint32_t* f) {
            ldmatrix4_t(f, vs + (d / 4) * kBox + v_row * 128 + (((2 * (d % 4) + v_piece) ^ (v_row & 7)) << 4));
        };
        // Of several new tokens the earlier ones do not see the later ones' keys: their probabilities there are 0, which takes
        // any value but an infinity or NaN out of the product. Where there is one, the rows of each limit take the product
        // by themselves, the greatest limit first, and the values that no row is left to see are zeroed.
        if (SEVERAL && min(highest, kb + kStepKeys - 1) > lowest) {
            const int last = min(highest, kb + kStepKeys - 1);
            if (__any_sync(0xffffffffu, any_odd(vs, max(lowest + 1 - kb, 0), last - kb, lane))) {
#pragma unroll 1
                for (int key = last; key >= max(lowest, kb); --key) {
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        uint32_t f[4];
                        values(d, f);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float x[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = o[n][d][e];
                            Mma<T>::mul(x, f, p[n]);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (min(limit[n][e % 2], last) == key) o[n][d][e] = x[e];
                        }
                    }
                    __syncwarp();
                    if (lane < 8 * (D / 64))
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs + lane / 8 * kBox + (key - kb) * 128 + lane % 8 * 16),
                                     "r"(0u)
                                     : "memory");
                    fence_proxy_async();
                    __syncwarp();
                }
                return;
            }
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            uint32_t f[4];
            values(d, f);
#pragma unroll
            for (int n = 0; n < NT; ++n) Mma<T>::mul(o[n][d], f, p[n]);
        }
    }
};

// Zeroes a staged V's keys from `keys` on.
template <int D>
__device__ __forceinline__ void zero_behind(uint32_t vs, int keys, int lane) {
    if (keys >= kStepKeys) return;
    for (int i = keys * 8 + lane; i < kStepKeys * 8; i += 32)
#pragma unroll
        for (int h = 0; h < D / 64; ++h)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vs + h * kStepKeys * 128 + i * 16), "r"(0u)
                         : "memory");
    fence_proxy_async();
    __syncwarp();
}

// Every warp is a worker: its lane 0 has the keys and values of the steps copied (TMA) into shared memory that no
// other warp touches, two steps ahead and across the units' borders, and the warp keeps the running maximum, sum
// and output of its unit in registers. No barrier, no atomics.
//
// The products are taken transposed, S^T = K Q^T and O^T = V^T P^T, with the keys (then the head dimension) along
// the 16 rows of mma.sync and the query rows along its 8 columns: a unit of few query rows pays for 8, not 16, and the
// fragments of K and V serve all NT column tiles.
//
// Every wait is bounded; one that runs out sets bit 1 of the fault word, and the worker waits (again with a limit) for
// its copies and leaves NaN in the slots of its unfinished shares.
template <typename T, int D, int NT, bool SEVERAL>
__global__ void __launch_bounds__(kWarps * 32, kCtas<D, NT>)
    stream_kernel(const __grid_constant__ CUtensorMap shared_k, const __grid_constant__ CUtensorMap shared_v,
                  const __grid_constant__ CUtensorMap own_k, const __grid_constant__ CUtensorMap own_v,
                  const StreamArgs a) {
    constexpr uint32_t kBox = kStepKeys * 128;       // 64 columns of a step's keys, 128-byte swizzled
    constexpr uint32_t kTile = kBox * (D / 64);      // K or V of a step
    // The next unit's query rows are loaded while this one's keys run, where there are registers to hold them:
    // loaded between two units they would hold up the copies by a memory latency.
    constexpr bool kAhead = NT <= 2;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[kWarps][kStages];
    __shared__ int abort_flag[kWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t mine = ((smem_u32(smem_raw) + 1023u) & ~1023u) + warp * (kStages * 2 * kTile);
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&full[warp][i], 1);
        abort_flag[warp] = 0;
        fence_barrier_init();
    }
    if (a.beside) fence_early();
    else pdl_wait();
    pdl_trigger();
    const int worker = (int)blockIdx.x * kWarps + warp;
    // The kernel that joins the parts waits for this one alone, so this one ends after the kernel ahead of it: its last
    // CTA waits. (Were they all to wait, those that are done would hold their places against those to come.)
    const bool waits = a.beside && blockIdx.x + 1 == gridDim.x;
    Cursor use = piece_of(a, worker, (int)gridDim.x * kWarps);
    if (use.left <= 0) {
        if (waits) pdl_wait();
        return;
    }
    Cursor get = use;
    int sent = 0;

    auto copy = [&](int stage) {  // the cursor's step into a stage
        if (get.left <= 0) return;
        if (lane == 0) {
            const bool shared = get.batch < 0;
            const CUtensorMap *mk = shared ? &shared_k : &own_k, *mv = shared ? &shared_v : &own_v;
            const int b = shared ? 0 : get.batch, key = get.step * kStepKeys;
            uint64_t* bar = &full[warp][stage];
            mbar_expect_tx(bar, 2 * kTile);
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                tma_load(mine + stage * 2 * kTile + h * kBox, mk, 64 * h, key, get.head, b, bar);
                tma_load(mine + stage * 2 * kTile + kTile + h * kBox, mv, 64 * h, key, get.head, b, bar);
            }
        }
        ++sent;
        get.next(a);
    };
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    // Column tile n of this lane's accumulators: query rows 8 n + 2 (lane % 4) and the next one.
    uint32_t qf[NT][D / 16][2], next_q[kAhead ? NT : 1][D / 16][2];
    int limit[NT][2], lowest = 0;  // last key a row sees; of the unit's rows, the least
    Rows<T, D, NT, SEVERAL> t;
    int nrows = 0;
    auto load_rows = [&](const Cursor& c, uint32_t(*q)[D / 16][2]) {
        const bool shared = c.batch < 0;
        const int first = c.tile * 8 * NT, rows = (shared ? a.rows : a.query.group * a.query.tokens) - first;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int in = 8 * n + (lane >> 2);  // past the last row: the first one again, whose result is not stored
            int seq = c.batch, g = first + (in < rows ? in : 0), tok = 0;
            if constexpr (SEVERAL) tok = g % a.query.tokens, g /= a.query.tokens;
            if (shared) seq = g / a.query.group, g %= a.query.group;
            const T* p = static_cast<const T*>(a.query.q) + seq * a.query.qb +
                         (int64_t)(c.head * a.query.group + g) * a.query.qh + tok * a.query.qt + 2 * (lane & 3);
#pragma unroll
            for (int d = 0; d < D / 16; ++d)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    q[n][d][h] = *reinterpret_cast<const uint32_t*>(p + 16 * d + 8 * h);
        }
    };
    auto begin = [&] {
        const bool shared = use.batch < 0;
        const int in_unit = use.tile * 8 * NT;
        nrows = min(8 * NT, (shared ? a.rows : a.query.group * a.query.tokens) - in_unit);
        lowest = shared ? use.keys - 1 : use.keys - a.query.tokens;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
                limit[n][e] = shared ? use.keys - 1
                              : lowest + (SEVERAL ? (in_unit + 8 * n + 2 * (lane & 3) + e) % a.query.tokens : 0);
        }
        t.clear();
        if (kAhead && use.left > use.steps - use.step) {
            Cursor c = use;
            c.next_unit(a);
            load_rows(c, next_q);
        }
    };
    load_rows(use, qf);
    begin();
    if (lane == 0 && use.step == 0) a.span[use.unit(a)].x = worker;

    bool ok = true;
    int stage = 0, done = 0;
    uint32_t phase = 0;
    for (;;) {
        ok = __all_sync(0xffffffffu, wait_bar(&full[warp][stage], phase, &abort_flag[warp]));
        if (!ok) break;
        // Everyone has left the stage that is filled next.
        copy(stage == 0 ? kStages - 1 : stage - 1);
        const uint32_t ks = mine + stage * (2 * kTile), vs = ks + kTile;
        const int kb = use.step * kStepKeys;
        // What a cache holds behind a sequence must not reach the products: 0 times an infinity is none.
        if (use.batch >= 0) zero_behind<D>(vs, use.keys - kb, lane);
        t.step(qf, ks, vs, kb, limit, lowest, use.keys - 1, a.sl2, a.slack, lane);

        ++done;
        if (++stage == kStages) stage = 0, phase ^= 1u;
        const bool ends = use.step + 1 == use.steps;
        if (use.left > 1 && !ends) {
            ++use.step;
            --use.left;
            continue;
        }
        // The worker's share of the unit is done.
        const int unit = use.unit(a);
        const int64_t slot = ((int64_t)worker + unit) * a.slot_rows;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) t.l[n][e] += __shfl_xor_sync(0xffffffffu, t.l[n][e], w);
                const int in = 8 * n + 2 * (lane & 3) + e;
                if (in < nrows) {
                    const float inv = t.l[n][e] == 0.f ? 0.f : 1.f / t.l[n][e];
                    float* dst = a.o + (slot + in) * D + (lane >> 2);
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        dst[16 * d] = t.o[n][d][e] * inv;
                        dst[16 * d + 8] = t.o[n][d][e + 2] * inv;
                    }
                    if (lane < 4) a.ml[slot + in] = make_float2(t.m[n][e], t.l[n][e]);
                }
            }
        if (lane == 0 && ends) a.span[unit].y = worker;
        use.next(a);
        if (use.left <= 0) break;
        if (lane == 0) a.span[use.unit(a)].x = worker;
        if constexpr (kAhead) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int d = 0; d < D / 16; ++d) qf[n][d][0] = next_q[n][d][0], qf[n][d][1] = next_q[n][d][1];
        } else {
            load_rows(use, qf);
        }
        begin();
    }
    if (!ok) {
        // Every copy lands before the CTA may exit; `sent` were issued, of which `done` have been waited for.
        for (int i = done; i < sent; ++i) drain_bar(&full[warp][i % kStages], (i / kStages) & 1u);
        for (;;) {
            const int unit = use.unit(a);
            for (int in = lane; in < a.slot_rows; in += 32) a.ml[((int64_t)worker + unit) * a.slot_rows + in] = make_float2(NB200_NAN, NB200_NAN);
            if (lane == 0 && use.ends_unit()) a.span[unit].y = worker;
            if (!use.skip_unit(a)) break;
            if (lane == 0) a.span[use.unit(a)].x = worker;
        }
    }
    if (waits) pdl_wait();
}

// The same in one kernel without parts in memory, where a CTA a sequence and key/value head is enough: its warps share the
// prefix and the cache, one list of keys for the same rows, and join in shared memory. (Rows as in stream_kernel; of a
// unit's two tiles the prefix's rows are the sequence's own.) The bound is latency, a launch and a few steps. A wait that
// runs out, as there: the CTA's rows read out as NaN.
template <typename T, int D, int NT, int W, bool SEVERAL>
__global__ void __launch_bounds__(W * 32, D == 64 || W == 4 ? 2 : 1)
    solo_kernel(const __grid_constant__ CUtensorMap shared_k, const __grid_constant__ CUtensorMap shared_v,
                const __grid_constant__ CUtensorMap own_k, const __grid_constant__ CUtensorMap own_v, const StreamArgs a,
                void* out, float* out_lse) {
    constexpr uint32_t kBox = kStepKeys * 128, kTile = kBox * (D / 64);
    constexpr int kPitch = D + 4;  // floats of a row in shared memory: no two lanes of a store meet in a bank
    static_assert(8 * NT * kPitch * 4 <= kStages * 2 * kTile, "a warp leaves its output in its stages");
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[W][kStages];
    __shared__ int abort_flag[W];
    __shared__ float sh_m[W][8 * NT], sh_l[W][8 * NT];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t all_stages = (smem_u32(smem_raw) + 1023u) & ~1023u, mine = all_stages + warp * (kStages * 2 * kTile);
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(&full[warp][i], 1);
        abort_flag[warp] = 0;
        fence_barrier_init();
    }
    pdl_wait();
    pdl_trigger();
    const int seq = (int)(blockIdx.x / (unsigned)a.kv_heads), head = (int)(blockIdx.x % (unsigned)a.kv_heads);
    const int group = a.query.group, tokens = SEVERAL ? a.query.tokens : 1, rows = group * tokens;
    const int own = a.tokens(seq), shared_steps = steps_of(a.prefix), steps = shared_steps + steps_of(own);
    const int share = (steps + W - 1) / W, begin = warp * share, end = min(begin + share, steps);
    int get = begin;
    auto copy = [&](int stage) {
        if (get >= end) return;
        if (lane == 0) {
            const bool shared = get < shared_steps;
            const CUtensorMap *mk = shared ? &shared_k : &own_k, *mv = shared ? &shared_v : &own_v;
            const int b = shared ? 0 : seq, key = (shared ? get : get - shared_steps) * kStepKeys;
            uint64_t* bar = &full[warp][stage];
            mbar_expect_tx(bar, 2 * kTile);
#pragma unroll
            for (int h = 0; h < D / 64; ++h) {
                tma_load(mine + stage * 2 * kTile + h * kBox, mk, 64 * h, key, head, b, bar);
                tma_load(mine + stage * 2 * kTile + kTile + h * kBox, mv, 64 * h, key, head, b, bar);
            }
        }
        ++get;
    };
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    uint32_t qf[NT][D / 16][2];
    int limit[NT][2];  // of the cache's keys
    Rows<T, D, NT, SEVERAL> t;
    t.clear();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int in = 8 * n + (lane >> 2), row = in < rows ? in : 0;
        const T* p = static_cast<const T*>(a.query.q) + seq * a.query.qb +
                     (int64_t)(head * group + row / tokens) * a.query.qh + row % tokens * a.query.qt + 2 * (lane & 3);
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
#pragma unroll
            for (int h = 0; h < 2; ++h) qf[n][d][h] = *reinterpret_cast<const uint32_t*>(p + 16 * d + 8 * h);
#pragma unroll
        for (int e = 0; e < 2; ++e) limit[n][e] = own - tokens + (8 * n + 2 * (lane & 3) + e) % tokens;
    }
    int ok = 1, stage = 0;
    uint32_t phase = 0;
    for (int i = begin; i < end; ++i) {
        ok = __all_sync(0xffffffffu, wait_bar(&full[warp][stage], phase, &abort_flag[warp]));
        if (!ok) {
            for (int c = i; c < get; ++c) drain_bar(&full[warp][(c - begin) % kStages], ((c - begin) / kStages) & 1u);
            break;
        }
        // Everyone has left the stage that is filled next.
        copy(stage == 0 ? kStages - 1 : stage - 1);
        const uint32_t ks = mine + stage * (2 * kTile), vs = ks + kTile;
        if (i < shared_steps) {
            int last[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) last[n][0] = last[n][1] = a.prefix - 1;
            t.step(qf, ks, vs, i * kStepKeys, last, a.prefix - 1, a.prefix - 1, a.sl2, a.slack, lane);
        } else {
            const int kb = (i - shared_steps) * kStepKeys;
            zero_behind<D>(vs, own - kb, lane);
            t.step(qf, ks, vs, kb, limit, own - tokens, own - 1, a.sl2, a.slack, lane);
        }
        if (++stage == kStages) stage = 0, phase ^= 1u;
    }
    // The warp's results, into its own stages, which no copy is under way to.
    float* part = static_cast<float*>(__cvta_shared_to_generic(mine));
    if (ok) {
        __syncwarp();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) t.l[n][e] += __shfl_xor_sync(0xffffffffu, t.l[n][e], w);
                const int in = 8 * n + 2 * (lane & 3) + e;
                if (lane < 4) sh_m[warp][in] = t.m[n][e], sh_l[warp][in] = t.l[n][e];
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    part[in * kPitch + 16 * d + (lane >> 2)] = t.o[n][d][e];
                    part[in * kPitch + 16 * d + 8 + (lane >> 2)] = t.o[n][d][e + 2];
                }
            }
    }
    const bool complete = __syncthreads_and(ok);
    constexpr int E = D / 32;
    for (int in = warp; in < rows; in += W) {
        float top = -NB200_INF, sum = complete ? 0.f : NB200_NAN, v[E];
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
        if (complete && own - tokens + in % tokens >= 0) {
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, sh_m[w][in]);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const float l = sh_l[w][in], m = sh_m[w][in];
                const float f = weight_of(m, l, top, a.sl2);
                sum += f * l;
                const float* o = static_cast<const float*>(__cvta_shared_to_generic(all_stages + w * (kStages * 2 * kTile))) +
                                 in * kPitch + lane * E;
#pragma unroll
                for (int e = 0; e < E; ++e) v[e] = f == 0.f ? v[e] : fmaf(f, o[e], v[e]);
            }
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t at = ((int64_t)seq * a.kv_heads + head) * rows + in;
        uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<T*>(out) + at * D) + lane * (E / 2);
#pragma unroll
        for (int e = 0; e < E; e += 2) dst[e / 2] = Elem<T>::pack_word(v[e] * inv, v[e + 1] * inv);
        if (out_lse && lane == 0)
            out_lse[at] = natural_lse<T>(top, sum, a.scale);
    }
}

struct JoinArgs {
    const float *tensor_o, *o;           // parts of the tensor cores, [splits][kv_heads][rows][D]; slots of the stream kernel
    const float2 *tensor_ml, *ml;        // the same without D
    float scale, sl2;
    const int2* span;
    int workers;                         // of the stream kernel
    void* out;                           // [batch, heads, tokens, D]
    float* out_lse;                      // nullable
    const int* lens;
    int kv_heads, group, tokens, rows, cache;
    int splits;                          // of the tensor cores (0: none)
    bool shared;                         // units of the prefix come first
    int own_tiles, tile_rows, slot_rows;
};

// WIDE: a CTA per query row, its eight warps taking turns at the parts; else a warp per row. The parts are the
// tensor cores' (or the prefix units' slots), then the own units' slots, weighed and added in a fixed order. The bound is
// latency: 3 to 5 us behind the other kernels. A query before its
// sequence's first token (a free slot of the batch) reads out as zero with a log-sum-exp of -inf; a row whose parts are
// not all there as NaN.
template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs a) {
    constexpr int E = D / 32, kTurns = WIDE ? 8 : 1;  // parts of a turn are kTurns apart
    __shared__ float sh[WIDE ? 8 : 1][D], sh_sum[8];
    const int64_t all = (int64_t)a.kv_heads * a.rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t id = WIDE ? blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
    if (id >= all) return;
    const int head = (int)(id / a.rows), r = (int)(id % a.rows);
    const int t = r % a.tokens, g = r / a.tokens % a.group, b = r / a.tokens / a.group;
    const int64_t at = ((int64_t)b * a.kv_heads * a.group + head * a.group + g) * a.tokens + t;
    const int len = a.lens ? max(0, min(ld_early(a.lens + b), a.cache)) : a.cache;
    pdl_wait();
    pdl_trigger();
    float top = -NB200_INF, sum = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    if (len - a.tokens + t >= 0) {
        // Two runs of parts: rows `far + i far_step` of one array, `near + i slot_rows` of another.
        const float* far_o = a.o;
        const float2* far_ml = a.ml;
        int64_t far = 0, far_step = a.slot_rows;
        int nfar = 0;
        const int in = r - b * a.group * a.tokens;
        const int unit = (a.shared ? a.kv_heads : 0) + (b * a.kv_heads + head) * a.own_tiles + in / a.tile_rows;
        const int2 w = a.span[unit];
        bool known = are_workers(w.x, w.y, a.workers);
        if (a.splits) {
            far_o = a.tensor_o, far_ml = a.tensor_ml, far = id, far_step = all, nfar = a.splits;
        } else if (a.shared) {
            const int2 u = a.span[head];
            known &= are_workers(u.x, u.y, a.workers);
            far = (int64_t)(u.x + head) * a.slot_rows + r;
            nfar = u.y - u.x + 1;
        }
        const int64_t near = (int64_t)(w.x + unit) * a.slot_rows + in % a.tile_rows;
        // Unless lengths change while a call runs, or a worker is lost, the spans are right; what they name is read only then.
        if (!known) atomicOr(&g_attn_fault, 2u);
        const int parts = known ? nfar + w.y - w.x + 1 : 0;
        if (!known) sum = NB200_NAN;
        auto row_of = [&](int i) { return i < nfar ? far + i * far_step : near + (int64_t)(i - nfar) * a.slot_rows; };
        auto ml_of = [&](int i) { return i < parts ? (i < nfar ? far_ml : a.ml)[row_of(i)] : make_float2(-NB200_INF, 0.f); };
        // Four o's in flight at a time, the first four before their weights are known.
        float o[4][E];
        auto load4 = [&](int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int part = min(i + k * kTurns, parts - 1);
                const float* p = (part < nfar ? far_o : a.o) + row_of(part) * D + lane * E;
                if constexpr (E == 4) *reinterpret_cast<float4*>(o[k]) = __ldg(reinterpret_cast<const float4*>(p));
                else *reinterpret_cast<float2*>(o[k]) = __ldg(reinterpret_cast<const float2*>(p));
            }
        };
        const int start = WIDE ? warp : 0;
        if (known) load4(start);
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, ml_of(i).x);
        top = warp_max(top);
        for (int i0 = start; i0 < parts; i0 += 32 * kTurns) {  // 32 parts, weighed by the 32 lanes
            const float2 ml = ml_of(i0 + lane * kTurns);
            const float mine = ml.y * weight_of(ml.x, ml.y, top, a.sl2);
            sum += mine;
            for (int i = 0; i < 32 && i0 + i * kTurns < parts; i += 4) {
                if (i0 + i > start) load4(i0 + i * kTurns);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float f = __shfl_sync(0xffffffffu, mine, i + k);
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = f == 0.f ? v[e] : fmaf(f, o[k][e], v[e]);
                }
            }
        }
        sum = warp_sum(sum);
    }
    if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < E; ++e) sh[warp][lane * E + e] = v[e];
        if (lane == 0) sh_sum[warp] = sum;
        __syncthreads();
        if (warp) return;
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            sum += sh_sum[w];
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += sh[w][lane * E + e];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint32_t w[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2) w[e / 2] = Elem<T>::pack_word(v[e] * inv, v[e + 1] * inv);
    uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at * D) + lane * (E / 2);
#pragma unroll
    for (int e = 0; e < E / 2; ++e) out[e] = w[e];
    if (a.out_lse && lane == 0) a.out_lse[at] = natural_lse<T>(top, sum, a.scale);
}

// ------------------------------------------------------------------ host side
// Up to kStreamRows query rows of a key/value head meet the prefix in the stream kernel, and up to kFewRows if it is no
// longer than kFewKeys; otherwise it goes to the tensor cores. bf16, 8 heads of 128: 4 rows, 8192 keys 12.4 us against
// 16.2; 16 rows, 131072 keys 99 us against 90; 16 rows, 1000 keys 12.4 against 10.6, 300 keys 8.3 against 10.3.
constexpr int kStreamRows = 8, kFewRows = 32, kFewKeys = 512;

struct Plan {
    int64_t rows;                  // query rows of a key/value head
    int nt;                        // 8-row tiles of a unit
    bool solo;                     // solo_kernel does it all
    int splits;                    // of the prefix on the tensor cores (0: it is in the stream kernel, or empty)
    bool shared;                   // the stream kernel's line has the prefix's units
    int64_t own_tiles, slot_rows, units, ctas;
    int64_t most_parts;            // parts of a row, at most
    // Workspace, in bytes from its start.
    int64_t tensor_o, tensor_ml, o, ml, span, bytes;
};

Plan plan_of(const nb200_prefix_attn_args& a) {
    Plan p = {};
    const int64_t own_rows = a.heads / a.kv_heads * a.tokens;
    p.rows = a.batch * own_rows;
    // One kernel while reading the prefix once a sequence, and a sequence's keys into one SM (about 190 keys of head
    // dimension 128 a us, in which everything here is counted), costs less than a second launch, the parts and the join.
    // bf16 on the GPU alone, 32 heads on 8 of 128, full caches, prefix and cache: 200 and 64, 1 sequence 4.5 us (with parts
    // in memory 5.9), 32 5.8 (12.0), 256 35 (26); 500 and 1024, 4 sequences 10.8 (11.1), 32 24 (32); 1000 and 1000, 1 sequence
    // 13.1 (8.8), 16 13.6 (17.4); 2000 and 100, 4 13.5 (10.5), 32 23.5 (19.0); 100 and 4096, 4 24 (16), 64 157 (171). The last
    // limit is for one long sequence among short ones.
    const int64_t units = a.batch * a.kv_heads, waves = (units + sm_count() - 1) / sm_count();
    const int64_t prefix_keys = waves * a.prefix * a.head_dim / 128, own_keys = waves * a.cache * a.head_dim / 128;
    p.solo = own_rows <= 16 && prefix_keys <= 1500 + own_keys / 7 &&
             (waves == 1 ? prefix_keys + own_keys <= 500 + 40 * units : a.cache * a.head_dim <= 4096 * 128);
    if (p.solo) {
        p.nt = own_rows <= 8 ? 1 : 2;
        p.bytes = 16;
        return p;
    }
    if (a.prefix && p.rows > (a.prefix > kFewKeys ? kStreamRows : kFewRows)) {
        // With lengths that only the device knows, the caches are taken to be half full.
        const int64_t bytes = a.batch * a.kv_heads * a.cache * a.head_dim * 4 / (a.seq_lens ? 2 : 1);
        p.splits = tensor_splits(a.kv_heads, p.rows, a.prefix, bytes);
    }
    p.shared = a.prefix && !p.splits;
    const int64_t most = p.shared ? p.rows : own_rows;
    p.nt = most <= 8 ? 1 : most <= 16 ? 2 : 4;  // one tile holds all rows that meet the prefix
    static_assert(kStreamRows <= 32 && kFewRows <= 32, "a tile's rows");
    const int64_t tile = 8 * p.nt;
    p.own_tiles = (own_rows + tile - 1) / tile;
    p.slot_rows = std::min(tile, most);
    p.units = a.kv_heads * (p.shared + a.batch * p.own_tiles);
    auto line = [](int64_t keys) { return keys ? kEntry + (keys + kStepKeys - 1) / kStepKeys : 0; };
    const int64_t prefix_steps = p.shared ? line(a.prefix) : 0, own_steps = line(a.cache);
    const int64_t steps = a.kv_heads * (prefix_steps + a.batch * p.own_tiles * own_steps);
    // Two CTAs an SM. Four where each worker still has 16 places and the SM holds four (caches of 256 sequences, head
    // dimension 64: 33.5 us, with two 37.4; with few places the more parts cost more than that gives, 12.8 us against
    // 10.9).
    // Four, two at a time, beside the tensor cores' kernel where pieces are short anyway, because SMs become free at
    // different times (32 sequences: 25.9 us against 26.9; 256 sequences, with long pieces, 101 against 96).
    const int64_t sms = sm_count(), places = steps / (2 * sms * kWarps);
    const bool four = (a.head_dim == 64 && p.nt <= 2 && places >= 32) || (p.splits && places < 32);
    p.ctas = std::max<int64_t>(1, std::min<int64_t>((steps + kWarps - 1) / kWarps, (four ? 4 : 2) * sms));
    const int64_t share = std::max<int64_t>(1, steps / (p.ctas * kWarps));
    p.most_parts = p.splits + (prefix_steps + own_steps) / share + 2;
    auto take = [&](int64_t floats) {
        const int64_t at = p.bytes;
        p.bytes += (floats * 4 + 15) / 16 * 16;
        return at;
    };
    const int64_t slots = p.units + p.ctas * kWarps;
    p.tensor_o = take(p.splits * a.kv_heads * p.rows * a.head_dim);
    p.o = take(slots * p.slot_rows * a.head_dim);
    p.tensor_ml = take(2 * p.splits * a.kv_heads * p.rows);
    p.ml = take(2 * slots * p.slot_rows);
    p.span = take(2 * p.units);
    return p;
}

constexpr int kVariants = 7;  // of a type, a head dimension, and one or several new tokens
SharedLimit g_shared[8 * kVariants];

struct Maps {
    CUtensorMap shared_k, shared_v, own_k, own_v;
};

template <typename T, int D, int NT, bool SEVERAL>
int launch_stream(const Maps& m, const StreamArgs& a, int64_t ctas, SharedLimit& limit, cudaStream_t st) {
    constexpr uint32_t bytes = kWarps * kStages * 2 * kStepKeys * D * 2 + 1024;  // + alignment slack
    if (const int rc = limit.raise("nb200_prefix_attention", stream_kernel<T, D, NT, SEVERAL>, bytes)) return rc;
    launch_pdl(stream_kernel<T, D, NT, SEVERAL>, (unsigned)ctas, kWarps * 32, bytes, st, m.shared_k, m.shared_v, m.own_k,
               m.own_v, a);
    count_launch();
    return finish_launch("nb200_prefix_attention");
}

template <typename T, int D, int NT, int W, bool SEVERAL>
int launch_solo(const Maps& m, const StreamArgs& a, void* o, float* lse, SharedLimit& limit, cudaStream_t st) {
    constexpr uint32_t bytes = W * kStages * 2 * kStepKeys * D * 2 + 1024;  // + alignment slack
    if (const int rc = limit.raise("nb200_prefix_attention", solo_kernel<T, D, NT, W, SEVERAL>, bytes)) return rc;
    launch_pdl(solo_kernel<T, D, NT, W, SEVERAL>, (unsigned)(a.batch * a.kv_heads), W * 32, bytes, st, m.shared_k, m.shared_v,
               m.own_k, m.own_v, a, o, lse);
    count_launch();
    return finish_launch("nb200_prefix_attention");
}

template <typename T, int D, bool SEVERAL>
int launch_all(const nb200_prefix_attn_args& n, const nb200_attn_strides* s, const void* q, const void* pk,
               const void* pv, const void* k, const void* v, void* o, float* lse, char* work, SharedLimit* limits,
               cudaStream_t st) {
    const Plan p = plan_of(n);
    const int64_t most = (int64_t)1 << 30;
    if (p.units > most || p.splits * n.kv_heads * p.rows > most * 16) {
        set_error("nb200_prefix_attention: the call exceeds the kernels' index range");
        return NB200_ERR_CAPACITY;
    }
    auto at = [&](int64_t offset) { return reinterpret_cast<float*>(work + offset); };
    auto pairs_at = [&](int64_t offset) { return reinterpret_cast<float2*>(work + offset); };
    const Query query = {q, s[0].batch, s[0].head, s[0].seq, (int)(n.heads / n.kv_heads), (int)n.tokens};
    const float sl2 = n.scale * 1.4426950408889634f;
    int rc;
    if (p.splits) {
        const TensorPart t = {query, (int)n.kv_heads, (int)p.rows, (int)n.prefix, p.splits, sl2, slack_of(sl2),
                              at(p.tensor_o), pairs_at(p.tensor_ml)};
        if ((rc = launch_tensor_part(t, n.dtype, n.head_dim, pk, s[1], pv, s[2], st))) return rc;
    }
    StreamArgs a = {};
    a.query = query;
    Maps maps = {};
    if ((p.shared || (p.solo && n.prefix)) &&
        ((rc = encode_keys(&maps.shared_k, "prefix_k", pk, n.dtype, D, n.prefix, n.kv_heads, 1, s[1], kStepKeys)) ||
         (rc = encode_keys(&maps.shared_v, "prefix_v", pv, n.dtype, D, n.prefix, n.kv_heads, 1, s[2], kStepKeys))))
        return rc;
    if (n.cache && ((rc = encode_keys(&maps.own_k, "k", k, n.dtype, D, n.cache, n.kv_heads, n.batch, s[3], kStepKeys)) ||
                    (rc = encode_keys(&maps.own_v, "v", v, n.dtype, D, n.cache, n.kv_heads, n.batch, s[4], kStepKeys))))
        return rc;
    a.lens = n.seq_lens;
    a.batch = (int)n.batch, a.kv_heads = (int)n.kv_heads;
    a.prefix = p.shared || p.solo ? (int)n.prefix : 0, a.cache = (int)n.cache;
    a.rows = (int)p.rows, a.own_tiles = (int)p.own_tiles;
    a.slot_rows = (int)p.slot_rows;
    a.scale = n.scale, a.sl2 = sl2, a.slack = slack_of(sl2);
    if (p.solo) {
        // Where there are more CTAs than SMs, two an SM: one starts while the other reads. Head dimension 128 has room for
        // them with four warps each.
        if (D == 128 && a.batch * (int64_t)a.kv_heads > sm_count())
            return p.nt == 1 ? launch_solo<T, D, 1, 4, SEVERAL>(maps, a, o, lse, limits[3], st)
                             : launch_solo<T, D, 2, 4, SEVERAL>(maps, a, o, lse, limits[4], st);
        return p.nt == 1 ? launch_solo<T, D, 1, 8, SEVERAL>(maps, a, o, lse, limits[5], st)
                         : launch_solo<T, D, 2, 8, SEVERAL>(maps, a, o, lse, limits[6], st);
    }
    a.o = at(p.o), a.ml = pairs_at(p.ml), a.span = reinterpret_cast<int2*>(at(p.span));
    a.beside = p.splits > 0;  // the tensor cores' kernel started after all that came before
    rc = p.nt == 1   ? launch_stream<T, D, 1, SEVERAL>(maps, a, p.ctas, limits[0], st)
         : p.nt == 2 ? launch_stream<T, D, 2, SEVERAL>(maps, a, p.ctas, limits[1], st)
                     : launch_stream<T, D, 4, SEVERAL>(maps, a, p.ctas, limits[2], st);
    if (rc) return rc;
    JoinArgs j = {};
    j.tensor_o = at(p.tensor_o), j.tensor_ml = pairs_at(p.tensor_ml), j.o = a.o, j.ml = a.ml, j.span = a.span;
    j.scale = a.scale, j.sl2 = a.sl2;
    j.workers = (int)p.ctas * kWarps;
    j.out = o, j.out_lse = lse, j.lens = n.seq_lens;
    j.kv_heads = a.kv_heads, j.group = query.group, j.tokens = query.tokens, j.rows = a.rows, j.cache = a.cache;
    j.splits = p.splits, j.shared = p.shared, j.own_tiles = a.own_tiles, j.tile_rows = 8 * p.nt;
    j.slot_rows = a.slot_rows;
    const int64_t rows = n.kv_heads * p.rows;
    // A warp per row while the rows fill the GPU and their parts are few.
    if (p.most_parts > 16 && rows < 8 * 8 * (int64_t)sm_count())
        launch_pdl(join_kernel<T, D, true>, (unsigned)rows, 256, 0, st, j);
    else
        launch_pdl(join_kernel<T, D, false>, (unsigned)((rows + 7) / 8), 256, 0, st, j);
    count_launch();
    return finish_launch("nb200_prefix_attention");
}

}  // namespace

int encode_keys(CUtensorMap* map, const char* what, const void* base, int dtype, int64_t d, int64_t keys, int64_t heads,
                int64_t batch, const nb200_attn_strides& s, uint32_t box_keys) {
    const auto enc = tensor_map_encoder("nb200_prefix_attention");
    if (!enc) return NB200_ERR_LAUNCH;
    auto bytes = [d](int64_t stride, int64_t size) { return (cuuint64_t)(size > 1 ? stride * 2 : d * 2); };
    const cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)keys, (cuuint64_t)heads, (cuuint64_t)batch};
    const cuuint64_t strides[3] = {bytes(s.seq, keys), bytes(s.head, heads), bytes(s.batch, batch)};
    const cuuint32_t box[4] = {64, box_keys, 1, 1}, one[4] = {1, 1, 1, 1};
    const CUresult rc = enc(map, dtype == NB200_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                            const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
        set_error("nb200_prefix_attention: cannot describe %s as a tensor map (CUresult %d)", what, (int)rc);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

}  // namespace prefix

using namespace prefix;

int64_t prefix_attention_work_bytes(const nb200_prefix_attn_args& a) { return plan_of(a).bytes; }

int prefix_stream_fault_take(unsigned int* bits) { return take_attn_fault(bits); }

int launch_prefix_attention(const nb200_prefix_attn_args& n, const nb200_attn_strides* s, const void* q, const void* pk,
                            const void* pv, const void* k, const void* v, void* o, float* lse, void* work,
                            cudaStream_t st) {
    char* w = static_cast<char*>(work);
    const int variant = (n.dtype == NB200_BF16 ? 0 : 4) + (n.head_dim == 128 ? 0 : 2) + (n.tokens > 1);
    auto launch = [&](auto kernels) { return kernels(n, s, q, pk, pv, k, v, o, lse, w, g_shared + variant * kVariants, st); };
    switch (variant) {
        case 0: return launch(launch_all<__nv_bfloat16, 128, false>);
        case 1: return launch(launch_all<__nv_bfloat16, 128, true>);
        case 2: return launch(launch_all<__nv_bfloat16, 64, false>);
        case 3: return launch(launch_all<__nv_bfloat16, 64, true>);
        case 4: return launch(launch_all<__half, 128, false>);
        case 5: return launch(launch_all<__half, 128, true>);
        case 6: return launch(launch_all<__half, 64, false>);
        default: return launch(launch_all<__half, 64, true>);
    }
}

}  // namespace nb200
