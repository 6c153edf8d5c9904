// Attention of a few new tokens per sequence against a prefix that all sequences of the batch share and
// each sequence's own cache:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q k_j),   j over the prefix and the sequence's own
//                                                              tokens up to the query's own position
//
// The keys are cut into parts. A part's result for a query row is the pair (o, log2 sum) over its keys
// alone, and pairs merge exactly: with w_i = 2^(l_i - max l), o = sum w_i o_i / sum w_i. So the prefix is
// read once for the query rows of all sequences, whatever their number, each own cache once for its
// sequence, and long key ranges are split until the GPU is full; one pass over the pairs joins them, in a
// fixed order.
//
// Rows. The query rows that share a key/value head are numbered r = (b G + g) T + t (G = query heads per
// key/value head, T = new tokens): a sequence's rows are neighbours, and all B G T of them meet the prefix.
//
// Three kernels: tensor_part_kernel (prefix_attention_tc.cu) for a prefix with many query rows; stream_kernel
// for the caches, and for a prefix with few rows, where the bound is the keys' bytes; join_kernel.
#include <algorithm>

#include "prefix_attention.cuh"
#include "stream.cuh"

namespace nb200 {
namespace prefix {
namespace {

constexpr int kWarps = 4;      // warps of a stream kernel's CTA, each a worker of its own
constexpr int kCtas = 2;       // its CTAs per SM
constexpr int kStepKeys = 16;  // keys of a worker's step
constexpr int kStages = 3;     // steps of a worker in shared memory: one in use, two in flight

struct Keys {  // one source of keys and values (strides in elements)
    const void *k, *v;
    int64_t kb, kh, ks, vb, vh, vs;
};

// A unit of the stream kernel is a tile of 16 MT query rows and the keys they share: units of the prefix
// (key/value head, row tile; none when the prefix runs on the tensor cores), then units of the caches
// (sequence, key/value head, row tile). All units' steps of 16 keys stand in one line, of which every worker
// takes an equal piece, whatever the sequences' lengths are. A piece covers the end of one unit, whole units,
// the beginning of another: worker w's result for unit u goes to slot w + u, which no other pair has, and
// span[u] says which workers had a share in u.
struct StreamArgs {
    Query query;
    Keys shared, own;
    const int* lens;  // tokens of each sequence (null: all of the cache)
    int batch, kv_heads, prefix, cache;
    int rows;                      // query rows of a key/value head over all sequences
    int prefix_tiles, own_tiles;   // row tiles of a unit's rows
    int slot_rows;
    float sl2;                     // scale * log2(e)
    float *o, *lse;                // [slots][slot_rows][D], [slots][slot_rows]
    int2* span;                    // [units]: first and last worker
    bool beside;                   // runs beside the kernel ahead of it, of which it needs nothing
};

template <typename T> struct Mma;
template <> struct Mma<__nv_bfloat16> {
    __device__ __forceinline__ static void mul(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct Mma<__half> {
    __device__ __forceinline__ static void mul(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ int tokens_of(const int* lens, int b, int keys) {
    return lens ? max(0, min(lens[b], keys)) : keys;
}
__device__ __forceinline__ int steps_of(int keys) { return (keys + kStepKeys - 1) / kStepKeys; }

// A position in the line of steps.
struct Cursor {
    int batch;  // -1: a unit of the prefix
    int head, tile, step, steps, keys;

    __device__ __forceinline__ void sequence(const StreamArgs& a, int b) {
        batch = b, head = 0, tile = 0, keys = tokens_of(a.lens, b, a.cache), steps = steps_of(keys);
    }
    // The next step; there is one.
    __device__ __forceinline__ void next(const StreamArgs& a) {
        if (++step < steps) return;
        step = 0;
        if (++tile < (batch < 0 ? a.prefix_tiles : a.own_tiles)) return;
        tile = 0;
        if (++head < a.kv_heads) return;
        int b = batch;
        do sequence(a, ++b);
        while (steps == 0 && b + 1 < a.batch);
    }
    __device__ __forceinline__ int unit(const StreamArgs& a) const {
        return batch < 0 ? head * a.prefix_tiles + tile
                         : a.kv_heads * a.prefix_tiles + (batch * a.kv_heads + head) * a.own_tiles + tile;
    }
};

// Steps per worker, and the cursor at step `at(per worker)`; a whole warp calls it.
__device__ __forceinline__ int64_t share_of(const StreamArgs& a, int64_t workers, int64_t& all) {
    const int lane = threadIdx.x & 31;
    int64_t own = 0;
    if (a.lens) {
        for (int b = lane; b < a.batch; b += 32) own += steps_of(tokens_of(a.lens, b, a.cache));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    } else {
        own = (int64_t)a.batch * steps_of(a.cache);
    }
    all = (int64_t)a.kv_heads * ((int64_t)a.prefix_tiles * steps_of(a.prefix) + a.own_tiles * own);
    return (all + workers - 1) / workers;
}
__device__ __forceinline__ Cursor cursor_at(const StreamArgs& a, int64_t at) {
    Cursor c;
    const int64_t shared = (int64_t)a.kv_heads * a.prefix_tiles * steps_of(a.prefix);
    if (at < shared) {
        c.batch = -1, c.keys = a.prefix, c.steps = steps_of(a.prefix);
        const int unit = (int)(at / c.steps);
        c.head = unit / a.prefix_tiles, c.tile = unit % a.prefix_tiles, c.step = (int)(at % c.steps);
        return c;
    }
    at -= shared;
    const int64_t each = (int64_t)a.kv_heads * a.own_tiles;
    int b = 0;
    if (a.lens) {  // 32 sequences at a time
        const int lane = threadIdx.x & 31;
        for (;; b += 32) {
            const int64_t mine = b + lane < a.batch ? each * steps_of(tokens_of(a.lens, b + lane, a.cache)) : 0;
            int64_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const unsigned past = __ballot_sync(0xffffffffu, upto > at);
            if (past || b + 32 >= a.batch) {
                const int pick = past ? __ffs(past) - 1 : 31;
                at -= __shfl_sync(0xffffffffu, upto - mine, pick);
                b += pick;
                break;
            }
            at -= __shfl_sync(0xffffffffu, upto, 31);
        }
    } else {
        const int64_t steps = each * steps_of(a.cache);
        b = (int)(at / steps);
        at %= steps;
    }
    c.sequence(a, b);
    const int unit = (int)(at / c.steps);
    c.head = unit / a.own_tiles, c.tile = unit % a.own_tiles, c.step = (int)(at % c.steps);
    return c;
}

// Every warp is a worker: it copies the keys and values of its steps into shared memory that no other warp
// touches, two steps ahead and across the units' borders, and keeps the running maximum, sum and output of its
// unit in registers. No barrier, no atomics.
template <typename T, int D, int MT>
__global__ void __launch_bounds__(kWarps * 32, kCtas) stream_kernel(const StreamArgs a) {
    constexpr int kChunks = D / 8;                // 16-byte pieces of a row
    constexpr uint32_t kTile = kStepKeys * D * 2; // K or V of a step
    extern __shared__ __align__(128) uint8_t smem[];
    if (!a.beside) pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int worker = (int)blockIdx.x * kWarps + (threadIdx.x >> 5);
    int64_t all;
    const int64_t share = share_of(a, (int64_t)gridDim.x * kWarps, all);
    const int64_t first = worker * share;
    // The kernel that joins the parts waits for this one alone, so this one ends after the kernel ahead of it.
    if (first >= all) {
        if (a.beside) pdl_wait();
        return;
    }
    int left = (int)min(share, all - first);  // steps to go
    Cursor use = cursor_at(a, first), get = use;
    int to_get = left;

    const uint32_t mine = smem_addr(smem) + (threadIdx.x >> 5) * (kStages * 2 * kTile);
    // The cursor's step into a stage. Keys past the end read as zero: what a cache holds behind a sequence must not
    // reach the products.
    auto copy = [&](int stage) {
        if (to_get > 0) {
            const bool shared = get.batch < 0;
            const Keys& s = shared ? a.shared : a.own;
            const T* kp = static_cast<const T*>(s.k) + (shared ? 0 : get.batch * s.kb) + get.head * s.kh;
            const T* vp = static_cast<const T*>(s.v) + (shared ? 0 : get.batch * s.vb) + get.head * s.vh;
            const int kb = get.step * kStepKeys;
            const uint32_t at = mine + stage * (2 * kTile);
#pragma unroll
            for (int c = lane; c < kStepKeys * kChunks; c += 32) {
                const int row = c / kChunks, ch = c % kChunks;
                const bool in = kb + row < get.keys;
                const int64_t key = in ? kb + row : get.keys - 1;
                const uint32_t off = (uint32_t)(row * D * 2 + ((ch ^ (row & 7)) << 4));
                cp_async16(at + off, kp + key * s.ks + ch * 8, in ? 16 : 0);
                cp_async16(at + kTile + off, vp + key * s.vs + ch * 8, in ? 16 : 0);
            }
            if (--to_get) get.next(a);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    // Row i of this lane's accumulators: lane / 4 + 8 i within the tile, i < 2 MT.
    uint32_t qf[MT][D / 16][4];
    int limit[2 * MT];  // last key the row sees
    float o[MT][D / 8][4], m[2 * MT], l[2 * MT];
    int nrows = 0;
    auto begin = [&] {
        const bool shared = use.batch < 0;
        const int in_unit = use.tile * 16 * MT, own_rows = a.query.group * a.query.tokens;
        const int row0 = (shared ? 0 : use.batch * own_rows) + in_unit;
        nrows = min(16 * MT, (shared ? a.rows : own_rows) - in_unit);
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int in = (lane >> 2) + 8 * i;
            const bool live = in < nrows;
            const int r = row0 + (live ? in : 0);
            limit[i] = shared ? use.keys - 1 : use.keys - a.query.tokens + r % a.query.tokens;
            const T* q = query_row<T>(a.query, use.head, r);
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    qf[i / 2][s][i % 2 + 2 * h] =
                        live ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 8 * h + 2 * (lane & 3)) : 0u;
            m[i] = -NB200_INF, l[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int c = 0; c < D / 8; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
    };
    begin();
    if (lane == 0 && use.step == 0) a.span[use.unit(a)].x = worker;

    for (int stage = 0;; stage = stage + 1 == kStages ? 0 : stage + 1) {
        cp_async_wait<kStages - 2>();
        __syncwarp();  // the step's data is there, and everyone has left the stage that is filled next
        copy(stage == 0 ? kStages - 1 : stage - 1);
        const uint32_t ks = mine + stage * (2 * kTile), vs = ks + kTile;
        const int kb = use.step * kStepKeys;
        float s[MT][2][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[mt][e / 4][e % 4] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            const int row = (lane >> 4) * 8 + (lane & 7), ch = 2 * d + (lane >> 3 & 1);
            uint32_t b[4];
            ldmatrix4(b, ks + row * D * 2 + ((ch ^ (row & 7)) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                Mma<T>::mul(s[mt][0], qf[mt][d], b[0], b[1]);
                Mma<T>::mul(s[mt][1], qf[mt][d], b[2], b[3]);
            }
        }
        // Scores in the log2 domain; keys past a row's last are masked.
        float top[2 * MT];
        bool grow = false;
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
            top[r] = -NB200_INF;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float& x = s[r / 2][e / 2][2 * (r % 2) + e % 2];
                x = kb + 8 * (e / 2) + 2 * (lane & 3) + e % 2 <= limit[r] ? x * a.sl2 : -NB200_INF;
                top[r] = fmaxf(top[r], x);
            }
            grow |= top[r] > m[r] + kSlack;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int r = 0; r < 2 * MT; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                const float next = fmaxf(m[r], top[r]);
                const float f = next == m[r] ? 1.f : ex2(m[r] - next);
                m[r] = next;
                l[r] *= f;
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    o[r / 2][c][2 * (r % 2)] *= f;
                    o[r / 2][c][2 * (r % 2) + 1] *= f;
                }
            }
        }
        uint32_t p[MT][4];
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
            const float ref = (m[r] == -NB200_INF ? 0.f : m[r]) - kLift<T>;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float x = ex2(s[r / 2][h][2 * (r % 2)] - ref), y = ex2(s[r / 2][h][2 * (r % 2) + 1] - ref);
                l[r] += x + y;
                p[r / 2][r % 2 + 2 * h] = Elem<T>::pack_word(x, y);
            }
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            const int row = (lane >> 3 & 1) * 8 + (lane & 7), ch = 2 * c + (lane >> 4);
            uint32_t b[4];
            ldmatrix4_t(b, vs + row * D * 2 + ((ch ^ (row & 7)) << 4));
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                Mma<T>::mul(o[mt][2 * c], p[mt], b[0], b[1]);
                Mma<T>::mul(o[mt][2 * c + 1], p[mt], b[2], b[3]);
            }
        }

        --left;
        const bool ends = use.step + 1 == use.steps;
        if (left && !ends) {
            ++use.step;
            continue;
        }
        // The worker's share of the unit is done.
        const int unit = use.unit(a);
        const int64_t slot = ((int64_t)worker + unit) * a.slot_rows;
#pragma unroll
        for (int r = 0; r < 2 * MT; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            const int in = (lane >> 2) + 8 * r;
            if (in < nrows) {
                const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
                float* dst = a.o + (slot + in) * D + 2 * (lane & 3);
#pragma unroll
                for (int c = 0; c < D / 8; ++c)
                    *reinterpret_cast<float2*>(dst + 8 * c) =
                        make_float2(o[r / 2][c][2 * (r % 2)] * inv, o[r / 2][c][2 * (r % 2) + 1] * inv);
                if ((lane & 3) == 0) a.lse[slot + in] = l[r] == 0.f ? -NB200_INF : m[r] + log2f(l[r]) - kLift<T>;
            }
        }
        if (lane == 0 && ends) a.span[unit].y = worker;
        if (!left) break;
        use.next(a);
        if (lane == 0) a.span[use.unit(a)].x = worker;
        begin();
    }
    cp_async_wait<0>();
    if (a.beside) pdl_wait();
}

struct JoinArgs {
    const float *tensor_o, *tensor_lse;  // parts of the tensor cores: [splits][kv_heads][rows][D], and without D
    const float *o, *lse;                // slots of the stream kernel
    const int2* span;
    void* out;                           // [batch, heads, tokens, D]
    float* out_lse;                      // nullable
    const int* lens;
    int kv_heads, group, tokens, rows, cache;
    int splits;                          // of the tensor cores (0: none)
    int prefix_tiles, own_tiles, tile_rows, slot_rows;
};

// WIDE: a CTA per query row, its eight warps taking turns at the parts; else a warp per row. The parts are the
// tensor cores' (or the prefix units' slots), then the own units' slots, weighed and added in a fixed order. A query before its
// sequence's first token (a free slot of the batch) reads out as zero with a log-sum-exp of -inf.
template <typename T, int D, bool WIDE>
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs a) {
    constexpr int E = D / 32, kTurns = WIDE ? 8 : 1;
    __shared__ float sh[WIDE ? 8 : 1][D], sh_sum[8];
    pdl_wait();
    pdl_trigger();
    const int64_t all = (int64_t)a.kv_heads * a.rows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t id = WIDE ? blockIdx.x : (int64_t)blockIdx.x * 8 + warp;
    if (id >= all) return;
    const int head = (int)(id / a.rows), r = (int)(id % a.rows);
    const int t = r % a.tokens, g = r / a.tokens % a.group, b = r / a.tokens / a.group;
    const int64_t at = ((int64_t)b * a.kv_heads * a.group + head * a.group + g) * a.tokens + t;
    const int len = tokens_of(a.lens, b, a.cache);
    float top = -NB200_INF, sum = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    if (len - a.tokens + t >= 0) {
        // Two runs of parts: rows `far + i far_step` of one array, `near + i near_step` of another.
        const float *far_o = a.o, *far_lse = a.lse;
        int64_t far = 0, far_step = a.slot_rows;
        int nfar = 0;
        if (a.splits) {
            far_o = a.tensor_o, far_lse = a.tensor_lse, far = id, far_step = all, nfar = a.splits;
        } else if (a.prefix_tiles) {
            const int unit = head * a.prefix_tiles + r / a.tile_rows;
            const int2 w = a.span[unit];
            far = (int64_t)(w.x + unit) * a.slot_rows + r % a.tile_rows;
            nfar = w.y - w.x + 1;
        }
        const int in = r - b * a.group * a.tokens;
        const int unit = a.kv_heads * a.prefix_tiles + (b * a.kv_heads + head) * a.own_tiles + in / a.tile_rows;
        const int2 w = a.span[unit];
        const int64_t near = (int64_t)(w.x + unit) * a.slot_rows + in % a.tile_rows;
        const int parts = nfar + w.y - w.x + 1;
        auto row_of = [&](int i) { return i < nfar ? far + i * far_step : near + (int64_t)(i - nfar) * a.slot_rows; };
        auto lse_of = [&](int i) { return i < parts ? (i < nfar ? far_lse : a.lse)[row_of(i)] : -NB200_INF; };
        for (int i = lane; i < parts; i += 32) top = fmaxf(top, lse_of(i));
        top = warp_max(top);
        for (int i0 = WIDE ? warp : 0; i0 < parts; i0 += 32 * kTurns) {
            const float x = lse_of(i0 + lane * kTurns);
            const float mine = x == -NB200_INF ? 0.f : ex2(x - top);  // NaN stays
            sum += mine;
            // Four parts in flight; one without weight is not read.
            for (int i = 0; i < 32 && i0 + i * kTurns < parts; i += 4) {
                float f[4], o[4][E];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    f[k] = __shfl_sync(0xffffffffu, mine, i + k);
#pragma unroll
                    for (int e = 0; e < E; ++e) o[k][e] = 0.f;
                    if (f[k] != 0.f) {
                        const int part = i0 + (i + k) * kTurns;
                        const float* p = (part < nfar ? far_o : a.o) + row_of(part) * D + lane * E;
                        if constexpr (E == 4) *reinterpret_cast<float4*>(o[k]) = __ldg(reinterpret_cast<const float4*>(p));
                        else *reinterpret_cast<float2*>(o[k]) = __ldg(reinterpret_cast<const float2*>(p));
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int e = 0; e < E; ++e) v[e] = fmaf(f[k], o[k][e], v[e]);
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
    if (a.out_lse && lane == 0) a.out_lse[at] = sum == 0.f ? -NB200_INF : (top + log2f(sum)) * 0.69314718055994531f;
}

// ------------------------------------------------------------------ host side
// Up to this many query rows of a key/value head meet the prefix in the stream kernel; more go to the tensor
// cores.
constexpr int kStreamRows = 32;

struct Plan {
    int64_t rows;                  // query rows of a key/value head
    int mt;                        // 16-row tiles of a unit
    int splits;                    // of the prefix on the tensor cores (0: it is in the stream kernel, or empty)
    int64_t prefix_tiles, own_tiles, slot_rows, units, ctas;
    int64_t most_parts;            // parts of a row, at most
    // Workspace, in bytes from its start.
    int64_t tensor_o, tensor_lse, o, lse, span, bytes;
};

Plan plan_of(const nb200_prefix_attn_args& a) {
    Plan p = {};
    const int64_t own_rows = a.heads / a.kv_heads * a.tokens;
    p.rows = a.batch * own_rows;
    p.mt = own_rows > 16 ? 2 : 1;
    const int64_t tile = 16 * p.mt;
    if (a.prefix && p.rows > kStreamRows) p.splits = tensor_splits(a.kv_heads, p.rows, a.prefix);
    p.prefix_tiles = a.prefix && !p.splits ? (p.rows + tile - 1) / tile : 0;
    p.own_tiles = (own_rows + tile - 1) / tile;
    p.slot_rows = std::min(tile, p.prefix_tiles ? p.rows : own_rows);
    p.units = a.kv_heads * (p.prefix_tiles + a.batch * p.own_tiles);
    const int64_t prefix_steps = p.prefix_tiles ? (a.prefix + kStepKeys - 1) / kStepKeys : 0;
    const int64_t own_steps = (a.cache + kStepKeys - 1) / kStepKeys;
    const int64_t steps = a.kv_heads * (p.prefix_tiles * prefix_steps + a.batch * p.own_tiles * own_steps);
    p.ctas = std::max<int64_t>(1, std::min<int64_t>((steps + kWarps - 1) / kWarps, kCtas * (int64_t)sm_count()));
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
    p.tensor_lse = take(p.splits * a.kv_heads * p.rows);
    p.lse = take(slots * p.slot_rows);
    p.span = take(2 * p.units);
    return p;
}

SharedLimit g_shared[8];

template <typename T, int D, int MT>
int launch_stream(const StreamArgs& a, int64_t ctas, SharedLimit& limit, cudaStream_t st) {
    constexpr uint32_t bytes = kWarps * kStages * 2 * kStepKeys * D * 2;
    if (const int rc = limit.raise("nb200_prefix_attention", stream_kernel<T, D, MT>, bytes)) return rc;
    launch_pdl(stream_kernel<T, D, MT>, (unsigned)ctas, kWarps * 32, bytes, st, a);
    count_launch();
    return finish_launch("nb200_prefix_attention");
}

template <typename T, int D>
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
    const Query query = {q, s[0].batch, s[0].head, s[0].seq, (int)(n.heads / n.kv_heads), (int)n.tokens};
    const float sl2 = n.scale * 1.4426950408889634f;
    int rc;
    if (p.splits) {
        const TensorPart t = {query, (int)n.kv_heads, (int)p.rows, (int)n.prefix, p.splits, sl2, at(p.tensor_o), at(p.tensor_lse)};
        if ((rc = launch_tensor_part(t, n.dtype, n.head_dim, pk, s[1], pv, s[2], st))) return rc;
    }
    StreamArgs a = {};
    a.query = query;
    a.shared = {pk, pv, 0, s[1].head, s[1].seq, 0, s[2].head, s[2].seq};
    a.own = {k, v, s[3].batch, s[3].head, s[3].seq, s[4].batch, s[4].head, s[4].seq};
    a.lens = n.seq_lens;
    a.batch = (int)n.batch, a.kv_heads = (int)n.kv_heads, a.prefix = p.prefix_tiles ? (int)n.prefix : 0, a.cache = (int)n.cache;
    a.rows = (int)p.rows, a.prefix_tiles = (int)p.prefix_tiles, a.own_tiles = (int)p.own_tiles;
    a.slot_rows = (int)p.slot_rows;
    a.sl2 = sl2;
    a.o = at(p.o), a.lse = at(p.lse), a.span = reinterpret_cast<int2*>(at(p.span));
    a.beside = p.splits > 0;  // the tensor cores' kernel started after all that came before
    rc = p.mt == 1 ? launch_stream<T, D, 1>(a, p.ctas, limits[0], st) : launch_stream<T, D, 2>(a, p.ctas, limits[1], st);
    if (rc) return rc;
    JoinArgs j = {};
    j.tensor_o = at(p.tensor_o), j.tensor_lse = at(p.tensor_lse), j.o = a.o, j.lse = a.lse, j.span = a.span;
    j.out = o, j.out_lse = lse, j.lens = n.seq_lens;
    j.kv_heads = a.kv_heads, j.group = query.group, j.tokens = query.tokens, j.rows = a.rows, j.cache = a.cache;
    j.splits = p.splits, j.prefix_tiles = a.prefix_tiles, j.own_tiles = a.own_tiles, j.tile_rows = 16 * p.mt;
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
}  // namespace prefix

using namespace prefix;

int64_t prefix_attention_work_bytes(const nb200_prefix_attn_args& a) { return plan_of(a).bytes; }

int launch_prefix_attention(const nb200_prefix_attn_args& n, const nb200_attn_strides* s, const void* q, const void* pk,
                            const void* pv, const void* k, const void* v, void* o, float* lse, void* work,
                            cudaStream_t st) {
    char* w = static_cast<char*>(work);
    if (n.dtype == NB200_BF16)
        return n.head_dim == 128
                   ? launch_all<__nv_bfloat16, 128>(n, s, q, pk, pv, k, v, o, lse, w, g_shared, st)
                   : launch_all<__nv_bfloat16, 64>(n, s, q, pk, pv, k, v, o, lse, w, g_shared + 2, st);
    return n.head_dim == 128 ? launch_all<__half, 128>(n, s, q, pk, pv, k, v, o, lse, w, g_shared + 4, st)
                             : launch_all<__half, 64>(n, s, q, pk, pv, k, v, o, lse, w, g_shared + 6, st);
}

}  // namespace nb200
