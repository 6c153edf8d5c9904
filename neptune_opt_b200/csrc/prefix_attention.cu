// Attention of a few new tokens per sequence against a prefix that all sequences of the batch share and
// each sequence's own cache:
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q k_j),   j over the prefix and the sequence's own
//                                                              tokens up to the query's own position
//
// The keys are cut into parts. A part's result for a query row is the pair (o, log2 sum) over its keys
// alone, and pairs merge exactly: with w_i = 2^(l_i - max l), o = sum w_i o_i / sum w_i. So the prefix is
// read once for the query rows of all sequences, whatever their number, each own cache once for its
// sequence, and long key ranges are split until the GPU is full; one pass over the pairs joins them, in
// ascending order of the parts.
//
// Rows. The query rows that share a key/value head are numbered r = (b G + g) T + t (G = query heads per
// key/value head, T = new tokens): a sequence's rows are neighbours, and all B G T of them meet the prefix.
#include <algorithm>

#include "prefix_attention.cuh"
#include "stream.cuh"

namespace nb200 {
namespace prefix {
namespace {

constexpr int kWarps = 4;      // warps of a part kernel's CTA; each takes every fourth step of the keys
constexpr int kStepKeys = 16;  // keys of a warp's step
constexpr int kStages = 3;     // steps in flight per warp

struct Keys {  // one source of keys and values (strides in elements)
    const void *k, *v;
    int64_t kb, kh, ks, vb, vh, vs;
};

struct PartArgs {
    Query query;
    Keys src;
    const int* lens;     // own keys: tokens of each sequence (null: all); unused for the prefix
    int kv_heads;
    int keys;            // keys of the source (the prefix, or the cache's length)
    int rows;            // query rows of a key/value head over all sequences
    int unit_rows;       // rows that share this source's keys: all, or a sequence's
    int tiles, splits, split_keys;
    float sl2;           // scale * log2(e)
    float *o, *lse;      // [splits][kv_heads][rows][D], [splits][kv_heads][rows]
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

// One part: MT tiles of 16 query rows against the keys [k0, k1) of one source. Each warp keeps its own running
// maximum, sum and output over its steps, in registers, and copies its keys and values into shared memory
// that no other warp touches; the four results meet at the end.
template <typename T, int D, int MT, bool OWN>
__global__ void __launch_bounds__(kWarps * 32, 2) part_kernel(const PartArgs a) {
    constexpr int kChunks = D / 8;                      // 16-byte pieces of a row
    constexpr uint32_t kTile = kStepKeys * D * 2;       // K or V of a step
    constexpr uint32_t kWarpBytes = kStages * 2 * kTile;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float sh_m[kWarps][16 * MT], sh_l[kWarps][16 * MT];
    pdl_wait();
    pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned block = blockIdx.x;
    const int tile = (int)(block % (unsigned)a.tiles);
    block /= (unsigned)a.tiles;
    const int split = (int)(block % (unsigned)a.splits);
    block /= (unsigned)a.splits;
    const int head = (int)(block % (unsigned)a.kv_heads), batch = (int)(block / (unsigned)a.kv_heads);

    const int row0 = batch * a.unit_rows + tile * 16 * MT;            // first row of the tile
    const int nrows = min(16 * MT, (batch + 1) * a.unit_rows - row0);
    const int len = OWN ? tokens_of(a.lens, batch, a.keys) : a.keys;
    const int k0 = split * a.split_keys, k1 = min(k0 + a.split_keys, len);
    const int64_t out0 = ((int64_t)split * a.kv_heads + head) * a.rows + row0;
    if (k0 >= k1) {
        for (int i = threadIdx.x; i < nrows; i += kWarps * 32) a.lse[out0 + i] = -NB200_INF;
        return;
    }

    // Row i of this lane's accumulators: lane / 4 + 8 i within the tile, i < 2 MT.
    uint32_t qf[MT][D / 16][4];
    int limit[2 * MT];  // last key the row sees
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        const int in = (lane >> 2) + 8 * i;
        const bool live = in < nrows;
        const int r = row0 + (live ? in : 0);
        limit[i] = OWN ? len - a.query.tokens + r % a.query.tokens : k1 - 1;
        const T* q = query_row<T>(a.query, head, r);
#pragma unroll
        for (int s = 0; s < D / 16; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                qf[i / 2][s][i % 2 + 2 * h] =
                    live ? *reinterpret_cast<const uint32_t*>(q + 16 * s + 8 * h + 2 * (lane & 3)) : 0u;
    }

    float o[MT][D / 8][4];
    float m[2 * MT], l[2 * MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][c][e] = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) m[i] = -NB200_INF, l[i] = 0.f;

    const T* kp = static_cast<const T*>(a.src.k) + (OWN ? batch * a.src.kb : 0) + head * a.src.kh;
    const T* vp = static_cast<const T*>(a.src.v) + (OWN ? batch * a.src.vb : 0) + head * a.src.vh;
    const uint32_t mine = smem_addr(smem) + warp * kWarpBytes;
    const int steps = (k1 - k0 + kStepKeys - 1) / kStepKeys;
    // Step i of this warp begins at key k0 + 16 (warp + 4 i). Keys past the end read as zero: what a cache
    // holds behind a sequence must not reach the products.
    auto copy = [&](int i) {
        const int step = warp + kWarps * i;
        if (step < steps) {
            const int kb = k0 + step * kStepKeys;
            const uint32_t at = mine + (uint32_t)(i % kStages) * 2 * kTile;
#pragma unroll
            for (int c = lane; c < kStepKeys * kChunks; c += 32) {
                const int row = c / kChunks, ch = c % kChunks;
                const bool in = kb + row < k1;
                const int64_t key = in ? kb + row : k1 - 1;
                const uint32_t off = (uint32_t)(row * D * 2 + ((ch ^ (row & 7)) << 4));
                cp_async16(at + off, kp + key * a.src.ks + ch * 8, in ? 16 : 0);
                cp_async16(at + kTile + off, vp + key * a.src.vs + ch * 8, in ? 16 : 0);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) copy(i);

    for (int i = 0; warp + kWarps * i < steps; ++i) {
        cp_async_wait<kStages - 2>();
        __syncwarp();  // the step's data is there, and everyone has left the stage that is filled next
        copy(i + kStages - 1);
        const uint32_t ks = mine + (uint32_t)(i % kStages) * 2 * kTile, vs = ks + kTile;
        const int kb = k0 + (warp + kWarps * i) * kStepKeys;
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
    }

    // The four warps' results meet in shared memory.
    cp_async_wait<0>();
    __syncthreads();
    float* sh_o = reinterpret_cast<float*>(smem);  // [kWarps][16 MT][D]
#pragma unroll
    for (int r = 0; r < 2 * MT; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        const int in = (lane >> 2) + 8 * r;
        if ((lane & 3) == 0) {
            sh_m[warp][in] = m[r];
            sh_l[warp][in] = l[r];
        }
        float* dst = sh_o + (warp * 16 * MT + in) * D + 2 * (lane & 3);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
            *reinterpret_cast<float2*>(dst + 8 * c) = make_float2(o[r / 2][c][2 * (r % 2)], o[r / 2][c][2 * (r % 2) + 1]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nrows * (D / 4); i += kWarps * 32) {
        const int in = i / (D / 4), c = i % (D / 4) * 4;
        float top = sh_m[0][in];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh_m[w][in]);
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            // Without a finite score the sum is 0, or NaN.
            const float f = sh_m[w][in] == -NB200_INF ? sh_l[w][in] : ex2(sh_m[w][in] - top);
            const float4 u = *reinterpret_cast<const float4*>(sh_o + (w * 16 * MT + in) * D + c);
            sum += f * sh_l[w][in];
            if (f != 0.f) v.x += f * u.x, v.y += f * u.y, v.z += f * u.z, v.w += f * u.w;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<float4*>(a.o + (out0 + in) * D + c) = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
        if (c == 0) a.lse[out0 + in] = sum == 0.f ? -NB200_INF : top + log2f(sum) - kLift<T>;
    }
}

struct JoinArgs {
    const float *o, *lse;  // [parts][kv_heads][rows][D], [parts][kv_heads][rows]
    void* out;             // [batch, heads, tokens, D]
    float* out_lse;        // nullable
    const int* lens;
    int kv_heads, group, tokens, rows, parts, cache;
};

// One warp per query row: the parts' pairs merged in ascending order. A query before its sequence's first
// token (a free slot of the batch) reads out as zero with a log-sum-exp of -inf.
template <typename T, int D>
__global__ void __launch_bounds__(256) join_kernel(const JoinArgs a) {
    constexpr int E = D / 32;
    pdl_wait();
    pdl_trigger();
    const int64_t all = (int64_t)a.kv_heads * a.rows;
    const int64_t id = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (id >= all) return;
    const int head = (int)(id / a.rows), r = (int)(id % a.rows);
    const int t = r % a.tokens, g = r / a.tokens % a.group, b = r / a.tokens / a.group;
    const int64_t at = ((int64_t)b * a.kv_heads * a.group + head * a.group + g) * a.tokens + t;
    float top = -NB200_INF, sum = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    if (tokens_of(a.lens, b, a.cache) - a.tokens + t >= 0) {
        for (int i = 0; i < a.parts; ++i) {
            const float x = a.lse[i * all + id];
            top = x != x ? x : fmaxf(top, x);
        }
        for (int i = 0; i < a.parts; ++i) {
            const float x = a.lse[i * all + id];
            if (x == -NB200_INF) continue;  // no key of the part counts; its o is not written
            const float w = ex2(x - top);
            sum += w;
            const float* o = a.o + (i * all + id) * D + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += w * o[e];
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
struct Split {
    int tiles, splits, keys;  // row tiles of 16 mt rows, key splits and the keys of one
    int mt;
};

// Enough CTAs for four on every SM, but no split below 64 keys (a step for each warp).
Split plan_split(int64_t units, int64_t rows, int64_t keys) {
    Split s = {0, 0, 0, rows > 16 ? 2 : 1};
    s.tiles = (int)((rows + 16 * s.mt - 1) / (16 * s.mt));
    if (keys == 0) return s;
    const int64_t ctas = units * s.tiles, want = 4 * (int64_t)sm_count();
    int64_t splits = (want + ctas - 1) / ctas;
    splits = std::max<int64_t>(1, std::min(splits, (keys + 63) / 64));
    s.keys = (int)(((keys + splits - 1) / splits + 63) / 64 * 64);
    s.splits = (int)((keys + s.keys - 1) / s.keys);
    return s;
}

// Up to this many query rows of a key/value head meet the prefix in the part kernel above; more go to the
// tensor cores.
constexpr int kMmaRows = 32;

struct Plan {
    Split prefix, own;
    bool tensor;          // the prefix runs on the tensor cores
    int64_t rows, pairs;  // query rows of a key/value head; pairs of a part over all heads
};

Plan plan_of(const nb200_prefix_attn_args& a) {
    Plan p;
    const int64_t group = a.heads / a.kv_heads;
    p.rows = a.batch * group * a.tokens;
    p.tensor = a.prefix && p.rows > kMmaRows;
    p.prefix = p.tensor ? Split{0, tensor_splits(a.kv_heads, p.rows, a.prefix), 0, 0}
                        : plan_split(a.kv_heads, p.rows, a.prefix);
    p.own = plan_split(a.kv_heads * a.batch, group * a.tokens, a.cache);
    p.pairs = a.kv_heads * p.rows;
    return p;
}

SharedLimit g_shared[16];

template <typename T, int D, int MT, bool OWN>
int launch_part(const PartArgs& p, unsigned grid, SharedLimit& limit, cudaStream_t st) {
    constexpr uint32_t bytes = kWarps * kStages * 2 * kStepKeys * D * 2;
    static_assert(bytes >= kWarps * 16 * MT * D * 4, "the warps' results fit in the stages");
    if (const int rc = limit.raise("nb200_prefix_attention", part_kernel<T, D, MT, OWN>, bytes)) return rc;
    launch_pdl(part_kernel<T, D, MT, OWN>, grid, kWarps * 32, bytes, st, p);
    count_launch();
    return finish_launch("nb200_prefix_attention");
}

template <typename T, int D>
int launch_all(const nb200_prefix_attn_args& n, const nb200_attn_strides* s, const void* q, const void* pk,
               const void* pv, const void* k, const void* v, void* o, float* lse, float* work, SharedLimit* limits,
               cudaStream_t st) {
    const Plan plan = plan_of(n);
    const int parts = plan.prefix.splits + plan.own.splits;
    float* part_o = work;
    float* part_lse = work + (int64_t)parts * plan.pairs * D;
    PartArgs a = {};
    a.query = {q, s[0].batch, s[0].head, s[0].seq, (int)(n.heads / n.kv_heads), (int)n.tokens};
    a.lens = n.seq_lens;
    a.kv_heads = (int)n.kv_heads;
    a.rows = (int)plan.rows;
    a.sl2 = n.scale * 1.4426950408889634f;
    auto run = [&](const Split& sp, bool own, int64_t first) {
        if (!sp.splits) return (int)NB200_OK;
        a.tiles = sp.tiles, a.splits = sp.splits, a.split_keys = sp.keys;
        a.o = part_o + first * plan.pairs * D;
        a.lse = part_lse + first * plan.pairs;
        const int64_t grid = (int64_t)sp.tiles * sp.splits * n.kv_heads * (own ? n.batch : 1);
        if (grid > 0x7fffffffLL) {
            set_error("nb200_prefix_attention: the call exceeds the kernel's index range");
            return (int)NB200_ERR_CAPACITY;
        }
        if (own) {
            a.src = {k, v, s[3].batch, s[3].head, s[3].seq, s[4].batch, s[4].head, s[4].seq};
            a.keys = (int)n.cache, a.unit_rows = a.query.group * a.query.tokens;
            return sp.mt == 1 ? launch_part<T, D, 1, true>(a, (unsigned)grid, limits[0], st)
                              : launch_part<T, D, 2, true>(a, (unsigned)grid, limits[1], st);
        }
        a.src = {pk, pv, 0, s[1].head, s[1].seq, 0, s[2].head, s[2].seq};
        a.keys = (int)n.prefix, a.unit_rows = a.rows;
        return sp.mt == 1 ? launch_part<T, D, 1, false>(a, (unsigned)grid, limits[2], st)
                          : launch_part<T, D, 2, false>(a, (unsigned)grid, limits[3], st);
    };
    int rc;
    if (plan.tensor) {
        const TensorPart t = {a.query, a.kv_heads, a.rows, (int)n.prefix, plan.prefix.splits, a.sl2, part_o, part_lse};
        rc = launch_tensor_part(t, n.dtype, n.head_dim, pk, s[1], pv, s[2], st);
    } else {
        rc = run(plan.prefix, false, 0);
    }
    if (rc || (rc = run(plan.own, true, plan.prefix.splits))) return rc;
    const JoinArgs j = {part_o, part_lse, o, lse, n.seq_lens, a.kv_heads, a.query.group, a.query.tokens, a.rows, parts,
                        (int)n.cache};
    launch_pdl(join_kernel<T, D>, (unsigned)((plan.pairs + 7) / 8), 256, 0, st, j);
    count_launch();
    return finish_launch("nb200_prefix_attention");
}

}  // namespace
}  // namespace prefix

using namespace prefix;

int64_t prefix_attention_work_bytes(const nb200_prefix_attn_args& a) {
    const Plan p = plan_of(a);
    return (int64_t)(p.prefix.splits + p.own.splits) * p.pairs * (a.head_dim + 1) * 4;
}

int launch_prefix_attention(const nb200_prefix_attn_args& n, const nb200_attn_strides* s, const void* q, const void* pk,
                            const void* pv, const void* k, const void* v, void* o, float* lse, void* work,
                            cudaStream_t st) {
    float* w = static_cast<float*>(work);
    if (n.dtype == NB200_BF16)
        return n.head_dim == 128
                   ? launch_all<__nv_bfloat16, 128>(n, s, q, pk, pv, k, v, o, lse, w, g_shared, st)
                   : launch_all<__nv_bfloat16, 64>(n, s, q, pk, pv, k, v, o, lse, w, g_shared + 4, st);
    return n.head_dim == 128 ? launch_all<__half, 128>(n, s, q, pk, pv, k, v, o, lse, w, g_shared + 8, st)
                             : launch_all<__half, 64>(n, s, q, pk, pv, k, v, o, lse, w, g_shared + 12, st);
}

}  // namespace nb200
