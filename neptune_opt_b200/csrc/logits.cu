// What a server does to the logits of each sequence before it samples:
//
//   x = l > 0 ? l / repetition : l * repetition    for tokens of the sequence's history (prompt or output)
//   x -= frequency * count + presence              for tokens of its output, count = how often
//   x += bias                                      for the row's biased tokens (one that is named twice adds)
//   x /= temperature
//   x = -inf                                       where the row's bit mask forbids the token
//
// Nearly all tokens need only temperature and mask. The few that the history or the biases name are found first:
// name_kernel marks them in bit maps of the vocabulary (one CTA per row; integer atomics, no order changes the result) and
// leaves one entry for each, bucket by bucket of the vocabulary. sweep_kernel streams the logits through registers, tile by
// tile, and writes a tile's named tokens once more while the tile's logits are in L1 and its results in L2.
//
// The bound is HBM traffic, a read and a write of the logits. Two other ways were built and measured on bf16
// [512, 262144] with histories of 4096: counting in every tile of one kernel took 332 us (every tile reads the whole
// history and waits for it), rewriting the named tokens behind the sweep 157 us (1% of the tokens, but a third of the
// logits' sectors: they come from HBM a second time); this one takes 143. A mask alone, bf16 [512, 131072], takes 46 us,
// 5.9 TB/s.
#include <algorithm>

#include "common.cuh"
#include "launch.h"
#include "logits_rows.h"

namespace nb200 {
namespace {

struct Logits {
    nb200_logits_args n;
    void* out;
    int tiles;             // of a row
    int parts, range;      // CTAs of a row, each for `range` tokens of the vocabulary, that name tokens (0: there are none)
    int slots;             // of a table of tokens that come again
    int buckets, span;     // buckets of a row, each of 2^span tiles
    int64_t most;          // entries of a part, at most
    bool self;             // the sweep finds the named tokens by itself
    int* starts;           // [rows][parts][buckets + 1]: where a bucket's entries begin
    uint4* entries;        // [rows][parts][most]: token, count in the output, bias, whether the history has it
};

constexpr int kSweepThreads = 256, kSweepCtas = 6;  // an SM holds that many
constexpr int kVectors = 4;  // of a thread, in flight together
template <typename T> constexpr int kTileBits = 10 + (Elem<T>::V == 8 ? 3 : 2);
template <typename T> constexpr int kTile = 1 << kTileBits<T>;
static_assert(kTile<float> == kSweepThreads * kVectors * 4, "a tile is what a CTA's threads hold");

// A row's pointers, and how it is cut.
template <typename T>
struct Row : RowCut<(int)sizeof(T)> {
    const T* x;
    T* out;
    const int32_t* allowed;
    __device__ __forceinline__ Row(const Logits& a, int64_t row)
        : Row(a, static_cast<const T*>(a.n.logits) + row * a.n.stride_logits, static_cast<T*>(a.out) + row * a.n.vocab,
              a.n.allowed ? a.n.allowed + row * a.n.stride_allowed : nullptr) {}
    __device__ __forceinline__ Row(const Logits& a, const T* x, T* out, const int32_t* allowed)
        : RowCut<(int)sizeof(T)>(reinterpret_cast<uintptr_t>(x), reinterpret_cast<uintptr_t>(out), a.n.vocab), x(x), out(out),
          allowed(allowed) {}
    // V tokens from v on, of the blocks that hold them.
    __device__ __forceinline__ uint4 joined(int64_t v) const {
        const T* p = x + v - this->shift;
        const uint4 lo = ld_keep(p);
        uint4 hi = lo;  // not looked at where there is one block
        if (this->blocks() > 1) hi = ld_keep(p + Elem<T>::V);
        uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        const int bytes = this->shift * (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = bytes & 8 ? w[i + 2] : w[i];
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = bytes & 4 ? w[i + 1] : w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (bytes & 3));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// ------------------------------------------------------------------ the named tokens
constexpr int kNameThreads = 512;
// Counters of a bucket, for a warp to choose by its number: atomics on one address take their time one after another.
constexpr int kCopies = 8;
constexpr int kBiased = 1 << 30, kAlone = 1 << 29;  // beside a count: the token is biased, and not in the history
constexpr int kTogether = 8;  // tokens of a thread on their way together

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int dtype) {
    return dtype == NB200_I64 ? __ldg(static_cast<const long long*>(p) + i) : __ldg(static_cast<const int*>(p) + i);
}

// The finaliser of MurmurHash3 (Appleby): neighbours and arithmetic progressions spread like random numbers.
__device__ __forceinline__ unsigned scatter(unsigned h) {
    h = (h ^ (h >> 16)) * 0x85ebca6bu;
    h = (h ^ (h >> 13)) * 0xc2b2ae35u;
    return h ^ (h >> 16);
}

// The named tokens of a row, or of `range` tokens of its vocabulary. A token's first mention sets its bit and makes its
// entry, its first mention in the output sets another; only what comes again in the output, and what is biased, is kept
// in a hash table with linear probing that the host makes large enough. (With all of them in the table the searches, a
// warp's longest each time, made this kernel four times slower.) The kernel lives a few us (19.5 for 256 rows with
// histories of 4096), so latencies count: what a thread loads goes out together, before the lengths are known.
template <typename T>
__global__ void __launch_bounds__(kNameThreads) name_kernel(const Logits a) {
    extern __shared__ __align__(16) uint8_t smem[];
    const nb200_logits_args& n = a.n;
    const int biases = (int)n.biases, words = (a.range + 127) / 128 * 4;
    uint32_t* named = reinterpret_cast<uint32_t*>(smem);                  // [words]: bit v of the tokens that have an entry
    uint32_t* put_out = named + words;                                    // [words]: those in the output
    int* keys = reinterpret_cast<int*>(put_out + words);                  // [slots]: those tokens, -1 where empty
    int* again = keys + a.slots;                                          // [slots]: how often after the first time, and flags
    int* starts = again + a.slots;                                        // [buckets][kCopies], and the end
    int* bias_token = starts + a.buckets * kCopies + 1;
    float* bias_value = reinterpret_cast<float*>(bias_token + biases);
    __shared__ int warp_sum[kNameThreads / 32 + 1], any_again, bias_again;
    for (int i = threadIdx.x; i < words / 2; i += kNameThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0u, 0u, 0u, 0u);
    for (int i = threadIdx.x; i < a.slots; i += kNameThreads) keys[i] = -1, again[i] = 0;
    const int counters = a.buckets * kCopies;
    for (int i = threadIdx.x; i <= counters; i += kNameThreads) starts[i] = 0;
    if (threadIdx.x == 0) any_again = bias_again = 0;
    pdl_wait();
    pdl_trigger();
    const int64_t row = blockIdx.x / (unsigned)a.parts;
    const int low = (int)(blockIdx.x % (unsigned)a.parts) * a.range;
    const int64_t high = min((int64_t)low + a.range, n.vocab);
    const Row<T> r(a, row);
    const int64_t tokens = row * n.stride_tokens;
    auto here = [&](int64_t v) { return v >= low && v < high ? (int)v : -1; };
    int token[kTogether], bias[2];
    auto load = [&](int64_t i0) {
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            const int64_t i = i0 + k * kNameThreads;
            token[k] = i < n.history ? here(index_at(n.tokens, tokens + i, n.token_dtype)) : -1;
        }
    };
    load(threadIdx.x);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int i = threadIdx.x + k * kNameThreads;
        bias[k] = i < biases ? here(index_at(n.bias_index, row * n.stride_bias_index + i, n.bias_dtype)) : -1;
        if (i < biases) {
            bias_token[i] = bias[k];
            bias_value[i] = __ldg(n.bias_value + row * n.stride_bias_value + i);
        }
    }
    const int64_t len = n.token_lens ? min((int64_t)n.token_lens[row], n.history) : n.history;
    const int64_t prompt = n.prompt_lens ? n.prompt_lens[row] : 0;
    __syncthreads();

    const int shift = a.span + kTileBits<T>, copy = threadIdx.x / 32 % kCopies;
    auto place = [&](int v, int c) { return (max(v - r.head, 0) >> shift) * kCopies + c; };
    auto bit = [&](int v) { return 1u << ((v - low) & 31); };
    // Whether v's bit in a map was set; it is now.
    auto mark = [&](uint32_t* map, int v) { return (atomicOr(&map[(v - low) >> 5], bit(v)) & bit(v)) != 0u; };
    // An entry for v, if it has none yet: its rank in its bucket (of the copy that the warp counts in), else -1.
    auto enter = [&](int v) { return v < 0 || mark(named, v) ? -1 : atomicAdd(&starts[place(v, copy)], 1); };
    // The table's slot of v, which is put there unless only looked for; -1 where it is not.
    auto slot_of = [&](int v, bool put) {
        unsigned s = __umulhi(scatter((unsigned)v), (unsigned)a.slots);
        for (;; s = s + 1u == (unsigned)a.slots ? 0u : s + 1u) {
            int key = *reinterpret_cast<volatile int*>(keys + s);
            if (key == -1 && put) key = atomicCAS(&keys[s], -1, v);
            if (key == v || (key == -1 && put)) return (int)s;
            if (key == -1) return -1;
        }
    };
    int rank[kTogether], bias_rank[2];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) rank[k] = -1;
    for (int64_t i0 = threadIdx.x; i0 < len;) {
#pragma unroll
        for (int k = 0; k < kTogether; ++k) {
            const int64_t i = i0 + k * kNameThreads;
            if (i >= len) break;
            const int v = token[k];
            rank[k] = enter(v);
            if (v >= 0 && i >= prompt && mark(put_out, v)) {
                any_again = 1;
                atomicAdd(&again[slot_of(v, true)], 1);
            }
        }
        if ((i0 += kTogether * kNameThreads) < len) load(i0);
    }
    // A biased token's entry belongs to the history where that names it, else to the bias that makes it.
    if (biases) {
        int at[2] = {-1, -1};
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (bias[k] >= 0) {
                at[k] = slot_of(bias[k], true);
                if (atomicOr(&again[at[k]], kBiased) & kBiased) bias_again = 1;
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            bias_rank[k] = enter(bias[k]);
            if (bias_rank[k] >= 0) atomicOr(&again[at[k]], kAlone);
        }
    }
    __syncthreads();
    // Counts of the buckets to their first places: exclusive sums, kNameThreads counters at a time.
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int* out_starts = a.starts + blockIdx.x * (int64_t)(a.buckets + 1);
    int before = 0;
    for (int b0 = 0; b0 <= counters; b0 += kNameThreads) {
        const int b = b0 + threadIdx.x, own = b <= counters ? starts[b] : 0;
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) warp_sum[warp] = upto;
        __syncthreads();
        if (warp == 0) {
            const int sum = lane < kNameThreads / 32 ? warp_sum[lane] : 0;
            int all = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, all, o);
                if (lane >= o) all += x;
            }
            if (lane <= kNameThreads / 32) warp_sum[lane] = all - sum;  // the last one: of all
        }
        __syncthreads();
        const int base = before + warp_sum[warp];
        before += warp_sum[kNameThreads / 32];
        if (b <= counters) {  // a bucket's copies follow each other
            starts[b] = base + upto - own;
            if (b % kCopies == 0) out_starts[b / kCopies] = base + upto - own;
        }
        __syncthreads();
    }
    uint4* entries = a.entries + blockIdx.x * a.most;
    // The sum of a token's biases, in the order in which they are given.
    auto bias_of = [&](int v) {
        float sum = 0.f;
        for (int j = 0; j < biases; ++j)
            if (bias_token[j] == v) sum += bias_value[j];
        return sum;
    };
    const bool held = len <= kTogether * kNameThreads;  // every token's first finder still holds it
    auto leave = [&](int v, int rank, float b, bool history) {
        int count = (put_out[(v - low) >> 5] & bit(v)) ? 1 : 0;
        if (history && (any_again || biases)) {
            const int s = slot_of(v, false), c = s < 0 ? 0 : again[s];
            if (c & kAlone) return;
            if (c & kBiased) b = bias_of(v);
            count += c & ~(kBiased | kAlone);
        }
        // Without ranks any place of the bucket will do.
        const int at = held ? starts[place(v, copy)] + rank : atomicAdd(&starts[place(v, 0)], 1);
        entries[at] = make_uint4((uint32_t)v, (uint32_t)count, __float_as_uint(b), history);
    };
    if (held) {
#pragma unroll
        for (int k = 0; k < kTogether; ++k)
            if (rank[k] >= 0) leave(token[k], rank[k], 0.f, true);
    } else {
#pragma unroll 1
        for (int w = threadIdx.x; w < words; w += kNameThreads)
            for (uint32_t left = named[w]; left; left &= left - 1u) leave(low + 32 * w + __ffs(left) - 1, 0, 0.f, true);
    }
    if (biases) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (bias_rank[k] >= 0)
                leave(bias[k], bias_rank[k], bias_again ? bias_of(bias[k]) : bias_value[threadIdx.x + k * kNameThreads], false);
    }
}

// ------------------------------------------------------------------ the sweep
// The mask's bits of `count` tokens from v on, the first in bit 0.
__device__ __forceinline__ uint32_t mask_bits(const int32_t* allowed, int64_t v, int count) {
    const int shift = (int)(v & 31);
    const uint32_t lo = (uint32_t)__ldg(allowed + (v >> 5));
    return shift + count <= 32 ? lo >> shift : __funnelshift_r(lo, (uint32_t)__ldg(allowed + (v >> 5) + 1), shift);
}

// Where a sweep has a row's named tokens from: there are none; from name_kernel's entries; or, where that costs less, from
// the history itself, which every tile counts in shared memory.
enum Names { NONE, ENTRIES, SELF };
constexpr int kSelfTokens = 4096, kSelfBiases = kSweepThreads;
// SELF's word for a token: mentions in the history from kMention on, those in the output below, and between them whether it
// is biased, and whether more than once.
constexpr uint32_t kMention = 1u << 16, kWithBias = 1u << 14, kManyBiases = 1u << 15;
static_assert(kSelfTokens < (int)kWithBias, "a count's bits");

// x / d, d positive, by d's reciprocal. An fp32 quotient is corrected once by its remainder (Markstein's method), which leaves it
// rounded once; beside a 16-bit result's rounding of 2^-11 or 2^-8 the reciprocal's 2^-24 counts for nothing. Where fp32 does
// not hold the reciprocal (d below 2^-128) its largest value stands in: 0 / d stays 0.
template <typename T>
struct Divisor {
    float d, inv;
    __device__ __forceinline__ explicit Divisor(const float* p) : d(p ? *p : 1.f), inv(fminf(1.f / d, 0x1.fffffep127f)) {}
    __device__ __forceinline__ float operator()(float x) const {
        const float q = x * inv;
        if constexpr (sizeof(T) != 4) return q;
        const float exact = fmaf(fmaf(-q, d, x), inv, q);
        return exact == exact ? exact : q;  // beside an infinite x, q or d the remainder is NaN
    }
};

// Temperature and mask of a tile, and all of it for its named tokens. JOINED: rows of input and output are cut by different
// 16-byte boundaries (a vocabulary that is padded on the one side), and a vector of the output is joined from two. bf16
// [1024, 131071] of rows 131072 apart: 157 us, token by token 336; [256, 32001] 7.6 and 16.3.
template <typename T, Names NAMES, bool JOINED>
__global__ void __launch_bounds__(kSweepThreads, NAMES == SELF || JOINED ? 4 : kSweepCtas) sweep_kernel(const Logits a) {
    constexpr int V = Elem<T>::V;
    constexpr bool NAMED = NAMES == ENTRIES;
    pdl_wait();
    pdl_trigger();
    const nb200_logits_args& n = a.n;
    const int64_t row = blockIdx.x / (unsigned)a.tiles;
    const int tile = (int)(blockIdx.x % (unsigned)a.tiles);
    const Row<T> r(a, row);
    const int64_t lo = r.begin(tile, kTile<T>, n.vocab), hi = r.end(tile, kTile<T>, n.vocab);
    const int64_t body = r.body(tile, kTile<T>, n.vocab);
    const int vectors = JOINED ? r.vectors(body, hi, n.vocab) : (int)((hi - body) / V);
    uint4 raw[kVectors];
    uint32_t ok[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
        const int i = threadIdx.x + k * kSweepThreads;
        if (i < vectors) {
            if constexpr (JOINED) raw[k] = r.joined(body + (int64_t)i * V);
            else raw[k] = NAMES ? ld_keep(r.x + body + (int64_t)i * V) : ld_stream(r.x + body + (int64_t)i * V);
            ok[k] = r.allowed ? mask_bits(r.allowed, body + (int64_t)i * V, V) : ~0u;
        }
    }
    const Divisor<T> cool(n.temperature ? n.temperature + row : nullptr);
    // The entries are on their way with the logits.
    const int* starts = a.starts + row * a.parts * (a.buckets + 1) + (NAMED ? tile >> a.span : 0);
    const uint4* entries = a.entries + row * a.parts * a.most;
    int e0 = 0, e1 = 0;
    uint4 entry = make_uint4(0u, 0u, 0u, 0u);
    if (NAMED) {
        e0 = starts[0], e1 = starts[1];
        if (e0 + (int)threadIdx.x < e1) entry = entries[e0 + threadIdx.x];
    }
    // SELF: a word for each of the tile's tokens, those that the history names, in any order, and the biases.
    constexpr int kCounts = NAMES == SELF ? kTile<T> + 16 : 4;
    __shared__ __align__(16) uint32_t counts[kCounts];
    __shared__ uint16_t list[NAMES == SELF ? kSelfTokens : 1];
    __shared__ int bias_token[NAMES == SELF ? kSelfBiases : 1], listed;
    __shared__ float bias_value[NAMES == SELF ? kSelfBiases : 1];
    const int biases = (int)n.biases;
    int bias = -1;  // the thread's biased token, if no thread before it has the same
    if constexpr (NAMES == SELF) {
        constexpr int kAtOnce = 4;  // of a thread, on their way together
        const int size = (int)(hi - lo);
        auto here = [&](int64_t v) { return v >= lo && v < hi ? (int)(v - lo) : -1; };
        auto put = [&](int v) { list[atomicAdd(&listed, 1)] = (uint16_t)v; };
        int token[kAtOnce];
        auto load = [&](int64_t i0) {
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int64_t i = i0 + k * kSweepThreads;
                token[k] = i < n.history ? here(index_at(n.tokens, row * n.stride_tokens + i, n.token_dtype)) : -1;
            }
        };
        load(threadIdx.x);
        if (threadIdx.x < biases) {
            bias = here(index_at(n.bias_index, row * n.stride_bias_index + threadIdx.x, n.bias_dtype));
            bias_token[threadIdx.x] = bias;
            bias_value[threadIdx.x] = __ldg(n.bias_value + row * n.stride_bias_value + threadIdx.x);
        }
        const int64_t len = n.token_lens ? min((int64_t)n.token_lens[row], n.history) : n.history;
        const int64_t prompt = n.prompt_lens ? n.prompt_lens[row] : 0;
        for (int i = threadIdx.x * 4; i < size; i += kSweepThreads * 4)
            *reinterpret_cast<uint4*>(counts + i) = make_uint4(0u, 0u, 0u, 0u);
        if (threadIdx.x == 0) listed = 0;
        __syncthreads();
        for (int64_t i0 = threadIdx.x; i0 < len;) {
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int64_t i = i0 + k * kSweepThreads;
                if (i < len && token[k] >= 0 && atomicAdd(&counts[token[k]], kMention + (i >= prompt)) < kMention) put(token[k]);
            }
            if ((i0 += kAtOnce * kSweepThreads) < len) load(i0);
        }
        if (bias >= 0 && (atomicOr(&counts[bias], kWithBias) & kWithBias)) {
            atomicOr(&counts[bias], kManyBiases);
            bias = -1;
        }
    }
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
        const int i = threadIdx.x + k * kSweepThreads;
        if (i < vectors) {
            float f[V];
            Elem<T>::unpack(raw[k], f);
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = ok[k] >> j & 1u ? cool(f[j]) : -NB200_INF;
            const uint4 o = Elem<T>::pack(f);
            if (NAMES) *reinterpret_cast<uint4*>(r.out + body + (int64_t)i * V) = o;
            else st_stream(r.out + body + (int64_t)i * V, o);
        }
    }
    // What lies before the first vector and behind the last one, or all of it.
    auto allows = [&](int64_t v) { return !r.allowed || ((uint32_t)__ldg(r.allowed + (v >> 5)) >> (v & 31) & 1u); };
    auto one = [&](int64_t v) { r.out[v] = Elem<T>::from_f(allows(v) ? cool(Elem<T>::to_f(r.x[v])) : -NB200_INF); };
    for (int64_t v = lo + threadIdx.x; v < body; v += kSweepThreads) one(v);
    for (int64_t v = body + (int64_t)vectors * V + threadIdx.x; v < hi; v += kSweepThreads) one(v);
    if constexpr (NAMES != NONE) {
        const Divisor<T> rep(n.repetition ? n.repetition + row : nullptr);
        const float freq = n.frequency ? n.frequency[row] : 0.f, pres = n.presence ? n.presence[row] : 0.f;
        auto again = [&](int64_t v, uint32_t count, float bias, bool history) {
            float f = Elem<T>::to_f(r.x[v]);
            if (history) f = f > 0.f ? rep(f) : f * rep.d;
            if (count) f = f - freq * (float)count - pres;
            f = cool(f + bias);
            r.out[v] = Elem<T>::from_f(allows(v) ? f : -NB200_INF);
        };
        __syncthreads();  // the tile is written
        if constexpr (NAMED) {
#pragma unroll 1
            for (int part = 0;;) {
#pragma unroll 1
                for (int e = e0 + threadIdx.x; e < e1;) {
                    const int64_t v = entry.x;
                    // Not those of another tile of the bucket.
                    if (v >= lo && v < hi) again(v, entry.y, __uint_as_float(entry.z), entry.w);
                    if ((e += kSweepThreads) < e1) entry = entries[e];
                }
                if (++part == a.parts) break;
                starts += a.buckets + 1, entries += a.most;
                e0 = starts[0], e1 = starts[1];
                if (e0 + (int)threadIdx.x < e1) entry = entries[e0 + threadIdx.x];
            }
        } else {
            for (int e = threadIdx.x; e < listed; e += kSweepThreads) {
                const int v = list[e];
                if (!(counts[v] & kWithBias)) again(lo + v, counts[v] & (kWithBias - 1u), 0.f, true);
            }
            if (bias >= 0) {
                const uint32_t word = counts[bias];
                float sum = bias_value[threadIdx.x];
                if (word & kManyBiases) {  // in the order in which they are given
                    sum = 0.f;
                    for (int j = 0; j < biases; ++j)
                        if (bias_token[j] == bias) sum += bias_value[j];
                }
                again(lo + bias, word & (kWithBias - 1u), sum, word >= kMention);
            }
        }
    }
}

// ------------------------------------------------------------------ host side
constexpr int kMostBuckets = 256, kMostBiases = 1024;
constexpr int kMostTable = 5120, kMostRange = 1 << 18;  // tokens of a CTA that may come again; of its bit maps
constexpr int slots_of(int tokens) { return tokens * 8 / 5 + 8; }
constexpr int name_bytes(int range, int slots, int buckets, int biases) {
    return (range + 127) / 128 * 32 + slots * 8 + (buckets * kCopies + 1) * 4 + biases * 8;
}
static_assert(kMostBiases <= 2 * kNameThreads, "two biases a thread");
static_assert(name_bytes(kMostRange, slots_of(kMostTable + kMostBiases), kMostBuckets, kMostBiases) <= 200 << 10, "shared memory");
SharedLimit g_shared[3];

// Whether a grid holds that many CTAs a row.
int64_t held(const nb200_logits_args& n, int64_t ctas) {
    if (n.rows * ctas <= 0x7fffffffLL) return NB200_OK;
    set_error("nb200_penalize_logits: rows=%lld, vocab=%lld exceed the kernel's index range", (long long)n.rows,
              (long long)n.vocab);
    return NB200_ERR_CAPACITY;
}

// The shapes of a call, and the bytes of its workspace (negative: an error).
int64_t plan(Logits& a, int tile) {
    const nb200_logits_args& n = a.n;
    a.tiles = (int)((n.vocab + tile - 1) / tile);
    if (const int64_t rc = held(n, a.tiles)) return rc;
    const int64_t entries = std::min(n.history + n.biases, n.vocab);
    if (!entries) return 0;
    // A few tiles a row, or a few an SM: every tile counts the history itself, without a second launch and its workspace.
    // bf16 [8, 32000] on the GPU alone, histories of 512: 3.5 us, with both kernels 4.8; of 2048: 6.2 and 9.3, 512 rows 27.9
    // and 32.4. [32, 131072], 3.5 tiles an SM: histories of 512 5.9 and 5.3, of 4096 13.0 and 13.5; 128 rows, 14 tiles an
    // SM: 13.8 and 11.8, 32.9 and 24.3.
    a.self = n.history <= kSelfTokens && n.biases <= kSelfBiases && (a.tiles <= 4 || n.rows * a.tiles <= 6 * sm_count());
    if (a.self) return 0;
    // The table stays three eighths empty at least. Where it, or the bit maps, would be too large, the vocabulary is dealt
    // out to as many CTAs as it takes for every token of a range to fit, whatever the history holds.
    const int64_t fits = n.history / 2 <= kMostTable ? kMostRange : kMostTable;
    a.parts = (int)((n.vocab + fits - 1) / fits);
    if (const int64_t rc = held(n, a.parts)) return rc;
    a.range = (int)((n.vocab + a.parts - 1) / a.parts);
    a.slots = slots_of((int)std::min<int64_t>(n.history / 2, a.range) + (int)n.biases);
    a.most = std::min<int64_t>(entries, a.range);
    while (((a.tiles - 1) >> a.span) >= kMostBuckets) ++a.span;
    a.buckets = ((a.tiles - 1) >> a.span) + 1;
    return n.rows * a.parts * (a.most * 16 + (a.buckets + 1) * 4);
}

int tile_of(int dtype) { return dtype == NB200_F32 ? kTile<float> : kTile<__half>; }

template <typename T>
int launch(const Logits& a, SharedLimit& shared, cudaStream_t st) {
    const char* what = "nb200_penalize_logits";
    const nb200_logits_args& n = a.n;
    const unsigned grid = (unsigned)(n.rows * a.tiles);
    const bool alike = ((reinterpret_cast<uintptr_t>(n.logits) ^ reinterpret_cast<uintptr_t>(a.out)) & 15u) == 0 &&
                       (n.rows == 1 || (n.stride_logits - n.vocab) % Elem<T>::V == 0);
    if (a.parts) {
        const int most = name_bytes(kMostRange, slots_of(kMostTable + kMostBiases), kMostBuckets, kMostBiases);
        if (const int rc = shared.raise(what, name_kernel<T>, most)) return rc;
        launch_pdl(name_kernel<T>, (unsigned)(n.rows * a.parts), kNameThreads,
                   name_bytes(a.range, a.slots, a.buckets, (int)n.biases), st, a);
        count_launch();
        if (const int rc = finish_launch(what)) return rc;  // the sweep takes addresses from what the names' kernel leaves
        launch_pdl(alike ? sweep_kernel<T, ENTRIES, false> : sweep_kernel<T, ENTRIES, true>, grid, kSweepThreads, 0, st, a);
        count_launch();
    } else {
        auto kernel = a.self ? alike ? sweep_kernel<T, SELF, false> : sweep_kernel<T, SELF, true>
                             : alike ? sweep_kernel<T, NONE, false> : sweep_kernel<T, NONE, true>;
        launch_pdl(kernel, grid, kSweepThreads, 0, st, a);
        count_launch();
    }
    return finish_launch(what);
}

}  // namespace

int64_t logits_work_bytes(const nb200_logits_args& n) {
    Logits a = {n};
    return plan(a, tile_of(n.dtype));
}

int launch_logits(const nb200_logits_args& n, void* out, void* work, cudaStream_t st) {
    Logits a = {n, out};
    if (const int64_t rc = plan(a, tile_of(n.dtype)); rc < 0) return (int)rc;
    a.entries = static_cast<uint4*>(work);
    a.starts = reinterpret_cast<int*>(a.entries + n.rows * a.parts * a.most);
    if (n.dtype == NB200_F32) return launch<float>(a, g_shared[0], st);
    if (n.dtype == NB200_BF16) return launch<__nv_bfloat16>(a, g_shared[1], st);
    return launch<__half>(a, g_shared[2], st);
}

}  // namespace nb200
