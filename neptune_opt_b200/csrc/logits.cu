// What a server does to the logits of each sequence before it samples, in one pass:
//
//   x = l > 0 ? l / repetition : l * repetition    for tokens of the sequence's history (prompt or output)
//   x -= frequency * count + presence              for tokens of its output, count = how often
//   x += bias                                      for the row's biased tokens (one that is named twice adds)
//   x /= temperature
//   x = -inf                                       where the row's bit mask forbids the token
//
// A CTA owns one chunk of one row's vocabulary. It counts the row's history tokens of its chunk in shared
// memory (integer atomics: no order changes the result), streams the chunk through registers and then
// redoes the few biased tokens. The bound is HBM traffic, a read and a write of the logits; each chunk
// reads the whole history again, from L2.
#include "common.cuh"
#include "launch.h"

namespace nb200 {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kPrompt = 0x80000000u;  // beside the count of output tokens: the token is in the prompt

struct Logits {
    nb200_logits_args n;
    void* out;
    int chunk, chunks;
};

struct RowParams {
    float repetition, presence, frequency, inv_temperature;
};

__device__ __forceinline__ int64_t index_at(const void* p, int64_t i, int dtype) {
    return dtype == NB200_I64 ? static_cast<const int64_t*>(p)[i] : static_cast<const int32_t*>(p)[i];
}

// Penalties of one logit; c = its count and prompt bit.
__device__ __forceinline__ float penalize(float x, uint32_t c, const RowParams& p) {
    if (c == 0) return x;
    x = x > 0.f ? x / p.repetition : x * p.repetition;
    const uint32_t n = c & ~kPrompt;
    return n ? x - p.frequency * (float)n - p.presence : x;
}

// 32 mask bits from token v on (those past the last word are 0).
__device__ __forceinline__ uint32_t mask_bits(const int32_t* allowed, int64_t v, int64_t words) {
    const int64_t w = v >> 5;
    const uint32_t lo = (uint32_t)__ldg(allowed + w), hi = w + 1 < words ? (uint32_t)__ldg(allowed + w + 1) : 0u;
    return __funnelshift_r(lo, hi, (uint32_t)v & 31u);
}

template <typename T, bool HISTORY>
__global__ void __launch_bounds__(kThreads) logits_kernel(const Logits a) {
    constexpr int V = Elem<T>::V;
    extern __shared__ uint32_t counts[];
    pdl_wait();
    pdl_trigger();
    const nb200_logits_args& n = a.n;
    const int64_t row = blockIdx.x / (unsigned)a.chunks;
    const int part = (int)(blockIdx.x % (unsigned)a.chunks);
    const T* x = static_cast<const T*>(n.logits) + row * n.stride_logits;
    T* out = static_cast<T*>(a.out) + row * n.vocab;
    const int32_t* allowed = n.allowed ? n.allowed + row * n.stride_allowed : nullptr;
    const int64_t words = (n.vocab + 31) / 32;
    // Whole vectors start at the first 16-byte boundary of the row, where input and output share it.
    const uint32_t skew = (uint32_t)reinterpret_cast<uintptr_t>(x) & 15u;
    const bool vec = skew == ((uint32_t)reinterpret_cast<uintptr_t>(out) & 15u);
    const int64_t head = min((int64_t)((16u - skew) & 15u) / (int64_t)sizeof(T), n.vocab);
    const int64_t lo = part ? head + (int64_t)part * a.chunk : 0;
    const int64_t hi = min(head + (int64_t)(part + 1) * a.chunk, n.vocab);
    if (lo >= hi) return;

    RowParams p;
    p.repetition = n.repetition ? n.repetition[row] : 1.f;
    p.presence = n.presence ? n.presence[row] : 0.f;
    p.frequency = n.frequency ? n.frequency[row] : 0.f;
    p.inv_temperature = n.temperature ? 1.f / n.temperature[row] : 1.f;

    if constexpr (HISTORY) {
        for (int i = threadIdx.x; i < (int)(hi - lo); i += kThreads) counts[i] = 0u;
        __syncthreads();
        const int64_t len = n.token_lens ? max((int64_t)0, min((int64_t)n.token_lens[row], n.history)) : n.history;
        const int64_t prompt = n.prompt_lens ? n.prompt_lens[row] : 0;
        for (int64_t i = threadIdx.x; i < len; i += kThreads) {
            const int64_t v = index_at(n.tokens, row * n.stride_tokens + i, n.token_dtype);
            if (v >= lo && v < hi) {
                if (i < prompt) atomicOr(&counts[v - lo], kPrompt);
                else atomicAdd(&counts[v - lo], 1u);
            }
        }
        __syncthreads();
    }
    auto one = [&](int64_t v, float bias) {
        float f = Elem<T>::to_f(x[v]);
        if constexpr (HISTORY) f = penalize(f, counts[v - lo], p);
        f = (f + bias) * p.inv_temperature;
        if (allowed && !((uint32_t)allowed[v >> 5] >> (v & 31) & 1u)) f = -NB200_INF;
        return Elem<T>::from_f(f);
    };
    if (vec) {
        const int64_t body = part ? lo : head;
        const int vectors = (int)((hi - body) / V);
        if (!part)
            for (int64_t v = threadIdx.x; v < head; v += kThreads) out[v] = one(v, 0.f);
        for (int64_t v = body + (int64_t)vectors * V + threadIdx.x; v < hi; v += kThreads) out[v] = one(v, 0.f);
        for (int i = threadIdx.x; i < vectors; i += kThreads) {
            const int64_t v = body + (int64_t)i * V;
            const uint4 raw = ld_stream(x + v);
            const uint32_t ok = allowed ? mask_bits(allowed, v, words) : ~0u;
            float f[V];
            Elem<T>::unpack(raw, f);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (HISTORY) f[j] = penalize(f[j], counts[v - lo + j], p);
                f[j] = (ok >> j & 1u) ? f[j] * p.inv_temperature : -NB200_INF;
            }
            st_stream(out + v, Elem<T>::pack(f));
        }
    } else {
        for (int64_t v = lo + threadIdx.x; v < hi; v += kThreads) out[v] = one(v, 0.f);
    }
    if (n.biases) {
        __syncthreads();  // the chunk is written
        const int64_t at = row * n.stride_bias_index, val = row * n.stride_bias_value;
        for (int64_t i = threadIdx.x; i < n.biases; i += kThreads) {
            const int64_t v = index_at(n.bias_index, at + i, n.bias_dtype);
            if (v < lo || v >= hi) continue;
            // The first entry of a token adds all of them, in their order.
            bool first = true;
            for (int64_t j = 0; j < i && first; ++j) first = index_at(n.bias_index, at + j, n.bias_dtype) != v;
            if (!first) continue;
            float bias = n.bias_value[val + i];
            for (int64_t j = i + 1; j < n.biases; ++j)
                if (index_at(n.bias_index, at + j, n.bias_dtype) == v) bias += n.bias_value[val + j];
            out[v] = one(v, bias);
        }
    }
}

SharedLimit g_shared[3];

template <typename T>
int launch(Logits a, SharedLimit& shared, cudaStream_t st) {
    const char* what = "nb200_penalize_logits";
    const nb200_logits_args& n = a.n;
    // Chunks of 16384 tokens (64 KB of counts, three CTAs an SM), shorter ones while the CTAs do not fill the GPU.
    int chunk = 16384;
    while (chunk > 2048 && n.rows * ((n.vocab + chunk - 1) / chunk) < 3 * (int64_t)sm_count()) chunk /= 2;
    a.chunk = chunk;
    a.chunks = (int)((n.vocab + chunk - 1) / chunk);
    if (n.rows * a.chunks > 0x7fffffffLL) {
        set_error("%s: rows=%lld, vocab=%lld exceed the kernel's index range", what, (long long)n.rows, (long long)n.vocab);
        return NB200_ERR_CAPACITY;
    }
    const unsigned grid = (unsigned)(n.rows * a.chunks);
    if (n.history) {
        const uint32_t bytes = (16384 + 16) * 4;
        if (const int rc = shared.raise(what, logits_kernel<T, true>, bytes)) return rc;
        launch_pdl(logits_kernel<T, true>, grid, kThreads, (size_t)(chunk + 16) * 4, st, a);
    } else {
        launch_pdl(logits_kernel<T, false>, grid, kThreads, 0, st, a);
    }
    count_launch();
    return finish_launch(what);
}

}  // namespace

int launch_logits(const nb200_logits_args& n, void* out, cudaStream_t st) {
    const Logits a = {n, out, 0, 0};
    if (n.dtype == NB200_F32) return launch<float>(a, g_shared[0], st);
    if (n.dtype == NB200_BF16) return launch<__nv_bfloat16>(a, g_shared[1], st);
    return launch<__half>(a, g_shared[2], st);
}

}  // namespace nb200
