// Divergence of a student's full-vocabulary distribution from a teacher of which only the top logits
// were kept, and its gradient.
//
//   p_j  = exp(t_j / T - Z)   Z = logsumexp over the row's kept t / T, or given by the caller
//   q    = softmax(x / T)     over the whole vocabulary
//   loss = sum_j p_j (log p_j - log q[idx_j])
//   dx_c = g / T * (mass q_c - sum_{j: idx_j = c} p_j),   mass = sum_j p_j
//
// An index outside [0, vocab) marks an entry that was not kept. A row without kept entries has loss 0
// and gradient 0 whatever its logits hold.
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "fastmath.cuh"
#include "launch.h"

namespace nb200 {
namespace {

constexpr int kMaxTop = 256;  // entries a row may keep: one per thread of its CTA
constexpr float kL2e = 1.4426950408889634f;

struct Row {  // what both directions read of the teacher
    const void* teacher;
    const void* index;
    int teacher_dtype, index_dtype, top;
    int64_t teacher_stride, index_stride, vocab;
    float inv_t;

    // t_j / T of entry j, and its index; index -1 when the entry was not kept.
    __device__ __forceinline__ float logit(int64_t row, int j) const {
        const int64_t i = row * teacher_stride + j;
        const float t = teacher_dtype == NB200_F32    ? static_cast<const float*>(teacher)[i]
                        : teacher_dtype == NB200_BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(teacher)[i])
                                                      : __half2float(static_cast<const __half*>(teacher)[i]);
        return t * inv_t;
    }
    __device__ __forceinline__ int64_t at(int64_t row, int j) const {
        const int64_t i = row * index_stride + j;
        const int64_t c = index_dtype == NB200_I64 ? static_cast<const int64_t*>(index)[i]
                                                   : (int64_t) static_cast<const int32_t*>(index)[i];
        return c >= 0 && c < vocab ? c : -1;
    }
};

// Elements before the first 16-byte boundary at or after p.
template <typename T>
__device__ __forceinline__ int64_t lead(const T* p) {
    return (int64_t)((16 - (reinterpret_cast<uintptr_t>(p) & 15u)) & 15u) / (int64_t)sizeof(T);
}

// Running state of a row: s = sum of 2^(x scale - c) with scale = log2(e) / T and c the largest x scale so far,
// rounded; c is the exact shift of every term, so its rounding costs nothing. A row of -inf alone keeps
// c = -inf and s = 0.
struct LogSum {
    float c = -HUGE_VALF, s = 0.f;
    __device__ __forceinline__ static float shift(float c) { return c == -NB200_INF ? 0.f : c; }
    __device__ __forceinline__ void merge(float c2, float s2) {
        const float t = fmaxf(c, c2), m = shift(t);
        s = s * ex2_ftz(c - m) + s2 * ex2_ftz(c2 - m);
        c = t;
    }
    __device__ __forceinline__ void merge_warp(int from) {
        for (int o = from; o > 0; o >>= 1) {
            const float c2 = __shfl_xor_sync(0xffffffffu, c, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
            merge(c2, s2);
        }
    }
    // E logits (E even): half an instruction each for the maximum, the exponent and the sum (three-input max,
    // packed pairs), one exponential each, one more for the whole batch.
    template <int E>
    __device__ __forceinline__ void add(const float* x, float scale) {
        float t0 = x[0], t1 = x[1];
#pragma unroll
        for (int i = 2; i + 3 < E; i += 4) {
            t0 = max3(t0, x[i], x[i + 1]);
            t1 = max3(t1, x[i + 2], x[i + 3]);
        }
        if (E % 4 == 0) t0 = max3(t0, x[E - 2], x[E - 1]);
        const float top = fmaxf(c, fmaxf(t0, t1) * scale), m = shift(top);
        const uint64_t scale2 = f2(scale, scale), m2 = f2(-m, -m);
        uint64_t a0 = f2(s * ex2_ftz(c - m), 0.f), a1 = 0;
#pragma unroll
        for (int i = 0; i < E; i += 2) {
            const uint64_t e = fma2(f2(x[i], x[i + 1]), scale2, m2);
            const uint64_t p = f2(ex2_ftz(f2lo(e)), ex2_ftz(f2hi(e)));
            if (i & 2) a1 = add2(a1, p);
            else a0 = add2(a0, p);
        }
        const uint64_t a = add2(a0, a1);
        s = f2lo(a) + f2hi(a);
        c = top;
    }
    __device__ __forceinline__ void add_one(float x, float scale) { merge(x * scale, x == -NB200_INF ? 0.f : 1.f); }
};

// ------------------------------------------------------------------ forward
// One cluster of CTAs per row (one CTA when there are rows enough): each folds a share of the row's 16-byte
// vectors, the states meet in the first CTA's shared memory, and that CTA's first warp takes the kept
// entries, which were fetched before the fold. One pass over the logits, no scratch.
// 256 threads: bf16 [4096, 131072] 164 us (6.5 TB/s); 191 us with 512 and 175 us with 128.
constexpr int kFwdThreads = 256;
constexpr int kMaxCluster = 16;

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Stores v at p's place in the shared memory of the cluster's first CTA.
__device__ __forceinline__ void store_first(float* p, float v) {
    uint32_t to;
    const uint32_t local = static_cast<uint32_t>(__cvta_generic_to_shared(p));
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(local));
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to), "f"(v) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kFwdThreads)
    distill_fwd_kernel(const T* x, int64_t stride, Row r, const float* teacher_lse, float* loss, float* stats) {
    constexpr int V = Elem<T>::V, U = 4;  // U vectors in flight per thread
    __shared__ float ec[32], es[32], cc[kMaxCluster], cs[kMaxCluster], teach[kMaxTop], stud[kMaxTop];
    const uint32_t rank = cluster_rank(), size = cluster_size();
    const int64_t row = blockIdx.x / size;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const T* xr = x + row * stride;
    // The kept entries, one per thread: t_j / T (-inf: not kept, its probability is 0) and x / T.
    if (rank == 0 && t < r.top) {
        const int64_t at = r.at(row, t);
        teach[t] = at >= 0 ? r.logit(row, t) : -NB200_INF;
        stud[t] = at >= 0 ? Elem<T>::to_f(xr[at]) * r.inv_t : 0.f;
    }
    const float scale = r.inv_t * kL2e;
    LogSum acc;
    const int64_t head = min(lead(xr), r.vocab), nv = (r.vocab - head) / V, tail = head + nv * V;
    int64_t v0, v1;
    split_range(nv, size, rank, v0, v1);
    const uint4* p = reinterpret_cast<const uint4*>(xr + head);
    int64_t v = v0 + t;
    for (; v + (U - 1) * kFwdThreads < v1; v += U * kFwdThreads) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k) u[k] = ld_stream(p + v + k * kFwdThreads);
        float f[U * V];
#pragma unroll
        for (int k = 0; k < U; ++k) Elem<T>::unpack(u[k], f + k * V);
        acc.add<U * V>(f, scale);
    }
    for (; v < v1; v += kFwdThreads) {
        float f[V];
        Elem<T>::unpack(ld_stream(p + v), f);
        acc.add<V>(f, scale);
    }
    if (rank == 0) {  // what lies outside the vectors: fewer than 2 V elements
        if (t < head) acc.add_one(Elem<T>::to_f(xr[t]), scale);
        else if (t >= 32 && tail + t - 32 < r.vocab) acc.add_one(Elem<T>::to_f(xr[tail + t - 32]), scale);
    }
    acc.merge_warp(16);
    if (lane == 0) {
        ec[warp] = acc.c;
        es[warp] = acc.s;
    }
    __syncthreads();
    if (warp == 0) {
        acc = LogSum{};
        if (lane < kFwdThreads / 32) acc.merge(ec[lane], es[lane]);
        acc.merge_warp(16);
        if (size > 1 && lane == 0) {
            store_first(&cc[rank], acc.c);
            store_first(&cs[rank], acc.s);
        }
    }
    if (size > 1) {
        __syncwarp();
        cluster_sync();
        if (rank != 0) return;
        if (warp == 0) {
            acc = LogSum{};
            if (lane < size) acc.merge(cc[lane], cs[lane]);
            acc.merge_warp(16);
        }
    }
    if (warp != 0) return;
    // The first warp takes the kept entries.
    const float lse = (acc.c + log2f(acc.s)) * 0.69314718055994531f;
    float z;
    if (teacher_lse) {
        z = teacher_lse[row];
    } else {
        float top = -NB200_INF, sum = 0.f;
        for (int j = lane; j < r.top; j += 32) top = fmaxf(top, teach[j]);
        top = warp_max(top);
        const float c = LogSum::shift(top);
        for (int j = lane; j < r.top; j += 32) sum += expf(teach[j] - c);
        z = c + logf(warp_sum(sum));
    }
    float mass = 0.f, l = 0.f;
    for (int j = lane; j < r.top; j += 32) {
        if (teach[j] == -NB200_INF) continue;
        const float q = expf(teach[j] - z);
        mass += q;
        if (q != 0.f) l += q * ((teach[j] - z) - (stud[j] - lse));
    }
    mass = warp_sum(mass);
    l = warp_sum(l);
    if (lane == 0) {
        loss[row] = l;
        stats[3 * row] = lse;
        stats[3 * row + 1] = z;
        stats[3 * row + 2] = mass;
    }
}

// CTAs per row: enough for four on every SM, no more than leaves each at least two rounds of loads. Every
// further CTA of a row pays the merge again: bf16 [512, 262144] 54.0, 52.3, 53.5 us with 1, 2, 4;
// [1024, 50001] 24.9, 29.1, 45.3 us; [160, 131072] 20.5, 15.6, 14.7 us.
template <typename T>
int cluster_for(int64_t rows, int64_t vocab) {
    const int64_t round = (int64_t)kFwdThreads * Elem<T>::V;
    int c = 1;
    while (c < kMaxCluster && rows * c < 4 * sm_count() && vocab >= 2 * c * round) c *= 2;
    return c;
}

// ------------------------------------------------------------------ backward
// One CTA per row and chunk of columns: write the softmax part of the chunk, then the chunk's kept
// columns once more with their probabilities taken off.
constexpr int kBwdThreads = 256;
constexpr int kChunk = 16384;  // columns
static_assert(kMaxTop <= kBwdThreads && kMaxTop <= kFwdThreads, "one kept entry per thread");

template <typename T>
__global__ void __launch_bounds__(kBwdThreads)
    distill_bwd_kernel(const float* grad, int64_t grad_stride, const T* x, int64_t stride, Row r, const float* stats,
                       int chunks, T* dx) {
    constexpr int V = Elem<T>::V, U = 4;
    __shared__ int64_t at[kMaxTop];
    __shared__ float p[kMaxTop];
    const int64_t row = blockIdx.x / chunks, c0 = (int64_t)(blockIdx.x % chunks) * kChunk;
    const int64_t c1 = min(c0 + kChunk, r.vocab);
    const int t = threadIdx.x;
    const float lse = stats[3 * row], z = stats[3 * row + 1], mass = stats[3 * row + 2];
    const float w = grad[row * grad_stride] * r.inv_t;
    const T* xr = x + row * stride;
    T* dr = dx + row * r.vocab;
    const int64_t mine = t < r.top ? r.at(row, t) : -1;
    const float pm = mine >= 0 ? expf(r.logit(row, t) - z) : 0.f;
    if (t < r.top) {
        at[t] = mine;
        p[t] = pm;
    }
    const bool any = __syncthreads_or(mine >= 0);
    const float wm = w * mass;
    // w mass q, the difference taken before the change of base so that large logits keep their digits; a
    // row without kept entries is 0 whatever its logits hold.
    auto soft = [&](float f) { return any ? wm * ex2_ftz(fmaf(f, r.inv_t, -lse) * kL2e) : 0.f; };
    const int64_t head = min(lead(dr + c0), c1 - c0);
    const bool together = lead(xr + c0) == lead(dr + c0);  // both sides meet the same 16-byte boundaries
    const int64_t nv = together ? (c1 - c0 - head) / V : 0;
    const uint4* src = reinterpret_cast<const uint4*>(xr + c0 + head);
    uint4* dst = reinterpret_cast<uint4*>(dr + c0 + head);
    auto one = [&](const uint4& u, int64_t v) {
        float f[V];
        Elem<T>::unpack(u, f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = soft(f[e]);
        __stcs(dst + v, Elem<T>::pack(f));
    };
    int64_t v = t;
    for (; v + (U - 1) * kBwdThreads < nv; v += U * kBwdThreads) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k) u[k] = ld_stream(src + v + k * kBwdThreads);
#pragma unroll
        for (int k = 0; k < U; ++k) one(u[k], v + k * kBwdThreads);
    }
    for (; v < nv; v += kBwdThreads) one(ld_stream(src + v), v);
    if (t < head) dr[c0 + t] = Elem<T>::from_f(soft(Elem<T>::to_f(xr[c0 + t])));
    for (int64_t c = c0 + head + nv * V + t; c < c1; c += kBwdThreads)
        dr[c] = Elem<T>::from_f(soft(Elem<T>::to_f(xr[c])));
    __syncthreads();
    // By the first entry that names a column: entries of one column add in order.
    if (mine >= c0 && mine < c1) {
        float sum = 0.f;
        bool first = true;
        for (int j = 0; j < r.top; ++j) {
            if (at[j] != mine) continue;
            first = first && j >= t;
            sum += p[j];
        }
        if (first) dr[mine] = Elem<T>::from_f(soft(Elem<T>::to_f(xr[mine])) - w * sum);
    }
}

Row make_row(const nb200_distill_args& a) {
    Row r;
    r.teacher = a.teacher;
    r.index = a.index;
    r.teacher_dtype = a.teacher_dtype;
    r.index_dtype = a.index_dtype;
    r.top = (int)a.top;
    r.teacher_stride = a.stride_teacher;
    r.index_stride = a.stride_index;
    r.vocab = a.vocab;
    r.inv_t = (float)(1.0 / a.temperature);
    return r;
}

int check_sizes(const char* what, const nb200_distill_args& a) {
    if (a.top > kMaxTop) {
        set_error("%s: %lld kept logits per row exceed the kernel's %d", what, (long long)a.top, kMaxTop);
        return NB200_ERR_CAPACITY;
    }
    if (a.rows * ((a.vocab + kChunk - 1) / kChunk) > 0x7fffffffLL || a.rows > 0x7fffffffLL / kMaxCluster) {
        set_error("%s: %lld rows of %lld exceed the kernel's index range", what, (long long)a.rows,
                  (long long)a.vocab);
        return NB200_ERR_CAPACITY;
    }
    return NB200_OK;
}

}  // namespace

int launch_distill_fwd(const nb200_distill_args& a, const float* teacher_lse, float* loss, float* stats,
                       cudaStream_t st) {
    const int rc = check_sizes("nb200_distill_loss", a);
    if (rc) return rc;
    const Row r = make_row(a);
    auto go = [&](auto* x) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(x)>>;
        const auto kernel = distill_fwd_kernel<T>;
        const int size = cluster_for<T>(a.rows, a.vocab);
        if (size > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(a.rows * size));
        cfg.blockDim = dim3(kFwdThreads);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, kernel, x, a.stride_x, r, teacher_lse, loss, stats);
    };
    if (a.dtype == NB200_F32) go(static_cast<const float*>(a.x));
    else if (a.dtype == NB200_BF16) go(static_cast<const __nv_bfloat16*>(a.x));
    else go(static_cast<const __half*>(a.x));
    count_launch();
    return finish_launch("nb200_distill_loss");
}

int launch_distill_bwd(const nb200_distill_args& a, const float* grad, int64_t stride_grad, const float* stats,
                       void* dx, cudaStream_t st) {
    const int rc = check_sizes("nb200_distill_loss_bwd", a);
    if (rc) return rc;
    const Row r = make_row(a);
    auto go = [&](auto* d) {
        using T = std::remove_pointer_t<decltype(d)>;
        const int chunks = (int)((a.vocab + kChunk - 1) / kChunk);
        distill_bwd_kernel<T><<<(unsigned)(a.rows * chunks), kBwdThreads, 0, st>>>(
            grad, stride_grad, static_cast<const T*>(a.x), a.stride_x, r, stats, chunks, d);
    };
    if (a.dtype == NB200_F32) go(static_cast<float*>(dx));
    else if (a.dtype == NB200_BF16) go(static_cast<__nv_bfloat16*>(dx));
    else go(static_cast<__half*>(dx));
    count_launch();
    return finish_launch("nb200_distill_loss_bwd");
}

}  // namespace nb200
