// Divergence of a student's full-vocabulary distribution from a teacher of which only the top logits
// were kept, and its gradient.
//
//   p_j  = exp(t_j / T - Z)   Z = logsumexp over the row's kept t / T, or given by the caller
//   q    = softmax(x / T)     over the whole vocabulary
//   loss = sum_j p_j (log p_j - log q[idx_j])
//   dx_c = g / T * (mass q_c - sum_{j: idx_j = c} p_j),   mass = sum_j p_j
//
// An index outside [0, vocab) marks an entry that was not kept, and so does a teacher logit of -inf: its
// probability is 0. A row without kept entries has loss 0 and gradient 0 whatever its logits hold.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "fastmath.cuh"
#include "launch.h"

namespace nb200 {
namespace {

constexpr int kMaxTop = 256;  // entries a row may keep
constexpr float kL2e = 1.4426950408889634f;
// A CTA of 256 threads takes a row, or a chunk of one (bf16 [4096, 131072] forward 164 us, 6.5 TB/s; 191 us with 512
// and 175 us with 128). Narrow rows, where there are many, go to a warp each, kWarpRows of them in a CTA: there a CTA's
// launch and barriers count for more than its loads (CTA -> warp, forward: bf16 [8192, 1000] 39 -> 15 us,
// [8192, 10007] 62 -> 40, [8192, 32001] 105 -> 99, fp32 [8192, 32000] 152 -> 164; backward: bf16 [8192, 1000] 30 -> 19,
// [8192, 10007] 81 -> 89). With fewer rows the warps leave SMs idle: [1200, 5000] 9.7 -> 8.1 and 10.0 -> 8.7 us, but
// [600, 5000] 6.1 -> 6.8 and 5.5 -> 7.7 us.
constexpr int kWide = 256, kWarpRows = 8;
constexpr int64_t kNarrowFwd = 65536, kNarrowBwd = 16384;  // bytes of a row

bool narrow_rows(const nb200_distill_args& a, int64_t most, int64_t esize) {
    return a.vocab * esize <= most && a.vocab <= 5 * a.rows;
}

// A barrier of the threads that share a row.
template <int kThreads>
__device__ __forceinline__ void row_sync() {
    if constexpr (kThreads == 32) __syncwarp();
    else __syncthreads();
}

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
// rounded up; c is the exact shift of every term, so its rounding costs nothing, and no exponent is positive: rounded
// to nearest, it can fall short of the product by more than fp32's 2^128 holds where a thread has met nothing but a
// mask's -1e10 or below. A row of -inf alone keeps c = -inf and s = 0.
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
        const float top = fmaxf(c, __fmul_ru(fmaxf(t0, t1), scale)), m = shift(top);
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
    __device__ __forceinline__ void add_one(float x, float scale) { merge(__fmul_ru(x, scale), x == -NB200_INF ? 0.f : 1.f); }
};

// Rows whose largest logit is that far from 0 (in base 2) are folded once more, by one warp: there c's own rounding
// amounts to something. A mask that leaves a row nothing makes such rows, training does not.
constexpr float kFar = 1048576.f;

// The largest logit over T, and log sum exp((x - largest) / T), of a row with a finite largest logit; else NaN.
template <typename T>
__device__ __noinline__ float2 far_row(const T* x, int64_t vocab, float inv_t, int lane) {
    float top = -NB200_INF, sum = 0.f;
#pragma unroll 8
    for (int64_t i = lane; i < vocab; i += 32) top = fmaxf(top, Elem<T>::to_f(x[i]));
    top = warp_max(top);
#pragma unroll 8
    for (int64_t i = lane; i < vocab; i += 32) sum += expf((Elem<T>::to_f(x[i]) - top) * inv_t);
    return make_float2(__fmul_rn(top, inv_t), logf(warp_sum(sum)));
}

// ------------------------------------------------------------------ forward
// One cluster of CTAs per row (one CTA, or a warp, when there are rows enough): each folds a share of the row's 16-byte
// vectors, the states meet in the first CTA's shared memory, and that CTA's first warp takes the kept
// entries, which were fetched before the fold. One pass over the logits, no scratch.
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

template <typename T, int kThreads>
__global__ void __launch_bounds__(kWide)
    distill_fwd_kernel(const T* x, int64_t rows, int64_t stride, Row r, const float* teacher_lse, float* loss,
                       float* stats) {
    constexpr int V = Elem<T>::V, U = 4, kRows = kWide / kThreads;  // U vectors in flight per thread
    __shared__ float ec[32], es[32], cc[kMaxCluster], cs[kMaxCluster], teach_[kRows][kMaxTop], stud_[kRows][kMaxTop];
    const int sub = kRows > 1 ? threadIdx.y : 0;  // which of the CTA's rows
    float *teach = teach_[sub], *stud = stud_[sub];
    const uint32_t rank = kRows > 1 ? 0 : cluster_rank(), size = kRows > 1 ? 1 : cluster_size();
    const int64_t row = (int64_t)(blockIdx.x / size) * kRows + sub;
    if (kRows > 1 && row >= rows) return;
    if (size > 1) cluster_arrive_started();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const T* xr = x + row * stride;
    // The kept entries: t_j / T (-inf: not kept, its probability is 0) and x / T.
    for (int j = rank == 0 ? t : r.top; j < r.top; j += kThreads) {
        const int64_t at = r.at(row, j);
        teach[j] = at >= 0 ? r.logit(row, j) : -NB200_INF;
        stud[j] = at >= 0 ? Elem<T>::to_f(xr[at]) * r.inv_t : 0.f;
    }
    const float scale = r.inv_t * kL2e;
    LogSum acc;
    const int64_t head = min(lead(xr), r.vocab), nv = (r.vocab - head) / V, tail = head + nv * V;
    int64_t v0, v1;
    split_range(nv, size, rank, v0, v1);
    const uint4* p = reinterpret_cast<const uint4*>(xr + head);
    int64_t v = v0 + t;
    for (; v + (U - 1) * kThreads < v1; v += U * kThreads) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k) u[k] = ld_stream(p + v + k * kThreads);
        float f[U * V];
#pragma unroll
        for (int k = 0; k < U; ++k) Elem<T>::unpack(u[k], f + k * V);
        acc.add<U * V>(f, scale);
    }
    for (; v < v1; v += kThreads) {
        float f[V];
        Elem<T>::unpack(ld_stream(p + v), f);
        acc.add<V>(f, scale);
    }
    if (rank == 0) {  // what lies outside the vectors: fewer than 2 V elements
        if (t < head) acc.add_one(Elem<T>::to_f(xr[t]), scale);
        if (tail + t < r.vocab) acc.add_one(Elem<T>::to_f(xr[tail + t]), scale);
    }
    acc.merge_warp(16);
    if (kThreads > 32 && lane == 0) {
        ec[warp] = acc.c;
        es[warp] = acc.s;
    }
    if (size > 1) cluster_wait_started();
    row_sync<kThreads>();
    if (kThreads > 32 && warp == 0) {
        acc = LogSum{};
        if (lane < kThreads / 32) acc.merge(ec[lane], es[lane]);
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
    // log sum exp(x / T) = base + rest, apart where the sum of both would lose what the rest says.
    float base = 0.f, rest = (acc.c + log2f(acc.s)) * 0.69314718055994531f;
    if (fabsf(acc.c) >= kFar && acc.c != -NB200_INF) {
        const float2 far = far_row(xr, r.vocab, r.inv_t, lane);
        base = far.x;
        rest = far.y;
    }
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
        if (q != 0.f) l += q * ((teach[j] - z) - ((stud[j] - base) - rest));
    }
    mass = warp_sum(mass);
    l = warp_sum(l);
    if (lane == 0) {
        loss[row] = l;
        stats[3 * row] = base + rest;
        stats[3 * row + 1] = z;
        stats[3 * row + 2] = mass;
    }
}

// CTAs per row: enough for four on every SM, no more than leaves each at least two rounds of loads. Every
// further CTA of a row pays the merge again: bf16 [512, 262144] 54.0, 52.3, 53.5 us with 1, 2, 4;
// [1024, 50001] 24.9, 29.1, 45.3 us; [160, 131072] 20.5, 15.6, 14.7 us.
template <typename T>
int cluster_for(int64_t rows, int64_t vocab) {
    const int64_t round = (int64_t)kWide * Elem<T>::V;
    int c = 1;
    while (c < kMaxCluster && rows * c < 4 * sm_count() && vocab >= 2 * c * round) c *= 2;
    return c;
}

// ------------------------------------------------------------------ backward
// One CTA, or a warp, per row and chunk of columns: write the softmax part of the chunk, then the chunk's kept
// columns once more with their probabilities taken off.
constexpr int kChunk = 16384;   // columns, at most
constexpr int kChunkLeast = 2048;

template <typename T, int kThreads>
__global__ void __launch_bounds__(kWide)
    distill_bwd_kernel(const float* grad, int64_t grad_stride, const T* x, int64_t rows, int64_t stride, Row r,
                       const float* stats, unsigned chunks, int64_t chunk, T* dx) {
    constexpr int V = Elem<T>::V, U = 4, kRows = kWide / kThreads;
    __shared__ __align__(16) int at_[kRows][kMaxTop];  // the entry's column in the chunk, -1 outside it
    __shared__ float p_[kRows][kMaxTop];
    const int sub = kRows > 1 ? threadIdx.y : 0;  // which of the CTA's rows
    int* at = at_[sub];
    float* p = p_[sub];
    const unsigned item = blockIdx.x * kRows + sub;
    const int64_t row = item / chunks, c0 = item % chunks * chunk;
    if (kRows > 1 && row >= rows) return;
    const int n = (int)min(chunk, r.vocab - c0), t = threadIdx.x;
    const float lse = stats[3 * row], z = stats[3 * row + 1], mass = stats[3 * row + 2];
    const float w = grad[row * grad_stride] * r.inv_t, wm = w * mass;
    const T* xr = x + row * stride + c0;
    T* dr = dx + row * r.vocab + c0;
    bool mine = false;
    for (int j = t; j < (r.top + 3 & ~3); j += kThreads) {
        int64_t c = j < r.top ? r.at(row, j) : -1;
        const float logit = c >= 0 ? r.logit(row, j) : -NB200_INF;
        if (logit == -NB200_INF) c = -1;
        mine = mine || c >= 0;
        at[j] = c >= c0 && c < c0 + n ? (int)(c - c0) : -1;
        p[j] = c >= 0 ? expf(logit - z) : 0.f;
    }
    bool any;
    if constexpr (kThreads == 32) any = __any_sync(0xffffffffu, mine);
    else any = __syncthreads_or(mine);
    row_sync<kThreads>();
    // w mass q, the difference taken before the change of base so that large logits keep their digits, and from a
    // rounded x / T as the forward pass's: an exact one less a lse of -1e30 is anything, up to 2^75. A row without kept
    // entries is 0 whatever its logits hold.
    auto soft = [&](float f) { return any ? wm * ex2_ftz((__fmul_rn(f, r.inv_t) - lse) * kL2e) : 0.f; };
    const int head = (int)min(lead(dr), (int64_t)n);
    const bool together = lead(xr) == lead(dr);  // both sides meet the same 16-byte boundaries
    const int nv = together ? (n - head) / V : 0;
    const uint4* src = reinterpret_cast<const uint4*>(xr + head);
    uint4* dst = reinterpret_cast<uint4*>(dr + head);
    for (int v = t; v < nv; v += U * kThreads) {
        uint4 u[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (v + k * kThreads < nv) u[k] = ld_stream(src + v + k * kThreads);
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (v + k * kThreads >= nv) break;
            float f[V];
            Elem<T>::unpack(u[k], f);
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = soft(f[e]);
            __stcs(dst + v + k * kThreads, Elem<T>::pack(f));
        }
    }
    if (t < head) dr[t] = Elem<T>::from_f(soft(Elem<T>::to_f(xr[t])));
    for (int c = head + nv * V + t; c < n; c += kThreads) dr[c] = Elem<T>::from_f(soft(Elem<T>::to_f(xr[c])));
    row_sync<kThreads>();
    // By the first entry that names a column: entries of one column add in order.
    for (int j = t; j < r.top; j += kThreads) {
        const int c = at[j];
        if (c < 0) continue;
        float sum = 0.f;
        bool first = true;
        for (int i = 0; i < r.top; i += 4) {
            const int4 o = *reinterpret_cast<const int4*>(at + i);
            if (o.x != c && o.y != c && o.z != c && o.w != c) continue;
            const int a[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (a[e] == c) {
                    first = first && i + e >= j;
                    sum += p[i + e];
                }
        }
        if (first) dr[c] = Elem<T>::from_f(soft(Elem<T>::to_f(xr[c])) - w * sum);
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
    if (a.rows * ((a.vocab + kChunkLeast - 1) / kChunkLeast) > 0x7fffffffLL || a.rows > 0x7fffffffLL / kMaxCluster) {
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
        const bool narrow = narrow_rows(a, kNarrowFwd, sizeof(T));
        const auto kernel = narrow ? distill_fwd_kernel<T, 32> : distill_fwd_kernel<T, kWide>;
        const int size = narrow ? 1 : cluster_for<T>(a.rows, a.vocab);
        if (size > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)(narrow ? (a.rows + kWarpRows - 1) / kWarpRows : a.rows * size));
        cfg.blockDim = narrow ? dim3(32, kWarpRows) : dim3(kWide);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = size;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, kernel, x, a.rows, a.stride_x, r, teacher_lse, loss, stats);
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
        // Equal chunks of whole 128-byte lines, four CTAs on every SM where rows are few and wide enough.
        const int64_t want = (4 * (int64_t)sm_count() + a.rows - 1) / a.rows, least = (a.vocab + kChunk - 1) / kChunk;
        const int64_t cut = std::max(least, std::min(want, a.vocab / kChunkLeast));
        const int64_t chunk = ((a.vocab + cut - 1) / cut + 63) / 64 * 64, chunks = (a.vocab + chunk - 1) / chunk;
        const bool narrow = narrow_rows(a, kNarrowBwd, sizeof(T));
        const auto kernel = narrow ? distill_bwd_kernel<T, 32> : distill_bwd_kernel<T, kWide>;
        const int64_t items = a.rows * chunks;
        kernel<<<(unsigned)(narrow ? (items + kWarpRows - 1) / kWarpRows : items),
                 narrow ? dim3(32, kWarpRows) : dim3(kWide), 0, st>>>(grad, stride_grad, static_cast<const T*>(a.x),
                                                                     a.rows, a.stride_x, r, stats, (unsigned)chunks,
                                                                     chunk, d);
    };
    if (a.dtype == NB200_F32) go(static_cast<float*>(dx));
    else if (a.dtype == NB200_BF16) go(static_cast<__nv_bfloat16*>(dx));
    else go(static_cast<__half*>(dx));
    count_launch();
    return finish_launch("nb200_distill_loss_bwd");
}

}  // namespace nb200
