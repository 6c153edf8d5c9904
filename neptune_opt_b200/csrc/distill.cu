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
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace nb200 {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 256;  // entries a row may keep: one per thread

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

// Merge of two (maximum, sum of exp(x - maximum)) states; -inf maxima carry a zero sum.
__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
    const float mm = fmaxf(m, m2);
    const float a = m == mm ? s : s * expf(m - mm);
    const float b = m2 == mm ? s2 : s2 * expf(m2 - mm);
    m = mm;
    s = a + b;
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_fwd_kernel(const T* x, int64_t stride, Row r, const float* teacher_lse, float* loss, float* stats) {
    __shared__ float buf[64], sm[32], ss[32];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const T* xr = x + row * stride;
    float m = -NB200_INF, s = 0.f;
    for (int64_t c = t; c < r.vocab; c += kThreads) merge(m, s, Elem<T>::to_f(xr[c]) * r.inv_t, 1.f);
    for (int o = 16; o > 0; o >>= 1)
        merge(m, s, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o));
    if (lane == 0) {
        sm[warp] = m;
        ss[warp] = s;
    }
    __syncthreads();
    m = sm[0];
    s = ss[0];
    for (int w = 1; w < kThreads / 32; ++w) merge(m, s, sm[w], ss[w]);
    const float lse = m + logf(s);
    // The kept entries, one per thread.
    Group<true> g{buf, 0};
    const int64_t at = t < r.top ? r.at(row, t) : -1;
    const float tl = at >= 0 ? r.logit(row, t) : -NB200_INF;
    float z;
    if (teacher_lse) {
        z = teacher_lse[row];
    } else {
        const float top = g.reduce(tl, RED_MAX), shift = top == -NB200_INF ? 0.f : top;
        z = shift + logf(g.reduce(expf(tl - shift), RED_SUM));
    }
    const float p = at >= 0 ? expf(tl - z) : 0.f;
    const float mass = g.reduce(p, RED_SUM);
    const float d = at >= 0 && p != 0.f ? p * ((tl - z) - (Elem<T>::to_f(xr[at]) * r.inv_t - lse)) : 0.f;
    const float l = g.reduce(d, RED_SUM);
    if (t == 0) {
        loss[row] = l;
        stats[3 * row] = lse;
        stats[3 * row + 1] = z;
        stats[3 * row + 2] = mass;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_bwd_kernel(const float* grad, int64_t grad_stride, const T* x, int64_t stride, Row r, const float* stats,
                       T* dx) {
    __shared__ int64_t at[kMaxTop];
    __shared__ float p[kMaxTop];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x;
    const float lse = stats[3 * row], z = stats[3 * row + 1], mass = stats[3 * row + 2];
    const float w = grad[row * grad_stride] * r.inv_t;
    const T* xr = x + row * stride;
    T* dr = dx + row * r.vocab;
    at[t] = t < r.top ? r.at(row, t) : -1;
    p[t] = at[t] >= 0 ? expf(r.logit(row, t) - z) : 0.f;
    const bool any = __syncthreads_or(at[t] >= 0);
    for (int64_t c = t; c < r.vocab; c += kThreads)
        dr[c] = Elem<T>::from_f(any ? w * (mass * expf(Elem<T>::to_f(xr[c]) * r.inv_t - lse)) : 0.f);
    __syncthreads();
    // The kept columns again, by the first entry that names each: entries of one column add in order.
    if (at[t] >= 0) {
        float sum = 0.f;
        bool first = true;
        for (int j = 0; j < r.top; ++j) {
            if (at[j] != at[t]) continue;
            first = first && j >= t;
            sum += p[j];
        }
        if (first) dr[at[t]] = Elem<T>::from_f(w * (mass * expf(Elem<T>::to_f(xr[at[t]]) * r.inv_t - lse) - sum));
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
    if (a.rows > 0x7fffffffLL) {
        set_error("%s: %lld rows exceed the kernel's index range", what, (long long)a.rows);
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
        distill_fwd_kernel<<<(unsigned)a.rows, kThreads, 0, st>>>(x, a.stride_x, r, teacher_lse, loss, stats);
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
        distill_bwd_kernel<T><<<(unsigned)a.rows, kThreads, 0, st>>>(grad, stride_grad, static_cast<const T*>(a.x),
                                                                     a.stride_x, r, stats, d);
    };
    if (a.dtype == NB200_F32) go(static_cast<float*>(dx));
    else if (a.dtype == NB200_BF16) go(static_cast<__nv_bfloat16*>(dx));
    else go(static_cast<__half*>(dx));
    count_launch();
    return finish_launch("nb200_distill_loss_bwd");
}

}  // namespace nb200
