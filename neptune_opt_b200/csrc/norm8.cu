// Residual sum, RMSNorm and an 8-bit output with scales, in one pass over the rows:
//
//   y = x + residual (residual optional)       h = weight * y * rsqrt(mean(y^2) + eps)
//   scale = max(max |h| / most, 2^-126)        q = round(h / scale)
//
// per row, or per group of `group` consecutive columns; most = 448 (e4m3), 57344 (e5m2) or 127 (int8).
//
// rsqrt is one positive factor of the whole row, so max |h| = rsqrt * max |weight * y|: the sum of squares
// and the maxima are taken in the same sweep over registers and one reduction serves both. Every value is
// read once and kept in registers as fp32 until it is quantised.
//
// A row belongs to one warp (up to 1024 columns) or to one CTA. The bound is HBM traffic: two reads and
// one write of the row's type and one byte.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace nb200 {
namespace {

struct Norm8 {
    const void *x, *residual, *weight;
    void *q, *y;
    float* scale;
    int64_t rows, stride_x, stride_residual;
    int width, group;  // group = columns that share a scale
    int kind;
    float eps, per_most;  // 1 / the type's largest value
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Two quotients to two bytes, the first in the low one; round to nearest even, saturating. NaN stays NaN
// in the float types and becomes 0 in int8. (The same branch for the whole grid.)
__device__ __forceinline__ uint32_t to8x2(float a, float b, int kind) {
    if (kind == NB200_E4M3) return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    if (kind == NB200_E5M2) return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E5M2);
    const int i = max(-127, min(127, __float2int_rn(a))), j = max(-127, min(127, __float2int_rn(b)));
    return (uint32_t)(i & 0xff) | ((uint32_t)(j & 0xff) << 8);
}

// TPR threads per row (a warp, or the CTA), NV vectors of V columns each. Vector k of thread t holds the V
// columns from (t + k TPR) V on. Without VEC (a row off the 16-byte boundary, or a width that is no multiple
// of V) columns are loaded one by one, and with a scale per row they are dealt out singly, so that a warp's
// accesses stay side by side.
template <typename T, bool GROUPED, bool VEC, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm8_kernel(const Norm8 a) {
    constexpr int V = Elem<T>::V;
    constexpr int kWarps = TPR / 32;
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;  // rows of a CTA at a time
    __shared__ float red[2][kWarps > 1 ? 2 * kWarps : 1];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto column = [&](int k, int j) { return VEC || GROUPED ? (t + k * TPR) * V + j : t + (k * V + j) * TPR; };
    // The weight stays in registers over the rows.
    uint4 wv[VEC ? NV : 1];
    const T* weight = static_cast<const T*>(a.weight);
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            wv[k] = column(k, 0) < a.width ? ld_keep(weight + column(k, 0)) : make_uint4(0u, 0u, 0u, 0u);
    }
    // A row's loads go out together, and with whole vectors the next row's as soon as this one's are unpacked: they are in
    // flight while the row waits for its sums.
    const int64_t first = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR, stride = (int64_t)gridDim.x * kRows;
    uint4 xv[VEC ? NV : 1], rv[VEC ? NV : 1];
    auto load = [&](int64_t row) {
        const T* x = static_cast<const T*>(a.x) + row * a.stride_x;
        const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.stride_residual : nullptr;
#pragma unroll
        for (int k = 0; k < (VEC ? NV : 0); ++k) {
            const bool in = column(k, 0) < a.width;
            xv[k] = in ? ld_stream(x + column(k, 0)) : make_uint4(0u, 0u, 0u, 0u);
            rv[k] = in && r ? ld_stream(r + column(k, 0)) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    if (VEC && first < a.rows) load(first);
    int phase = 0;
    for (int64_t row = first; row < a.rows; row += stride, phase ^= 1) {
        T* yo = a.y ? static_cast<T*>(a.y) + row * a.width : nullptr;
        float y[NV * V], top[GROUPED ? NV : 1];
        float sum = 0.f;
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float f[V];
                Elem<T>::unpack(xv[k], y + k * V);
                Elem<T>::unpack(rv[k], f);
#pragma unroll
                for (int j = 0; j < V; ++j) y[k * V + j] += f[j];
            }
            if (row + stride < a.rows) load(row + stride);
        } else {
            const T* x = static_cast<const T*>(a.x) + row * a.stride_x;
            const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.stride_residual : nullptr;
            T xs[NV * V], rs[NV * V];
#pragma unroll
            for (int i = 0; i < NV * V; ++i) {
                const int c = min(column(i / V, i % V), a.width - 1);
                xs[i] = x[c];
                rs[i] = r ? r[c] : Elem<T>::from_f(0.f);
            }
#pragma unroll
            for (int i = 0; i < NV * V; ++i)
                y[i] = column(i / V, i % V) < a.width ? Elem<T>::to_f(xs[i]) + Elem<T>::to_f(rs[i]) : 0.f;
        }
        if (yo) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if constexpr (VEC) {
                    if (column(k, 0) < a.width) *reinterpret_cast<uint4*>(yo + column(k, 0)) = Elem<T>::pack(y + k * V);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (column(k, j) < a.width) yo[column(k, j)] = Elem<T>::from_f(y[k * V + j]);
                }
            }
        }
        // Sum of squares, then y becomes weight * y.
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float w[V];
            if constexpr (VEC) {
                Elem<T>::unpack(wv[k], w);
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j) w[j] = column(k, j) < a.width ? Elem<T>::to_f(weight[column(k, j)]) : 0.f;
            }
            float g = 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float& v = y[k * V + j];
                sum = fmaf(v, v, sum);
                v *= w[j];
                g = max_nan(g, fabsf(v));
            }
            if constexpr (GROUPED) top[k] = g;
            else most = max_nan(most, g);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if constexpr (!GROUPED) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        if constexpr (kWarps > 1) {
            if (lane == 0) {
                red[phase][warp] = sum;
                red[phase][kWarps + warp] = most;
            }
            __syncthreads();
            sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                sum += red[phase][w];
                if constexpr (!GROUPED) most = max_nan(most, red[phase][kWarps + w]);
            }
        }
        const float rstd = rsqrtf(sum / (float)a.width + a.eps);
        // A group's columns lie in neighbouring lanes.
        if constexpr (GROUPED) {
            for (int o = a.group / V / 2; o > 0; o >>= 1)
#pragma unroll
                for (int k = 0; k < NV; ++k) top[k] = max_nan(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
        }
        uint8_t* q = static_cast<uint8_t*>(a.q) + row * a.width;
        float s = 0.f, inv = 0.f;
        auto take = [&](float m) {
            s = m * rstd * a.per_most;
            s = s < 1.17549435e-38f ? 1.17549435e-38f : s;  // NaN stays
            inv = 1.f / s;
        };
        if constexpr (!GROUPED) {
            take(most);
            if (t == 0) a.scale[row] = s;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if constexpr (GROUPED) {
                take(top[k]);
                const int c = column(k, 0);
                if (c < a.width && c % a.group == 0) a.scale[row * (a.width / a.group) + c / a.group] = s;
            }
            uint32_t w[V / 2];
#pragma unroll
            for (int j = 0; j < V; j += 2)
                w[j / 2] = to8x2(y[k * V + j] * rstd * inv, y[k * V + j + 1] * rstd * inv, a.kind);
            if constexpr (VEC) {
                if (column(k, 0) < a.width) {
                    if constexpr (V == 8)
                        *reinterpret_cast<uint2*>(q + column(k, 0)) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
                    else
                        *reinterpret_cast<uint32_t*>(q + column(k, 0)) = w[0] | w[1] << 16;
                }
            } else {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (column(k, j) < a.width) q[column(k, j)] = (uint8_t)(w[j / 2] >> (8 * (j & 1)));
            }
        }
    }
}

template <typename T, bool GROUPED, bool VEC, int TPR, int NV>
int launch(const Norm8& a, cudaStream_t st) {
    constexpr int kThreads = TPR < 128 ? 128 : TPR;
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;
    auto kernel = norm8_kernel<T, GROUPED, VEC, TPR, NV>;
    // As many CTAs as the GPU holds; asked once (the same for every device this library is built for).
    static const int per_sm = [kernel] {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, 0) != cudaSuccess || n < 1) n = 1;
        return n;
    }();
    const int64_t grid = std::min((a.rows + kRows - 1) / kRows, (int64_t)per_sm * sm_count());
    launch_pdl(kernel, (unsigned)grid, kThreads, 0, st, a);
    count_launch();
    return finish_launch("nb200_norm8");
}

template <typename T, bool GROUPED, bool VEC>
int by_width(const Norm8& a, cudaStream_t st) {
    constexpr int V = Elem<T>::V;
    const int n = a.width;
    if (n <= 256) return launch<T, GROUPED, VEC, 32, 8 / V>(a, st);
    if (n <= 1024) return launch<T, GROUPED, VEC, 32, 32 / V>(a, st);
    if (n <= 2048) return launch<T, GROUPED, VEC, 128, 16 / V>(a, st);
    if (n <= 4096) return launch<T, GROUPED, VEC, 128, 32 / V>(a, st);
    if (n <= 8192) return launch<T, GROUPED, VEC, 256, 32 / V>(a, st);
    return launch<T, GROUPED, VEC, 512, 32 / V>(a, st);
}

template <typename T>
int by_layout(const Norm8& a, cudaStream_t st) {
    constexpr int V = Elem<T>::V;
    const bool vec = a.width % V == 0 && a.stride_x % V == 0 && (!a.residual || a.stride_residual % V == 0) &&
                     aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) && aligned16(a.y) &&
                     (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0;
    if (a.group != a.width) return vec ? by_width<T, true, true>(a, st) : by_width<T, true, false>(a, st);
    return vec ? by_width<T, false, true>(a, st) : by_width<T, false, false>(a, st);
}

}  // namespace

int launch_norm8(const nb200_norm8_args& n, void* q, float* scale, void* y, cudaStream_t st) {
    const float most = n.kind == NB200_E4M3 ? 448.f : n.kind == NB200_E5M2 ? 57344.f : 127.f;
    const Norm8 a = {n.x, n.residual, n.weight, q, n.residual ? y : nullptr, scale, n.rows, n.stride_x, n.stride_residual,
                     (int)n.width, (int)(n.group ? n.group : n.width), n.kind, (float)n.eps, 1.f / most};
    if (n.dtype == NB200_F32) return by_layout<float>(a, st);
    if (n.dtype == NB200_BF16) return by_layout<__nv_bfloat16>(a, st);
    return by_layout<__half>(a, st);
}

}  // namespace nb200
