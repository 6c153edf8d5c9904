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
// A row belongs to one warp (up to 512 columns) or to one CTA. The bound is HBM traffic, two reads and one write of the
// row's type and one byte, with issue slots close behind: the arithmetic runs on packed pairs, and what depends on the
// 8-bit type or the group is decided once per vector. bf16 [16384, 4096] with a residual and groups of 128: 77 us, 6.1 TB/s,
// 20 instructions a value, which take 57% of the issue slots; without the residual 47 us, 17 and 65%. fp32 [3003, 1001] 8 us,
// 4.8 TB/s.
#include <cuda_fp8.h>

#include <algorithm>

#include "common.cuh"
#include "fastmath.cuh"
#include "launch.h"

namespace nb200 {
namespace {

struct Norm8 {
    const void *x, *residual, *weight;
    void *q, *y;
    float* scale;
    int64_t rows, stride_x, stride_residual;
    int width, group;  // group = columns that share a scale
    int group_bits;    // log2 of it, where there is more than one
    int kind;
    float eps, most, per_most;  // the type's largest value, and one over it
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The bytes of V quotients, the first in the lowest one; round to nearest even, saturating. NaN stays NaN in the float
// types and becomes 0 in int8.
template <int V, __nv_fp8_interpretation_t F>
__device__ __forceinline__ void to_fp8(const uint64_t* x, uint32_t* w) {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f2lo(x[2 * j]), f2hi(x[2 * j])), __NV_SATFINITE, F);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f2lo(x[2 * j + 1]), f2hi(x[2 * j + 1])), __NV_SATFINITE, F);
        w[j] = lo | hi << 16;
    }
}
__device__ __forceinline__ uint32_t to_i8(float x) { return (uint32_t)max(-127, min(127, __float2int_rn(x))) & 0xffu; }
template <int V>
__device__ __forceinline__ void to_bytes(const uint64_t* x, uint32_t* w, int kind) {
    if (kind == NB200_E4M3) {
        to_fp8<V, __NV_E4M3>(x, w);
    } else if (kind == NB200_E5M2) {
        to_fp8<V, __NV_E5M2>(x, w);
    } else {
#pragma unroll
        for (int j = 0; j < V / 4; ++j)
            w[j] = to_i8(f2lo(x[2 * j])) | to_i8(f2hi(x[2 * j])) << 8 | to_i8(f2lo(x[2 * j + 1])) << 16 |
                   to_i8(f2hi(x[2 * j + 1])) << 24;
    }
}
__device__ __forceinline__ float reciprocal(float x) {
    float y;
    asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));  // 1 ulp
    return y;
}
// A 16-byte vector's values in pairs.
template <typename T>
__device__ __forceinline__ void unpack2(const uint4& u, uint64_t* p) {
    float f[Elem<T>::V];
    Elem<T>::unpack(u, f);
#pragma unroll
    for (int j = 0; j < Elem<T>::V / 2; ++j) p[j] = f2(f[2 * j], f[2 * j + 1]);
}

// How a row's columns are dealt out. TPR threads (a warp, or the CTA) hold NV vectors of V columns each.
//   WHOLE    every row starts on a 16-byte boundary and is whole vectors
//   SHIFTED  rows of a width that is no multiple of V, one behind the other: vectors start on 16-byte boundaries all the
//            same, and the first and the last one of a row hold columns of its neighbours, too, which are left out of the
//            sums and not stored (nor loaded, behind the last rows). The cut depends on the row's number modulo V alone; a
//            worker takes rows of one residue, and its weights stay in registers. (bf16 [16384, 4001] 87 us, column by
//            column 203.)
//   SINGLE   any strides: columns are moved one by one, with a scale per row side by side over the threads
enum Layout { WHOLE, SHIFTED, SINGLE };

// Elements [c, c + V) of a row as a vector, 0 outside of it.
template <typename T>
__device__ __forceinline__ uint4 gather(const T* row, int c, int width) {
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < Elem<T>::V; ++j) {
        if (c + j < 0 || c + j >= width) continue;
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(row[c + j]);
        else w[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[c + j] << (16 * (j & 1));
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <typename T, bool GROUPED, Layout L, int TPR, int NV>
__global__ void __launch_bounds__(TPR < 128 ? 128 : TPR) norm8_kernel(const Norm8 a) {
    constexpr int V = Elem<T>::V;
    constexpr int kWarps = TPR / 32;
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;  // rows of a CTA at a time
    __shared__ float red[2][kWarps > 1 ? 2 * kWarps : 1];
    pdl_wait();
    pdl_trigger();
    const int t = threadIdx.x % TPR, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr bool VEC = L != SINGLE;
    const int64_t first = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR, stride = (int64_t)gridDim.x * kRows;
    // Columns that the first vector of this worker's rows has before them.
    const int lead = L == SHIFTED ? (int)(first * a.width % V) : 0;
    auto column = [&](int k, int j) { return VEC || GROUPED ? (t + k * TPR) * V + j - lead : t + (k * V + j) * TPR; };
    // Whether vector k lies in the row as a whole.
    auto whole = [&](int k) {
        return L == SHIFTED ? column(k, 0) >= 0 && column(k, 0) + V <= a.width : column(k, 0) < a.width;
    };
    auto fetch = [&](const T* row, int k, bool last) {
        if (L != SHIFTED ? whole(k) : column(k, 0) < a.width && (!last || whole(k))) return ld_stream(row + column(k, 0));
        if (L == SHIFTED && last) return gather(row, column(k, 0), a.width);
        return make_uint4(0u, 0u, 0u, 0u);
    };
    // The weight stays in registers over the rows.
    uint4 wv[VEC ? NV : 1];
    const T* weight = static_cast<const T*>(a.weight);
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if constexpr (L == SHIFTED) wv[k] = gather(weight, column(k, 0), a.width);
            else wv[k] = whole(k) ? ld_keep(weight + column(k, 0)) : make_uint4(0u, 0u, 0u, 0u);
        }
    }
    // A row's loads go out together, and with whole vectors the next row's as soon as this one's are unpacked: they are in
    // flight while the row waits for its sums.
    uint4 xv[VEC ? NV : 1], rv[VEC ? NV : 1];
    auto load = [&](int64_t row) {
        const T* x = static_cast<const T*>(a.x) + row * a.stride_x;
        const T* r = a.residual ? static_cast<const T*>(a.residual) + row * a.stride_residual : nullptr;
#pragma unroll
        for (int k = 0; k < (VEC ? NV : 0); ++k) {
            xv[k] = fetch(x, k, (a.rows - 1 - row) * a.stride_x < V);  // less than a vector behind the row
            if (r) rv[k] = fetch(r, k, (a.rows - 1 - row) * a.stride_residual < V);
        }
    };
    if (VEC && first < a.rows) load(first);
    int phase = 0;
    for (int64_t row = first; row < a.rows; row += stride, phase ^= 1) {
        T* yo = a.y ? static_cast<T*>(a.y) + row * a.width : nullptr;
        uint64_t y[NV * V / 2];  // in pairs
        float top[GROUPED ? NV : 1];
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < NV; ++k) unpack2<T>(xv[k], y + k * V / 2);
            if (a.residual) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    uint64_t f[V / 2];
                    unpack2<T>(rv[k], f);
#pragma unroll
                    for (int j = 0; j < V / 2; ++j) y[k * V / 2 + j] = add2(y[k * V / 2 + j], f[j]);
                }
            }
            if constexpr (L == SHIFTED) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    if (!whole(k)) {
#pragma unroll
                        for (int j = 0; j < V; j += 2) {
                            uint64_t& p = y[(k * V + j) / 2];
                            const int c = column(k, j);
                            p = f2(c >= 0 && c < a.width ? f2lo(p) : 0.f, c + 1 >= 0 && c + 1 < a.width ? f2hi(p) : 0.f);
                        }
                    }
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
            for (int i = 0; i < NV * V; i += 2) {
                float f[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    f[e] = column((i + e) / V, (i + e) % V) < a.width ? Elem<T>::to_f(xs[i + e]) + Elem<T>::to_f(rs[i + e]) : 0.f;
                y[i / 2] = f2(f[0], f[1]);
            }
        }
        auto value = [](const uint64_t* p, int i) { return i % 2 ? f2hi(p[i / 2]) : f2lo(p[i / 2]); };
        if (yo) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float f[V];
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = value(y, k * V + j);
                if (VEC && whole(k)) {
                    *reinterpret_cast<uint4*>(yo + column(k, 0)) = Elem<T>::pack(f);
                } else if (L != WHOLE) {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (column(k, j) >= 0 && column(k, j) < a.width) yo[column(k, j)] = Elem<T>::from_f(f[j]);
                }
            }
        }
        // Sum of squares, then y becomes weight * y.
        uint64_t sums = 0;
        float most = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            uint64_t w[V / 2];
            if constexpr (VEC) {
                unpack2<T>(wv[k], w);
            } else {
#pragma unroll
                for (int j = 0; j < V; j += 2)
                    w[j / 2] = f2(column(k, j) < a.width ? Elem<T>::to_f(weight[column(k, j)]) : 0.f,
                                  column(k, j + 1) < a.width ? Elem<T>::to_f(weight[column(k, j + 1)]) : 0.f);
            }
            float g = 0.f;
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                uint64_t& v = y[k * V / 2 + j];
                sums = fma2(v, v, sums);
                v = mul2(v, w[j]);
                g = max_nan(max_nan(g, fabsf(f2lo(v))), fabsf(f2hi(v)));
            }
            if constexpr (GROUPED) top[k] = g;
            else most = max_nan(most, g);
        }
        float sum = f2lo(sums) + f2hi(sums);
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
        // A group's scale, and what takes weight * y to its quotients: most / max |weight * y|, in which rsqrt has cancelled (two
        // roundings between the values and their quotients, so that few land on another byte than the exact ones do). The
        // smallest scale, an infinite one, NaN and a maximum whose own reciprocal leaves fp32 take the long way, in two factors.
        // 1 / m is the approximate reciprocal behind one step of Newton's iteration, r + r (1 - m r).
        float s = 0.f;
        uint64_t by = 0, then = 0;
        auto take = [&](float m) {
            s = m * rstd * a.per_most;
            const bool one = m > 1e-30f && m < 1e30f && s > 1.17549435e-38f && s < NB200_INF;
            if (one) {
                const float r = reciprocal(m), f = fmaf(r, fmaf(-m, r, 1.f), r) * a.most;
                by = f2(f, f);
            } else {
                s = s < 1.17549435e-38f ? 1.17549435e-38f : s;  // NaN stays
                const float inv = reciprocal(s);
                by = f2(rstd, rstd), then = f2(inv, inv);
            }
            return one;
        };
        bool one = true;
        if constexpr (!GROUPED) {
            one = take(most);
            if (t == 0) a.scale[row] = s;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if constexpr (GROUPED) {
                one = take(top[k]);
                const int c = column(k, 0);
                if (c < a.width && (c & (a.group - 1)) == 0)
                    a.scale[row * (a.width >> a.group_bits) + (c >> a.group_bits)] = s;
            }
            uint64_t x[V / 2];
#pragma unroll
            for (int j = 0; j < V / 2; ++j) x[j] = mul2(y[k * V / 2 + j], by);
            if (!one) {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) x[j] = mul2(x[j], then);
            }
            uint32_t w[V / 4];
            to_bytes<V>(x, w, a.kind);
            if (VEC && whole(k)) {
                if constexpr (V == 8) *reinterpret_cast<uint2*>(q + column(k, 0)) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t*>(q + column(k, 0)) = w[0];
            } else if (L != WHOLE) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (column(k, j) >= 0 && column(k, j) < a.width) q[column(k, j)] = (uint8_t)(w[j / 4] >> (8 * (j & 3)));
            }
        }
    }
}

template <typename T, bool GROUPED, Layout L, int TPR, int NV>
int launch(const Norm8& a, cudaStream_t st) {
    constexpr int kThreads = TPR < 128 ? 128 : TPR;
    constexpr int kRows = TPR < 128 ? 128 / TPR : 1;
    auto kernel = norm8_kernel<T, GROUPED, L, TPR, NV>;
    // As many CTAs as the GPU holds; asked once (the same for every device this library is built for).
    static const int per_sm = [kernel] {
        int n = 0;
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, kThreads, 0) != cudaSuccess || n < 1) n = 1;
        return n;
    }();
    int64_t grid = std::min((a.rows + kRows - 1) / kRows, (int64_t)per_sm * sm_count());
    if (L == SHIFTED) grid = std::max<int64_t>(grid / 8, 1) * 8;  // rows of one residue modulo V to a worker
    launch_pdl(kernel, (unsigned)grid, kThreads, 0, st, a);
    count_launch();
    return finish_launch("nb200_norm8");
}

template <typename T, bool GROUPED, Layout L>
int by_width(const Norm8& a, cudaStream_t st) {
    constexpr int V = Elem<T>::V;
    const int n = a.width + (L == SHIFTED ? V - 1 : 0);  // columns of a row's vectors, at most
    if (n <= 256) return launch<T, GROUPED, L, 32, 8 / V>(a, st);
    if (n <= 512) return launch<T, GROUPED, L, 32, 16 / V>(a, st);
    // From here on a CTA a row: bf16 [65536, 1024] 75 us (a warp a row 80), fp32 [3003, 1001] 7.8 us (10.8); at 512 columns
    // it is the other way round (137 us, 100).
    if (n <= 1024) return launch<T, GROUPED, L, 128, 8 / V>(a, st);
    if (n <= 2048) return launch<T, GROUPED, L, 128, 16 / V>(a, st);
    if (n <= 4096) return launch<T, GROUPED, L, 128, 32 / V>(a, st);
    if (n <= 8192) return launch<T, GROUPED, L, 256, 32 / V>(a, st);
    if (n <= 16384) return launch<T, GROUPED, L, 512, 32 / V>(a, st);
    return launch<T, GROUPED, SINGLE, 512, 32 / V>(a, st);  // the last few columns before the limit, shifted
}

template <typename T>
int by_layout(const Norm8& a, cudaStream_t st) {
    constexpr int V = Elem<T>::V;
    auto alike = [&](int64_t stride) { return stride >= a.width && (stride - a.width) % V == 0; };  // cut as y's rows are
    const bool one = a.rows == 1;
    const bool base = aligned16(a.x) && aligned16(a.residual) && aligned16(a.y) && (reinterpret_cast<uintptr_t>(a.q) & 7u) == 0;
    const bool vec = base && (one || alike(a.stride_x)) && (one || !a.residual || alike(a.stride_residual));
    auto even = [&](int64_t stride) { return one || stride % V == 0; };
    const bool whole = base && a.width % V == 0 && even(a.stride_x) && (!a.residual || even(a.stride_residual)) &&
                       aligned16(a.weight);
    if (a.group != a.width) return whole ? by_width<T, true, WHOLE>(a, st) : by_width<T, true, SINGLE>(a, st);
    if (whole) return by_width<T, false, WHOLE>(a, st);
    return vec ? by_width<T, false, SHIFTED>(a, st) : by_width<T, false, SINGLE>(a, st);
}

}  // namespace

int launch_norm8(const nb200_norm8_args& n, void* q, float* scale, void* y, cudaStream_t st) {
    const float most = n.kind == NB200_E4M3 ? 448.f : n.kind == NB200_E5M2 ? 57344.f : 127.f;
    Norm8 a = {n.x, n.residual, n.weight, q, n.residual ? y : nullptr, scale, n.rows, n.stride_x, n.stride_residual,
                     (int)n.width, (int)(n.group ? n.group : n.width), 0, n.kind, (float)n.eps, most, 1.f / most};
    while (n.group && (1 << a.group_bits) < n.group) ++a.group_bits;
    if (n.dtype == NB200_F32) return by_layout<float>(a, st);
    if (n.dtype == NB200_BF16) return by_layout<__nv_bfloat16>(a, st);
    return by_layout<__half>(a, st);
}

}  // namespace nb200
