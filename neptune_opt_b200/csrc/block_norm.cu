// RMSNorm after a block, its gate and residual scale, the residual sum and the RMSNorm before the
// next block, forward and backward.
//
//   z = w1 * x r1,  r1 = rsqrt(mean x^2 + eps)       (x itself without a post weight)
//   y = residual + scale * a(gate) * z               (a: identity, tanh or sigmoid; 1 without a gate)
//   h = w2 * y r2,  r2 = rsqrt(mean y^2 + eps)       (absent without a pre weight)
//
// Backward, from dy and dh with xhat = x r1, yhat = y r2, t = dh w2:
//   dY = dy + r2 (t - yhat mean(t yhat))             = gradient of residual
//   dz = scale a dY,  u = dz w1,  dx = r1 (u - xhat mean(u xhat))
//   dw2 = sum dh yhat,  dw1 = sum dz xhat,  dgate = scale a' z dY summed over the rows that share it
//
// y is formed in fp32 from x and residual in both directions; only what is returned is rounded.
// `group` consecutive rows share one gate row. A CTA of the backward kernel owns a chunk of rows: whole
// gate groups, whose gate gradients it writes itself, or a part of one group. Weight gradients (and the
// gate's, when a group spans chunks) leave as one fp32 row per chunk, summed in chunk order by a
// second kernel, so results do not depend on scheduling.
#include <type_traits>

#include "common.cuh"
#include "launch.h"

namespace nb200 {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kWarpRows = 8;  // rows a CTA of the warp-per-row form holds

struct Norm {
    int64_t rows, width, sx, sr, sg, sdy, sdh, group;
    float scale, eps, inv_n;
    int act;
};

// a(g) and its derivative.
__device__ __forceinline__ float gate_value(float g, int kind, float& slope) {
    if (kind == NB200_GATE_TANH) {
        const float a = tanhf(g);
        slope = 1.f - a * a;
        return a;
    }
    if (kind == NB200_GATE_SIGMOID) {
        const float a = 1.f / (1.f + expf(-g));
        slope = a * (1.f - a);
        return a;
    }
    slope = 1.f;
    return g;
}

// A row is held by a warp (CTA false, kWarpRows of them in a CTA) or a whole CTA, E = NV * V elements a
// thread; t is the thread's place in its row, item the row (forward) or chunk (backward) it works on.
template <bool CTA>
struct Place {
    int t, G;
    int64_t item, items;
    __device__ __forceinline__ Place() {
        t = threadIdx.x;
        G = blockDim.x;
        item = CTA ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
        items = CTA ? (int64_t)gridDim.x : (int64_t)gridDim.x * blockDim.y;
    }
};

template <typename T, int NV, bool VEC, bool CTA, int kThreads>
__global__ void __launch_bounds__(kThreads) norm_fwd_kernel(const T* x, const T* res, const T* gate, const T* w1, const T* w2, Norm n, T* y,
                                T* h, float* rstd) {
    using CH = Chunk<T, NV, VEC>;
    constexpr int V = CH::V, E = CH::E;
    __shared__ float buf[64];
    const Place<CTA> at;
    Group<CTA> grp{buf, 0};
    CH c1, c2;
    if (w1) c1.load(w1, 1, 0, n.width, at.t, at.G, false);
    if (w2) c2.load(w2, 1, 0, n.width, at.t, at.G, false);
    for (int64_t row = at.item; row < n.rows; row += at.items) {
        CH cx, cr, cg;
        cx.load(x + row * n.sx, 1, 0, n.width, at.t, at.G, true);
        cr.load(res + row * n.sr, 1, 0, n.width, at.t, at.G, true);
        if (gate) cg.load(gate + row / n.group * n.sg, 1, 0, n.width, at.t, at.G, false);
        float s = 0.f, r1 = 1.f, r2 = 1.f;
        if (w1) {
#pragma unroll
            for (int i = 0; i < E; ++i) s = fmaf(cx.get(i), cx.get(i), s);
            r1 = rsqrtf(grp.reduce(s, RED_SUM) * n.inv_n + n.eps);
        }
        float v[E];
        s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            float z = cx.get(i), slope;
            if (w1) z *= r1 * c1.get(i);
            v[i] = fmaf(n.scale * (gate ? gate_value(cg.get(i), n.act, slope) : 1.f), z, cr.get(i));
            s = fmaf(v[i], v[i], s);
        }
        if (w2) r2 = rsqrtf(grp.reduce(s, RED_SUM) * n.inv_n + n.eps);
#pragma unroll
        for (int k = 0; k < NV; ++k) store_vec<T, NV, VEC>(y + row * n.width, v + k * V, k, 0, n.width, at.t, at.G, VEC);
        if (w2) {
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] *= r2 * c2.get(i);
#pragma unroll
            for (int k = 0; k < NV; ++k)
                store_vec<T, NV, VEC>(h + row * n.width, v + k * V, k, 0, n.width, at.t, at.G, VEC);
        }
        if (at.t == 0) {
            rstd[2 * row] = r1;
            rstd[2 * row + 1] = r2;
        }
    }
}

// How the backward pass cuts the rows: `per_group` chunks of each gate group, or (per_group 1) chunks
// of whole groups.
struct Chunks {
    int64_t rows, per_group, count;
    __device__ __forceinline__ void range(int64_t i, const Norm& n, int64_t& r0, int64_t& r1) const {
        const int64_t base = i / per_group * (per_group > 1 ? n.group : rows);
        const int64_t end = per_group > 1 ? base + n.group : n.rows;
        r0 = base + i % per_group * rows;
        r1 = r0 + rows < end ? r0 + rows : end;
    }
};

Chunks make_chunks(const Norm& n, int64_t target) {
    const int64_t want = (n.rows + target - 1) / target;  // rows per chunk
    Chunks c;
    if (n.group > want) {
        c.rows = want;
        c.per_group = (n.group + want - 1) / want;
        c.count = n.rows / n.group * c.per_group;
    } else {
        c.per_group = 1;
        c.rows = (want + n.group - 1) / n.group * n.group;
        c.count = (n.rows + c.rows - 1) / c.rows;
    }
    return c;
}

// One fp32 row of a chunk's column sums.
template <typename T, int NV, bool VEC>
__device__ __forceinline__ void store_part(float* part, const float* acc, int64_t width, int t, int G) {
    using CH = Chunk<T, NV, VEC>;
#pragma unroll
    for (int i = 0; i < CH::E; ++i) {
        const int64_t c = CH::col_of(0, t, G, i);
        if (c < width) part[c] = acc[i];
    }
}

template <typename T, int NV, bool VEC, bool CTA, int kThreads>
__global__ void __launch_bounds__(kThreads) norm_bwd_kernel(const T* dy, const T* dh, const T* x, const T* res, const T* gate, const T* w1,
                                const T* w2, const float* rstd, Norm n, Chunks ch, T* dx, T* dres, T* dgate,
                                float* part1, float* part2, float* partg) {
    using CH = Chunk<T, NV, VEC>;
    constexpr int V = CH::V, E = CH::E;
    __shared__ float buf[64];
    const Place<CTA> at;
    Group<CTA> grp{buf, 0};
    if (at.item >= ch.count) return;
    int64_t row, end;
    ch.range(at.item, n, row, end);
    CH c1, c2;
    if (w1) c1.load(w1, 1, 0, n.width, at.t, at.G, false);
    if (w2) c2.load(w2, 1, 0, n.width, at.t, at.G, false);
    float a1[E], a2[E], ag[E];
#pragma unroll
    for (int i = 0; i < E; ++i) a1[i] = a2[i] = ag[i] = 0.f;
    for (; row < end; ++row) {
        CH cx, cr, cg, cdy, cdh;
        cx.load(x + row * n.sx, 1, 0, n.width, at.t, at.G, true);
        cr.load(res + row * n.sr, 1, 0, n.width, at.t, at.G, true);
        if (gate) cg.load(gate + row / n.group * n.sg, 1, 0, n.width, at.t, at.G, false);
        if (dy) cdy.load(dy + row * n.sdy, 1, 0, n.width, at.t, at.G, true);
        if (dh) cdh.load(dh + row * n.sdh, 1, 0, n.width, at.t, at.G, true);
        const float r1 = w1 ? rstd[2 * row] : 1.f, r2 = w2 ? rstd[2 * row + 1] : 1.f;
        float xhat[E], a[E], yhat[E], d[E];
        float s = 0.f, slope;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            xhat[i] = cx.get(i) * r1;
            a[i] = n.scale * (gate ? gate_value(cg.get(i), n.act, slope) : 1.f);
            yhat[i] = fmaf(a[i], w1 ? xhat[i] * c1.get(i) : xhat[i], cr.get(i)) * r2;
            d[i] = dh && w2 ? cdh.get(i) * c2.get(i) : 0.f;
            s = fmaf(d[i], yhat[i], s);
        }
        const float m2 = w2 ? grp.reduce(s, RED_SUM) * n.inv_n : 0.f;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            d[i] = fmaf(r2, d[i] - yhat[i] * m2, dy ? cdy.get(i) : 0.f);
            if (dh) a2[i] = fmaf(cdh.get(i), yhat[i], a2[i]);
            const float dz = a[i] * d[i];
            a1[i] = fmaf(dz, xhat[i], a1[i]);
            if (w1) s = fmaf(dz * c1.get(i), xhat[i], s);
        }
        if (gate) {
            const bool whole = !partg && (row + 1) % n.group == 0;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                gate_value(cg.get(i), n.act, slope);
                ag[i] = fmaf(n.scale * slope * (w1 ? xhat[i] * c1.get(i) : xhat[i]), d[i], ag[i]);
            }
            if (whole) {
                T* out = dgate + row / n.group * n.width;
#pragma unroll
                for (int k = 0; k < NV; ++k)
                    store_vec<T, NV, VEC>(out, ag + k * V, k, 0, n.width, at.t, at.G, VEC);
#pragma unroll
                for (int i = 0; i < E; ++i) ag[i] = 0.f;
            }
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
            store_vec<T, NV, VEC>(dres + row * n.width, d + k * V, k, 0, n.width, at.t, at.G, VEC);
        const float m1 = w1 ? grp.reduce(s, RED_SUM) * n.inv_n : 0.f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float u = a[i] * d[i];
            d[i] = w1 ? r1 * (u * c1.get(i) - xhat[i] * m1) : u;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
            store_vec<T, NV, VEC>(dx + row * n.width, d + k * V, k, 0, n.width, at.t, at.G, VEC);
    }
    if (part1) store_part<T, NV, VEC>(part1 + at.item * n.width, a1, n.width, at.t, at.G);
    if (part2) store_part<T, NV, VEC>(part2 + at.item * n.width, a2, n.width, at.t, at.G);
    if (partg) store_part<T, NV, VEC>(partg + at.item * n.width, ag, n.width, at.t, at.G);
}

// out[g, c] = sum over the chunks of group g, in order, of part[chunk, c].
template <typename T>
__global__ void __launch_bounds__(256) norm_sum_kernel(const float* part, int64_t chunks, int64_t width, T* out) {
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= width) return;
    const float* p = part + (int64_t)blockIdx.y * chunks * width + c;
    float s = 0.f;
    for (int64_t i = 0; i < chunks; ++i) s += p[i * width];
    out[(int64_t)blockIdx.y * width + c] = Elem<T>::from_f(s);
}

// Threads of a row and elements of a thread: a warp holds up to 512 elements, a CTA of at most 512
// threads up to 4096 (8 a thread) or 8192 (16), a CTA of 1024 the rest.
struct Shape {
    bool cta, vec, wide, huge;
    int threads;
};

Shape make_shape(int64_t width, int esize, bool aligned) {
    Shape s;
    s.vec = aligned && width * esize % 16 == 0;
    s.cta = width > 512;
    s.wide = s.cta ? width > 4096 : width > 256;
    s.huge = width > 8192;
    const int e = s.wide ? 16 : 8;
    s.threads = s.cta ? (int)((width + 32 * e - 1) / (32 * e)) * 32 : 32;
    return s;
}

// f(CTA, E, VEC, most threads) with the shape's compile-time values.
template <typename F>
void dispatch(const Shape& s, F&& f) {
    auto vec = [&](auto cta, auto e, auto most) {
        if (s.vec) f(cta, e, std::true_type{}, most);
        else f(cta, e, std::false_type{}, most);
    };
    using E8 = std::integral_constant<int, 8>;
    using E16 = std::integral_constant<int, 16>;
    if (!s.cta && !s.wide) vec(std::false_type{}, E8{}, std::integral_constant<int, 32 * kWarpRows>{});
    else if (!s.cta) vec(std::false_type{}, E16{}, std::integral_constant<int, 32 * kWarpRows>{});
    else if (!s.wide) vec(std::true_type{}, E8{}, std::integral_constant<int, 512>{});
    else if (!s.huge) vec(std::true_type{}, E16{}, std::integral_constant<int, 512>{});
    else vec(std::true_type{}, E16{}, std::integral_constant<int, 1024>{});
}

bool rows_aligned(const void* p, int64_t stride, int esize) { return !p || (aligned16(p) && stride * esize % 16 == 0); }

int check_width(const char* what, int64_t width) {
    if (width <= kMaxWidth) return NB200_OK;
    set_error("%s: width %lld exceeds the kernel's %d", what, (long long)width, kMaxWidth);
    return NB200_ERR_CAPACITY;
}

Norm make_norm(const nb200_norm_args& a) {
    Norm n;
    n.rows = a.rows;
    n.width = a.width;
    n.sx = a.stride_x;
    n.sr = a.stride_residual;
    n.sg = a.stride_gate;
    n.sdy = a.stride_grad_y;
    n.sdh = a.stride_grad_h;
    n.group = a.gate ? a.rows_per_gate : 1;
    n.scale = (float)a.scale;
    n.eps = (float)a.eps;
    n.inv_n = 1.f / (float)a.width;
    n.act = a.gate_act;
    return n;
}

template <typename T>
int norm_fwd(const nb200_norm_args& a, T* y, T* h, float* rstd, cudaStream_t st) {
    const Norm n = make_norm(a);
    constexpr int es = sizeof(T);
    const bool al = rows_aligned(a.x, n.sx, es) && rows_aligned(a.residual, n.sr, es) &&
                    rows_aligned(a.gate, n.sg, es) && rows_aligned(a.post_weight, 0, es) &&
                    rows_aligned(a.pre_weight, 0, es) && aligned16(y) && (!h || aligned16(h));
    const Shape s = make_shape(n.width, es, al);
    const int per = s.cta ? 1 : kWarpRows;
    dispatch(s, [&](auto cta, auto e, auto vec, auto most) {
        auto kernel = norm_fwd_kernel<T, decltype(e)::value / Elem<T>::V, decltype(vec)::value, decltype(cta)::value,
                                      decltype(most)::value>;
        const int grid = persistent_grid(kernel, s.threads * per, 0, (n.rows + per - 1) / per, 0);
        kernel<<<grid, dim3(s.threads, per), 0, st>>>(
            static_cast<const T*>(a.x), static_cast<const T*>(a.residual), static_cast<const T*>(a.gate),
            static_cast<const T*>(a.post_weight), static_cast<const T*>(a.pre_weight), n, y, h, rstd);
    });
    count_launch();
    return finish_launch("nb200_gated_norm");
}

constexpr int64_t kChunkTarget = 592;

template <typename T>
int norm_bwd(const nb200_norm_args& a, const float* rstd, const T* dy, const T* dh, T* dx, T* dres, T* dgate, T* dw1,
             T* dw2, float* work, cudaStream_t st) {
    const Norm n = make_norm(a);
    constexpr int es = sizeof(T);
    const bool al = rows_aligned(a.x, n.sx, es) && rows_aligned(a.residual, n.sr, es) &&
                    rows_aligned(a.gate, n.sg, es) && rows_aligned(a.post_weight, 0, es) &&
                    rows_aligned(a.pre_weight, 0, es) && rows_aligned(dy, n.sdy, es) && rows_aligned(dh, n.sdh, es) &&
                    aligned16(dx) && aligned16(dres) && (!dgate || aligned16(dgate));
    const Shape s = make_shape(n.width, es, al);
    const int per = s.cta ? 1 : kWarpRows;
    const Chunks ch = make_chunks(n, kChunkTarget);
    const int64_t size = ch.count * n.width;
    float* p1 = dw1 ? work : nullptr;
    float* p2 = dw2 ? work + size : nullptr;
    float* pg = dgate && ch.per_group > 1 ? work + 2 * size : nullptr;
    dispatch(s, [&](auto cta, auto e, auto vec, auto most) {
        auto kernel = norm_bwd_kernel<T, decltype(e)::value / Elem<T>::V, decltype(vec)::value, decltype(cta)::value,
                                      decltype(most)::value>;
        kernel<<<(unsigned)((ch.count + per - 1) / per), dim3(s.threads, per), 0, st>>>(
            dy, dh, static_cast<const T*>(a.x), static_cast<const T*>(a.residual), static_cast<const T*>(a.gate),
            static_cast<const T*>(a.post_weight), static_cast<const T*>(a.pre_weight), rstd, n, ch, dx, dres, dgate,
            p1, p2, pg);
    });
    count_launch();
    auto sum = [&](const float* part, int64_t groups, int64_t chunks, T* out) {
        norm_sum_kernel<T><<<dim3((unsigned)((n.width + 255) / 256), (unsigned)groups), 256, 0, st>>>(part, chunks,
                                                                                                      n.width, out);
        count_launch();
    };
    if (p1) sum(p1, 1, ch.count, dw1);
    if (p2) sum(p2, 1, ch.count, dw2);
    if (pg) sum(pg, ch.count / ch.per_group, ch.per_group, dgate);
    return finish_launch("nb200_gated_norm_bwd");
}

}  // namespace

int launch_norm_fwd(const nb200_norm_args& a, int dtype, void* y, void* h, float* rstd, cudaStream_t st) {
    const int rc = check_width("nb200_gated_norm", a.width);
    if (rc) return rc;
    if (dtype == NB200_F32) return norm_fwd(a, static_cast<float*>(y), static_cast<float*>(h), rstd, st);
    if (dtype == NB200_BF16)
        return norm_fwd(a, static_cast<__nv_bfloat16*>(y), static_cast<__nv_bfloat16*>(h), rstd, st);
    return norm_fwd(a, static_cast<__half*>(y), static_cast<__half*>(h), rstd, st);
}

int64_t norm_bwd_work_bytes(const nb200_norm_args& a) {
    const Norm n = make_norm(a);
    return 3 * make_chunks(n, kChunkTarget).count * n.width * (int64_t)sizeof(float);
}

int launch_norm_bwd(const nb200_norm_args& a, int dtype, const float* rstd, const void* dy, const void* dh, void* dx,
                    void* dres, void* dgate, void* dw1, void* dw2, float* work, cudaStream_t st) {
    const int rc = check_width("nb200_gated_norm_bwd", a.width);
    if (rc) return rc;
    auto go = [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return norm_bwd<T>(a, rstd, static_cast<const T*>(dy), static_cast<const T*>(dh), static_cast<T*>(dx),
                           static_cast<T*>(dres), static_cast<T*>(dgate), static_cast<T*>(dw1), static_cast<T*>(dw2),
                           work, st);
    };
    if (dtype == NB200_F32) return go((float*)nullptr);
    if (dtype == NB200_BF16) return go((__nv_bfloat16*)nullptr);
    return go((__half*)nullptr);
}

}  // namespace nb200
