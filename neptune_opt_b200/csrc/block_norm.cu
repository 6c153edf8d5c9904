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
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "fastmath.cuh"
#include "launch.h"
#include "stream.cuh"

namespace nb200 {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kWarpRows = 8;  // rows a CTA of the warp-per-row form holds

struct Norm {
    int64_t rows, width, sx, sr, sg, sdy, sdh;
    uint32_t group;  // rows that share a gate row
    float scale, eps, inv_n;
    int act;
};

// a(g), and its derivative in terms of a. The sigmoid's division is good to 2 ulp (and gives 0 where expf overflows):
// a gate row for each row, bf16 [16384, 4096] forward 148 us, rounded exactly 161 us; fp32 [16384, 1000] backward
// 103 us and 124 us. The fp32 forward kernel has no registers to spare and takes the exact one (EXACT), with which it
// spills less inside its loop ([16384, 2048] 91 us, else 95 us).
template <bool EXACT>
__device__ __forceinline__ float gate_value(float g, int kind) {
    if (kind == NB200_GATE_TANH) return tanhf(g);
    if (kind == NB200_GATE_SIGMOID) return EXACT ? 1.f / (1.f + expf(-g)) : __fdividef(1.f, 1.f + expf(-g));
    return g;
}
__device__ __forceinline__ float gate_slope(float a, int kind) {
    if (kind == NB200_GATE_TANH) return 1.f - a * a;
    if (kind == NB200_GATE_SIGMOID) return a * (1.f - a);
    return 1.f;
}

// NV 16-byte vectors' worth of a row's elements, zero past the row.
template <typename T, int NV>
struct Vecs {
    static constexpr int V = Elem<T>::V, P = NV * V / 2;
    uint4 raw[NV];
    __device__ __forceinline__ float get(int i) const { return Elem<T>::lane(raw[i / V], i % V); }
    __device__ __forceinline__ uint64_t pair(int i) const { return f2(get(2 * i), get(2 * i + 1)); }
};

// A row is held by a warp (CTA false, kWarpRows of them in a CTA) or a whole CTA, E = NV * V elements a
// thread, computed as packed fp32 pairs. A unit (warp or CTA) works through consecutive rows, so that the
// weights stay in registers and a gate row is read and put through its activation once per group.
//
// Element i of thread t is column (t + (i / V) G) V + i % V, less `lead` columns where rows do not start on a
// 16-byte boundary. Three forms:
//  ALIGNED  every row of every tensor starts on a 16-byte boundary and is whole vectors.
//  LINED    widths off the vector size, tensors laid out alike (contiguous ones are): all tensors' rows are off the
//           boundary by the same amount, which repeats every `step` rows (8 at most). A unit takes rows of one
//           residue, so that its vectors are aligned in every row, its columns stay the same, and only the
//           first and the last vector of a row are partial.
//  ANY      anything else (slices): 16-bit rows move in vectors that each thread shifts (the two aligned
//           vectors it straddles, never one without a byte of the row; a store passes its last elements
//           to the next lane, which writes the aligned vector they begin, and the few elements at the ends of a
//           warp's span go one by one), fp32 rows go element by element, column t + i G.
// bf16 [16384, 3001], backward: 195 us lined up, 427 us by shifted vectors, 795 us element by element.
enum Form { ALIGNED, LINED, ANY };
template <typename T, Form FORM>
constexpr bool kScalar = FORM == ANY && sizeof(T) == 4;

// KEEP: stored rows stay in L2 for whoever reads them next, ahead of what streams past (bf16 [16384, 4096] forward
// 97.4 us, 99.6 stored as they stream; the backward, which writes less than it reads, is as fast either way and
// leaves L2 to its partial sums).
template <typename T, int NV, Form FORM, bool CTA, bool KEEP>
struct Rows {
    using CH = Vecs<T, NV>;
    static constexpr int V = CH::V, P = CH::P;  // P pairs a thread
    int t, G;
    int64_t unit;
    int width, lead = 0;
    float* buf;  // 2 x 4 x 32 entries of shared memory when CTA
    int phase = 0;

    __device__ __forceinline__ Rows(int64_t w, float* b) : width((int)w), buf(b) {
        t = threadIdx.x;
        G = blockDim.x;
        unit = CTA ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    }
    // Columns ahead of the first whole vector: `row` is any row this unit works on.
    __device__ __forceinline__ void line_up(const T* row) {
        if (FORM == LINED) lead = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
    }
    __device__ __forceinline__ int col(int k) const { return (t + k * G) * V - (FORM == LINED ? lead : 0); }
    __device__ __forceinline__ int col_of(int i) const { return kScalar<T, FORM> ? t + i * G : col(i / V) + i % V; }
    __device__ __forceinline__ bool holds(int c) const { return c < width && (FORM != LINED || c >= 0); }
    __device__ __forceinline__ static uint4 fetch(const void* p, bool stream) {
        return stream ? ld_stream(p) : ld_keep(p);
    }
    // A row of one of the tensors the form speaks of; `finish` before use. (Clearing the partial vectors here would
    // make their warps wait for a prefetched row as soon as it is sent for.)
    __device__ __forceinline__ void load(CH& c, const T* row, bool stream) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int at = col(k);
            if constexpr (FORM == ALIGNED) {
                if (at < width) c.raw[k] = fetch(row + at, stream);
                else c.raw[k] = make_uint4(0u, 0u, 0u, 0u);
            } else if constexpr (FORM == LINED) {
                if (at < width && at + V > 0) c.raw[k] = fetch(row + at, stream);
                else c.raw[k] = make_uint4(0u, 0u, 0u, 0u);
            } else if constexpr (kScalar<T, FORM>) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int i = col_of(4 * k + j);
                    w[j] = i < width ? __float_as_uint(row[i]) : 0u;
                }
                c.raw[k] = make_uint4(w[0], w[1], w[2], w[3]);
            } else if (at >= width) {
                c.raw[k] = make_uint4(0u, 0u, 0u, 0u);
            } else {
                const uintptr_t a = reinterpret_cast<uintptr_t>(row + at);
                const uint32_t off = (uint32_t)a & 15u;  // the same for every thread of the row
                const char* p = reinterpret_cast<const char*>(a - off);
                uint4 lo = fetch(p, stream), hi = make_uint4(0u, 0u, 0u, 0u);
                if (off && p + 16 < reinterpret_cast<const char*>(row + width)) hi = fetch(p + 16, stream);
                c.raw[k] = shift_down(lo, hi, off);
                if (at + V > width) keep_range(c.raw[k], 0, width - at);
            }
        }
    }
    __device__ __forceinline__ void finish(CH& c) const {
        if constexpr (FORM == LINED) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int at = col(k);
                if (at < 0 || at + V > width) keep_range(c.raw[k], -at, width - at);
            }
        }
    }
    // A weight or a shared gate row, which need not be laid out like the rows.
    __device__ __forceinline__ void load_shared(CH& c, const T* row) const {
        if constexpr (FORM != LINED) {
            load(c, row, false);
        } else {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                float f[V];
#pragma unroll
                for (int j = 0; j < V; ++j) f[j] = holds(col(k) + j) ? Elem<T>::to_f(row[col(k) + j]) : 0.f;
                c.raw[k] = Elem<T>::pack(f);
            }
        }
    }
    // 16 bytes from byte `off` of lo:hi.
    __device__ __forceinline__ static uint4 shift_down(const uint4& lo, const uint4& hi, uint32_t off) {
        uint32_t w[7] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z};
        const uint32_t last = hi.w;
        if (off & 8u) {
            w[0] = w[2], w[1] = w[3], w[2] = w[4], w[3] = w[5], w[4] = w[6], w[5] = last;
        }
        if (off & 4u) {
            w[0] = w[1], w[1] = w[2], w[2] = w[3], w[3] = w[4], w[4] = w[5];
        }
        const uint32_t bits = (off & 2u) * 8u;
        return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                          __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
    }
    // Zeroes every element outside [from, to).
    __device__ __forceinline__ static void keep_range(uint4& u, int from, int to) {
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j >= from && j < to) continue;
            if constexpr (V == 4) w[j] = 0u;
            else w[j / 2] &= j & 1 ? 0xffffu : 0xffff0000u;
        }
        u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ static void put(T* row, int c, const uint4& u, int j) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (V == 4) reinterpret_cast<uint32_t*>(row)[c] = w[j];
        else reinterpret_cast<uint16_t*>(row)[c] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
    __device__ __forceinline__ static void put_vec(void* p, const uint4& u) {
        if (KEEP) *reinterpret_cast<uint4*>(p) = u;
        else st_stream(p, u);
    }
    __device__ __forceinline__ void store(T* row, const uint64_t* v) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float f[V];
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                f[2 * j] = f2lo(v[k * V / 2 + j]);
                f[2 * j + 1] = f2hi(v[k * V / 2 + j]);
            }
            const int at = col(k);
            if constexpr (FORM == ALIGNED) {
                if (at < width) put_vec(row + at, Elem<T>::pack(f));
            } else if constexpr (kScalar<T, FORM>) {
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (col_of(k * V + j) < width) row[col_of(k * V + j)] = f[j];
            } else if constexpr (FORM == LINED) {
                const uint4 u = Elem<T>::pack(f);
                if (at >= 0 && at + V <= width) {
                    put_vec(row + at, u);
                } else {
#pragma unroll
                    for (int j = 0; j < V; ++j)
                        if (holds(at + j)) put(row, at + j, u, j);
                }
            } else {
                store_shifted(row, at, Elem<T>::pack(f));
            }
        }
    }
    // Whole warps come here. `own` elements at the start of a vector share their aligned 16 bytes with the last
    // `pass` elements of the lane below.
    __device__ __forceinline__ void store_shifted(T* row, int at, const uint4& u) const {
        const uintptr_t a = reinterpret_cast<uintptr_t>(row) + (uintptr_t)at * sizeof(T);
        const uint32_t off = (uint32_t)a & 15u;
        const int pass = off / (int)sizeof(T), own = V - pass, lane = t & 31;
        const int valid = max(0, min(V, width - at)), above = max(0, min(V, width - at - V));
        uint4 below;
        below.x = __shfl_up_sync(0xffffffffu, u.x, 1);
        below.y = __shfl_up_sync(0xffffffffu, u.y, 1);
        below.z = __shfl_up_sync(0xffffffffu, u.z, 1);
        below.w = __shfl_up_sync(0xffffffffu, u.w, 1);
        const bool whole = (lane > 0 || pass == 0) && valid >= own;
        if (whole) put_vec(reinterpret_cast<void*>(a - off), pass ? shift_down(below, u, 16u - off) : u);
        // Elements no whole vector takes: the head of a warp's first lane, the tail of its last, the row's end.
        uint32_t single = whole ? 0u : (1u << own) - 1u;
        if (pass && (lane == 31 || above < own)) single |= ((1u << V) - 1u) & ~((1u << own) - 1u);
        single &= (1u << valid) - 1u;
        if (__any_sync(0xffffffffu, single)) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (single >> j & 1u) put(row, at + j, u, j);
        }
    }
    // The sum of v over the row's threads, in every thread: warp shuffles, then the warps' sums (one
    // barrier; the two buffers alternate).
    __device__ __forceinline__ float sum(float v) {
        v = warp_sum(v);
        if constexpr (CTA) {
            float* slot = buf + (phase ^= 1) * 4 * 32;
            if ((t & 31) == 0) slot[t >> 5] = v;
            __syncthreads();
            v = warp_sum((t & 31) < (G >> 5) ? slot[t & 31] : 0.f);
        }
        return v;
    }
    // Three sums at once. Each of the first two shuffle rounds halves the number of values a lane carries (it
    // keeps its half of them and adds the partner's), so six shuffles do what fifteen would.
    __device__ __forceinline__ void sum3(float& a, float& b, float& c) {
        const bool hi = t & 16, odd = t & 8;
        float k0 = hi ? c : a, k1 = hi ? 0.f : b;  // kept: (a, b) below lane 16, (c, -) above
        k0 += __shfl_xor_sync(0xffffffffu, hi ? a : c, 16);
        k1 += __shfl_xor_sync(0xffffffffu, hi ? b : 0.f, 16);
        float v = odd ? k1 : k0;  // lanes 0-7 a, 8-15 b, 16-23 c
        v += __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 8);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if constexpr (CTA) {
            float* slot = buf + (phase ^= 1) * 4 * 32;
            const int which = (t & 31) >> 3, warps = G >> 5;
            if ((t & 7) == 0) slot[which * 32 + (t >> 5)] = v;
            __syncthreads();
            v = 0.f;
            for (int w = t & 7; w < warps; w += 8) v += slot[which * 32 + w];
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        }
        a = __shfl_sync(0xffffffffu, v, 0);
        b = __shfl_sync(0xffffffffu, v, 8);
        c = __shfl_sync(0xffffffffu, v, 16);
    }
};

// Threads of a row and elements of a thread: a warp of 8 holds up to 256 elements, a CTA of at most 512 threads up
// to 4096 (8 a thread) or 8192 (16), a CTA of 1024 the rest.
struct Shape {
    bool cta;
    Form form;
    int e, threads;
};

Shape make_shape(int64_t width, Form form) {
    Shape s;
    s.form = form;
    const int64_t span = form == LINED ? width + 7 : width;  // columns ahead of the first vector
    s.cta = span > 256;
    s.e = span <= 4096 ? 8 : 16;
    s.threads = s.cta ? (int)((span + 32 * s.e - 1) / (32 * s.e)) * 32 : 32;
    return s;
}

// How the rows are cut into units' shares. Rows are planned in groups of `group` (all rows, unless whole gate groups
// have to stay together), per_group units each; `step` units take turns at consecutive rows.
struct Chunks {
    int64_t group, per_group, rows, step, count;
    __device__ __forceinline__ void range(int64_t i, const Norm& n, uint32_t& r0, uint32_t& r1) const {
        const int64_t g = i / per_group, u = i - g * per_group, base = g * group;
        const int64_t from = base + u / step * (rows * step), to = from + rows * step;
        r0 = (uint32_t)(from + u % step);
        r1 = (uint32_t)min(min(to, base + group), n.rows);
    }
};

Chunks make_chunks(const Norm& n, int64_t group, int64_t target, int64_t step) {
    Chunks c;
    c.step = step;
    const int64_t groups = n.rows / group;
    if (groups < target || step > 1) {  // parts of a group: at most `target` in all, or `step` for each group
        const int64_t turns = std::min((group + step - 1) / step, std::max<int64_t>(1, target / groups / step));
        c.group = group;
        c.rows = (group + turns * step - 1) / (turns * step);
        c.per_group = (group + c.rows * step - 1) / (c.rows * step) * step;
        c.count = groups * c.per_group;
    } else {  // whole groups
        c.group = c.rows = (groups + target - 1) / target * group;
        c.per_group = 1;
        c.count = (n.rows + c.rows - 1) / c.rows;
    }
    return c;
}

// A gate row: laid out like the rows when every row has its own; `finish` before use.
template <typename R, typename T>
__device__ __forceinline__ void load_gate(const R& r, typename R::CH& c, const T* gate, const Norm& n, uint32_t index) {
    if (n.group == 1) r.load(c, gate + index * n.sg, true);
    else r.load_shared(c, gate + index * n.sg);
}

template <typename T, int NV, Form FORM, bool CTA, int kThreads>
__global__ void __launch_bounds__(kThreads, (CTA || FORM == ALIGNED) && NV * Elem<T>::V == 8 ? 1024 / kThreads : 1)
    norm_fwd_kernel(const T* x, const T* res, const T* gate, const T* w1, const T* w2, Norm n, Chunks ch, T* y, T* h,
                    float* rstd) {
    using R = Rows<T, NV, FORM, CTA, true>;
    using CH = typename R::CH;
    constexpr int P = R::P;
    __shared__ float buf[CTA ? 256 : 1];
    R r(n.width, buf);
    if (r.unit >= ch.count) return;
    uint32_t row, end;
    ch.range(r.unit, n, row, end);
    if (row >= end) return;
    r.line_up(x + row * n.sx);
    CH c1, c2, cx, cr, cg;
    if (w1) r.load_shared(c1, w1);
    if (w2) r.load_shared(c2, w2);
    r.load(cx, x + row * n.sx, true);
    r.load(cr, res + row * n.sr, true);
    uint32_t index = 0;
    if (gate) {
        index = row / n.group;
        load_gate(r, cg, gate, n, index);
    }
    bool fresh = true;
    uint64_t b[P];  // scale * a(gate) * post weight
    for (; row < end; row += ch.step) {
        if (fresh) {
            if (gate) r.finish(cg);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint64_t a = gate ? f2(n.scale * gate_value<sizeof(T) == 4>(cg.get(2 * i), n.act),
                                             n.scale * gate_value<sizeof(T) == 4>(cg.get(2 * i + 1), n.act))
                                        : f2(n.scale, n.scale);
                b[i] = w1 ? mul2(a, c1.pair(i)) : a;
            }
        }
        r.finish(cx);
        r.finish(cr);
        // The next row is on its way while this one is reduced.
        CH nx, nr;
        fresh = false;
        const uint32_t next = row + ch.step;
        if (next < end) {
            r.load(nx, x + next * n.sx, true);
            r.load(nr, res + next * n.sr, true);
            if (gate && next / n.group != index) {
                index = next / n.group;
                load_gate(r, cg, gate, n, index);
                fresh = true;
            }
        }
        float r1 = 1.f, r2 = 1.f;
        uint64_t acc = 0;
        if (w1) {
#pragma unroll
            for (int i = 0; i < P; ++i) acc = fma2(cx.pair(i), cx.pair(i), acc);
            float s = f2lo(acc) + f2hi(acc);
            s = r.sum(s);
            r1 = rsqrtf(s * n.inv_n + n.eps);
        }
        uint64_t v[P];
        acc = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            v[i] = fma2(b[i], mul2(cx.pair(i), f2(r1, r1)), cr.pair(i));
            acc = fma2(v[i], v[i], acc);
        }
        r.store(y + (int64_t)row * n.width, v);
        if (w2) {
            float s = f2lo(acc) + f2hi(acc);
            s = r.sum(s);
            r2 = rsqrtf(s * n.inv_n + n.eps);
#pragma unroll
            for (int i = 0; i < P; ++i) v[i] = mul2(v[i], mul2(c2.pair(i), f2(r2, r2)));
            r.store(h + (int64_t)row * n.width, v);
        }
        if (r.t == 0) *reinterpret_cast<float2*>(rstd + 2 * (int64_t)row) = make_float2(r1, r2);
        cx = nx;
        cr = nr;
    }
}

// One fp32 row of a chunk's column sums.
template <typename R>
__device__ __forceinline__ void store_part(float* part, const uint64_t* acc, const R& r) {
#pragma unroll
    for (int i = 0; i < 2 * R::P; ++i) {
        const int c = r.col_of(i);
        if (r.holds(c)) part[c] = i & 1 ? f2hi(acc[i / 2]) : f2lo(acc[i / 2]);
    }
}

// Both row statistics come from one round of sums: with c = scale a w1 xhat,
//   n m2 = sum t yhat,   n m1 = sum c dY = sum c (dy + r2 t) - r2 m2 sum c yhat.
// Within a gate group the gate and post-weight gradients share one column sum, G = sum xhat dY:
// dgate = scale a' w1 G and dw1 += scale a G.
//
// A row's operands (its own gate row among them) come through a ring of shared-memory stages filled by bulk copies
// (RING: the CTA form of ALIGNED rows, where the stages fit), rows ahead of their use and without registers or issue
// slots; without a ring the next row waits in registers, where a thread's share of it is 8 elements (AHEAD). bf16
// [16384, 4096]: 161 us with the ring, 179 us in registers. Two stages beat no prefetch (bf16 [8192, 8192] 228 us and
// 243) but not registers (fp32 [4096, 4096] 103 us and 76), and LINED rows lost by a ring ([16384, 3001] 202 us
// against 195). One CTA of 512 threads per SM either way: two, at 64 registers a thread, spilled (250 us).
constexpr int kMaxRing = 4;
constexpr int kSmShared = 233472;  // shared memory of an SM, 228 KB
constexpr int kCtaShared = 1024 + 1280;  // what is reserved for each CTA, and the kernel's own 1.1 KB

template <typename T, int NV, Form FORM, bool CTA, bool RING, int kThreads>
__global__ void __launch_bounds__(kThreads)
    norm_bwd_kernel(const T* dy, const T* dh, const T* x, const T* res, const T* gate, const T* w1, const T* w2,
                    const float* rstd, Norm n, Chunks ch, int stages, T* dx, T* dres, T* dgate, float* part1,
                    float* part2, float* partg) {
    static_assert(!RING || (CTA && FORM == ALIGNED), "the ring holds whole aligned rows");
    using R = Rows<T, NV, FORM, CTA, false>;
    using CH = typename R::CH;
    constexpr int P = R::P;
    constexpr bool AHEAD = !RING && P == 4;
    __shared__ float buf[CTA ? 256 : 1];
    __shared__ uint64_t full[RING ? kMaxRing : 1];
    extern __shared__ __align__(16) uint8_t dyn[];
    R r(n.width, buf);
    // What a thread keeps across rows but touches little lives in shared memory, in slots of its own:
    // a(gate), b = scale a(gate) w1 and the post weight's sums (touched once per gate group).
    const int slots = (CTA ? 1 : kWarpRows) * r.G * P;
    uint64_t* bs = reinterpret_cast<uint64_t*>(dyn) + (CTA ? 0 : threadIdx.y * r.G * P) + r.t;
    uint64_t* as = bs + slots;
    uint64_t* a1 = as + slots;
    pdl_trigger();
    if (r.unit >= ch.count) return;
    uint32_t row, end;
    ch.range(r.unit, n, row, end);
    r.line_up(x + row * n.sx);
    const bool own = gate && n.group == 1;  // a gate row for each row: it comes along with the row
    // Stage s holds the vectors of x, residual, dy, dh and the gate that cover one row.
    uint8_t* ring = reinterpret_cast<uint8_t*>(bs - r.t + 3 * slots);
    const uint32_t bytes = r.width * (uint32_t)sizeof(T);
    const uint32_t pitch = (own ? 5 : 4) * bytes;
    auto fill = [&](int s, uint32_t i) {  // one thread
        uint8_t* to = ring + s * pitch;
        mbar_expect_tx(&full[s], (2 + (dy ? 1 : 0) + (dh ? 1 : 0) + (own ? 1 : 0)) * bytes);
        bulk_load(to, x + i * n.sx, bytes, &full[s]);
        bulk_load(to + bytes, res + i * n.sr, bytes, &full[s]);
        if (dy) bulk_load(to + 2 * bytes, dy + i * n.sdy, bytes, &full[s]);
        if (dh) bulk_load(to + 3 * bytes, dh + i * n.sdh, bytes, &full[s]);
        if (own) bulk_load(to + 4 * bytes, gate + i * n.sg, bytes, &full[s]);
    };
    int stage = 0;
    uint32_t parity = 0;
    bool primed = false;  // a row has been taken out of the ring
    // False once a wait of this thread has run out. From there on it waits no more and takes NaN for what it should
    // have read, which the row's sums carry to every thread: such rows, and the sums over rows, come out NaN. (Stopping
    // the CTA instead takes a word from all of them for every row: bf16 [16384, 4096] 173 us, 167 us this way.)
    bool arrived = true;
    if constexpr (RING) {
        if (threadIdx.x == 0) {
            for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
            fence_barrier_init();
            fence_proxy_async();
            for (int s = 0; s < stages; ++s)
                if (row + s * ch.step < end) fill(s, row + s * (uint32_t)ch.step);
        }
        __syncthreads();
    }
    CH c1, c2;
    if (w1) r.load_shared(c1, w1);
    if (w2) r.load_shared(c2, w2);
    uint64_t G[P], a2[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        G[i] = a2[i] = 0;
        a1[i * r.G] = 0;
    }
    uint32_t index = gate ? row / n.group : 0u;
    bool fresh = true;
    CH nx, nr, ndy, ndh, ng;
    float2 nrs;
    auto statistics = [&](uint32_t i) { nrs = *reinterpret_cast<const float2*>(rstd + 2 * (int64_t)i); };
    auto fetch = [&](uint32_t i) {
        statistics(i);
        r.load(nx, x + i * n.sx, true);
        r.load(nr, res + i * n.sr, true);
        if (dy) r.load(ndy, dy + i * n.sdy, true);
        if (dh) r.load(ndh, dh + i * n.sdh, true);
        if (own) r.load(ng, gate + i * n.sg, true);
    };
    if (AHEAD && row < end) fetch(row);
    if (RING && row < end) statistics(row);
    for (; row < end; row += ch.step) {
        const uint32_t next = row + ch.step, next_index = gate ? next / n.group : 0u;
        const bool last = next >= end;
        if (!AHEAD && !RING) fetch(row);
        if constexpr (RING) {
            arrived = arrived && mbar_wait(&full[stage], parity);
            auto staged = [&](CH& c, int i) {
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const uint4* p = reinterpret_cast<const uint4*>(ring + stage * pitch + i * bytes) + r.t + k * r.G;
                    c.raw[k] = r.col(k) < r.width ? *p : make_uint4(0u, 0u, 0u, 0u);
                }
            };
            staged(nx, 0);
            staged(nr, 1);
            if (dy) staged(ndy, 2);
            if (dh) staged(ndh, 3);
            if (own) staged(ng, 4);
            if (!arrived) {
#pragma unroll
                for (int k = 0; k < NV; ++k) nx.raw[k] = ndy.raw[k] = make_uint4(~0u, ~0u, ~0u, ~0u);
            }
        }
        CH cx = nx, cr = nr, cdy = ndy, cdh = ndh;
        r.finish(cx);
        r.finish(cr);
        if (dy) r.finish(cdy);
        if (dh) r.finish(cdh);
        const float2 rs = nrs;
        if (fresh) {
            CH cg = ng;
            if (gate && !own) load_gate(r, cg, gate, n, index);
            if (gate) r.finish(cg);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint64_t v = gate ? f2(gate_value<false>(cg.get(2 * i), n.act),
                                             gate_value<false>(cg.get(2 * i + 1), n.act))
                                        : f2(1.f, 1.f);
                const uint64_t a = mul2(v, f2(n.scale, n.scale));
                as[i * r.G] = v;
                bs[i * r.G] = w1 ? mul2(a, c1.pair(i)) : a;
            }
        }
        const float r1 = w1 ? rs.x : 1.f, r2 = w2 ? rs.y : 1.f;
        const uint64_t r1p = f2(r1, r1), r2p = f2(r2, r2);
        uint64_t yhat[P], e[P];  // e = dy + r2 t
        uint64_t s1 = 0, s2 = 0, s3 = 0;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint64_t c = mul2(bs[i * r.G], mul2(cx.pair(i), r1p));
            yhat[i] = mul2(add2(c, cr.pair(i)), r2p);
            const uint64_t t = dh ? mul2(cdh.pair(i), c2.pair(i)) : 0;
            e[i] = fma2(t, r2p, dy ? cdy.pair(i) : 0);
            s1 = fma2(t, yhat[i], s1);
            s2 = fma2(c, e[i], s2);
            s3 = fma2(c, yhat[i], s3);
            if (dh) a2[i] = fma2(cdh.pair(i), yhat[i], a2[i]);
        }
        // Issued here, the loads cover the sums' latency.
        if (AHEAD && !last) fetch(next);
        if (RING && !last) statistics(next);
        if (gate && !own && next_index != index && !last && (r.t & 7) == 0)
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                if (r.holds(r.col(k)))
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(gate + next_index * n.sg + r.col(k)));
            }
        float t1 = f2lo(s1) + f2hi(s1), t2 = f2lo(s2) + f2hi(s2), t3 = f2lo(s3) + f2hi(s3);
        r.sum3(t1, t2, t3);
        if constexpr (RING) {
            // Past the barrier in there, every thread is done with the previous row: its stage takes the row that is
            // `stages` behind it.
            const uint32_t ahead = row + (uint32_t)ch.step * (stages - 1);
            if (threadIdx.x == 0 && arrived && primed && ahead < end) fill(stage ? stage - 1 : stages - 1, ahead);
            primed = true;
            if (++stage == stages) {
                stage = 0;
                parity ^= 1u;
            }
        }
        const float k2 = r2 * t1 * n.inv_n, m1 = (t2 - k2 * t3) * n.inv_n;  // k2 = r2 m2
        const uint64_t k2p = f2(-k2, -k2), k1p = f2(w1 ? -m1 : 0.f, w1 ? -m1 : 0.f);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint64_t xhat = mul2(cx.pair(i), r1p);
            if (w2) e[i] = fma2(yhat[i], k2p, e[i]);  // dY
            G[i] = fma2(xhat, e[i], G[i]);
            yhat[i] = mul2(fma2(xhat, k1p, mul2(bs[i * r.G], e[i])), r1p);  // dx
        }
        r.store(dres + (int64_t)row * n.width, e);
        r.store(dx + (int64_t)row * n.width, yhat);
        // The end of a gate group, or of the chunk.
        fresh = gate && next_index != index;
        if (fresh || last) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint64_t a = as[i * r.G], g1 = mul2(G[i], f2(n.scale, n.scale));
                a1[i * r.G] = fma2(a, g1, a1[i * r.G]);
                G[i] = mul2(g1, f2(gate_slope(f2lo(a), n.act), gate_slope(f2hi(a), n.act)));
                if (w1) G[i] = mul2(G[i], c1.pair(i));
            }
            if (dgate && !partg) r.store(dgate + index * n.width, G);
            index = next_index;
            if (last) break;
#pragma unroll
            for (int i = 0; i < P; ++i) G[i] = 0;
        }
    }
    if (RING && !arrived && threadIdx.x == 0)  // copies may still be on their way: wait for them, again with a limit
        for (int s = 0; s < stages; ++s)
            for (uint32_t ph = 0; ph < 2; ++ph) mbar_wait(&full[s], ph);
    if (part2) store_part(part2 + r.unit * n.width, a2, r);
    if (part1) {
#pragma unroll
        for (int i = 0; i < P; ++i) a2[i] = a1[i * r.G];
        store_part(part1 + r.unit * n.width, a2, r);
    }
    if (partg) store_part(partg + r.unit * n.width, G, r);
}

// Column sums over chunks, in an order that depends on their number alone: out row blockIdx.y is dpost,
// dpre, then the gate rows. kSumRows threads of a column each add every kSumRows-th chunk, then meet.
constexpr int kSumCols = 32, kSumRows = 16;
template <typename T>
struct Sums {
    const float* part[3];  // of dpost, dpre, dgate; null: not wanted
    T* out[3];
    int64_t chunks, per_group, width;
};
template <typename T>
__global__ void __launch_bounds__(kSumCols* kSumRows) norm_sum_kernel(Sums<T> a) {
    __shared__ float buf[kSumRows][kSumCols];
    pdl_wait();
    const int64_t c = (int64_t)blockIdx.x * kSumCols + threadIdx.x;
    const int which = min((int)blockIdx.y, 2);
    const int64_t group = (int64_t)blockIdx.y - which;
    if (!a.part[which]) return;
    const int64_t chunks = which == 2 ? a.per_group : a.chunks;
    const float* p = a.part[which] + group * chunks * a.width + c;
    float s = 0.f;
    if (c < a.width) {
#pragma unroll 4
        for (int64_t i = threadIdx.y; i < chunks; i += kSumRows) s += p[i * a.width];
    }
    buf[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.y || c >= a.width) return;
    for (int i = 1; i < kSumRows; ++i) s += buf[i][threadIdx.x];
    a.out[which][group * a.width + c] = Elem<T>::from_f(s);
}

// f(CTA, E, FORM, most threads) with the shape's compile-time values.
template <typename F>
void dispatch(const Shape& s, F&& f) {
    auto pick = [&](auto cta, auto e, auto most) {
        if (s.form == ALIGNED) f(cta, e, std::integral_constant<Form, ALIGNED>{}, most);
        else if (s.form == LINED) f(cta, e, std::integral_constant<Form, LINED>{}, most);
        else f(cta, e, std::integral_constant<Form, ANY>{}, most);
    };
    using E8 = std::integral_constant<int, 8>;
    using E16 = std::integral_constant<int, 16>;
    if (!s.cta) pick(std::false_type{}, E8{}, std::integral_constant<int, 32 * kWarpRows>{});
    else if (s.e == 8) pick(std::true_type{}, E8{}, std::integral_constant<int, 512>{});
    else if (s.threads <= 512) pick(std::true_type{}, E16{}, std::integral_constant<int, 512>{});
    else pick(std::true_type{}, E16{}, std::integral_constant<int, 1024>{});
}

// What the rows of several tensors have in common: where they start within 16 bytes.
struct Layout {
    bool aligned = true, alike = true, any = false;
    uintptr_t base = 0;
    int64_t pitch = 0;
    void add(const void* p, int64_t stride, int esize) {
        if (!p) return;
        const uintptr_t at = reinterpret_cast<uintptr_t>(p) & 15u;
        const int64_t bytes = stride * esize & 15;
        aligned = aligned && at == 0 && bytes == 0;
        if (any) alike = alike && at == base && bytes == pitch;
        any = true;
        base = at;
        pitch = bytes;
    }
    int64_t step() const {  // rows until the offset repeats
        int64_t n = 1;
        while (n * pitch & 15) n *= 2;
        return n;
    }
};

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
    n.group = a.gate ? (uint32_t)a.rows_per_gate : 1u;
    n.scale = (float)a.scale;
    n.eps = (float)a.eps;
    n.inv_n = 1.f / (float)a.width;
    n.act = a.gate_act;
    return n;
}

// The form of a call whose row tensors have layout `l`, all tensors together `all`. Lined-up rows may need one
// vector more than a CTA holds.
Form pick_form(const Norm& n, const Layout& l, const Layout& all, int esize) {
    if (all.aligned && n.width * esize % 16 == 0) return ALIGNED;
    return l.alike && make_shape(n.width, LINED).threads <= 1024 ? LINED : ANY;
}

template <typename T>
int norm_fwd(const nb200_norm_args& a, T* y, T* h, float* rstd, cudaStream_t st) {
    const Norm n = make_norm(a);
    constexpr int es = sizeof(T);
    Layout l;
    l.add(a.x, n.sx, es);
    l.add(a.residual, n.sr, es);
    l.add(y, n.width, es);
    l.add(h, n.width, es);
    if (n.group == 1) l.add(a.gate, n.sg, es);
    Layout all = l;  // the shared rows count for ALIGNED
    if (n.group > 1) all.add(a.gate, n.sg, es);
    all.add(a.post_weight, 0, es);
    all.add(a.pre_weight, 0, es);
    const Shape s = make_shape(n.width, pick_form(n, l, all, es));
    const int per = s.cta ? 1 : kWarpRows;
    dispatch(s, [&](auto cta, auto e, auto form, auto most) {
        auto kernel = norm_fwd_kernel<T, decltype(e)::value / Elem<T>::V, decltype(form)::value, decltype(cta)::value,
                                      decltype(most)::value>;
        // Units enough to fill the GPU (1024 threads of 64 registers on an SM, or 512 of 128), each with an equal share
        // of the rows.
        const int64_t ctas = (int64_t)sm_count() * std::max(1, (s.e == 8 ? 1024 : 512) / (s.threads * per));
        const int64_t target = ctas * per, multiple = s.form == LINED ? l.step() : 1;
        Chunks ch = make_chunks(n, n.rows, target, multiple);  // a run of rows for each
        // Better, all units of a gate group take turns row by row: together they sweep through neighbouring rows (bf16
        // [16384, 4096] 99.6 us, runs 101.8; [8192, 8192] 104 and 107). Not where that makes a unit's share larger, nor
        // across gate groups, whose activations it would compute anew every few rows (64 groups of 256: 150 us, runs
        // 102). The backward, with more to fetch for each row, does not gain (bf16 [16384, 4096] 170.5 us, runs 168.7).
        const int64_t group = n.group > 1 ? n.group : n.rows, all_units = target / (n.rows / group);
        const Chunks turns = make_chunks(
            n, group, target, std::max<int64_t>(1, std::min(all_units, group) / multiple) * multiple);
        if (turns.rows <= ch.rows) ch = turns;
        kernel<<<(unsigned)((ch.count + per - 1) / per), dim3(s.threads, per), 0, st>>>(
            static_cast<const T*>(a.x), static_cast<const T*>(a.residual), static_cast<const T*>(a.gate),
            static_cast<const T*>(a.post_weight), static_cast<const T*>(a.pre_weight), n, ch, y, h, rstd);
    });
    count_launch();
    return finish_launch("nb200_gated_norm");
}

// 512 threads on every SM, about what fits one at a time, and one chunk for each unit of them: more chunks mean
// more partial sums to write and add (bf16 [32768, 1024] 91 us, with twice as many 105). Gate groups of more than
// one row stay apart, so that a unit's gate gradients are of one group, or of whole ones.
int64_t bwd_target(const Shape& s) {
    return (int64_t)sm_count() * (s.cta ? std::max(1, 512 / s.threads) : 2 * kWarpRows);
}
Chunks bwd_chunks(const Norm& n, const Shape& s, int64_t step) {
    return make_chunks(n, n.group > 1 ? n.group : n.rows, bwd_target(s), step);
}
// Lined-up rows cut every gate group at least `step` ways: not where many small groups would make that far more
// units (and partial sums) than the GPU needs.
bool lined_pays(const Norm& n, int64_t step) {
    return n.group == 1 || n.rows / n.group * step <= 2 * bwd_target(make_shape(n.width, LINED));
}

template <typename T>
int norm_bwd(const nb200_norm_args& a, const float* rstd, const T* dy, const T* dh, T* dx, T* dres, T* dgate, T* dw1,
             T* dw2, float* work, cudaStream_t st) {
    const Norm n = make_norm(a);
    constexpr int es = sizeof(T);
    Layout l;
    l.add(a.x, n.sx, es);
    l.add(a.residual, n.sr, es);
    l.add(dy, n.sdy, es);
    l.add(dh, n.sdh, es);
    l.add(dx, n.width, es);
    l.add(dres, n.width, es);
    if (n.group == 1) {
        l.add(a.gate, n.sg, es);
        l.add(dgate, n.width, es);
    }
    Layout all = l;
    if (n.group > 1) {
        all.add(a.gate, n.sg, es);
        all.add(dgate, n.width, es);
    }
    all.add(a.post_weight, 0, es);
    all.add(a.pre_weight, 0, es);
    Form form = pick_form(n, l, all, es);
    if (form == LINED && !lined_pays(n, l.step())) form = ANY;
    // Whole gate groups (rows whose offset never changes) store their gate's gradient themselves, in the rows' layout.
    if (form == LINED && l.step() == 1 && n.group > 1 && dgate) {
        Layout with = l;
        with.add(dgate, n.width, es);
        if (!with.alike) form = ANY;
    }
    const Shape s = make_shape(n.width, form);
    const int per = s.cta ? 1 : kWarpRows;
    const Chunks ch = bwd_chunks(n, s, s.form == LINED ? l.step() : 1);
    const int64_t size = ch.count * n.width;
    float* p1 = dw1 ? work : nullptr;
    float* p2 = dw2 ? work + size : nullptr;
    float* pg = dgate && n.group > 1 && ch.per_group > 1 ? work + 2 * size : nullptr;
    int rc = NB200_OK;
    dispatch(s, [&](auto cta, auto e, auto f, auto most) {
        constexpr int kNV = decltype(e)::value / Elem<T>::V, kMost = decltype(most)::value;
        constexpr Form kForm = decltype(f)::value;
        constexpr bool kCta = decltype(cta)::value;
        auto kernel = norm_bwd_kernel<T, kNV, kForm, kCta, false, kMost>;
        int smem = 3 * per * s.threads * decltype(e)::value * (int)sizeof(float), stages = 0;
        constexpr uint32_t kSlots = 3 * kMost * decltype(e)::value * sizeof(float);  // the most of them
        static SharedLimit limits[2];  // of this instance's two kernels
        bool ring = false;
        if constexpr (kCta && kForm == ALIGNED && kMost == 512) {
            // What the CTAs that share an SM leave of its shared memory beside their accumulators.
            const int room = kSmShared / std::max(1, 512 / s.threads) - kCtaShared - smem;
            const int stage = (a.gate && n.group == 1 ? 5 : 4) * (int)n.width * es;
            stages = std::min(kMaxRing, room / stage);
            if (stages >= (s.e == 8 ? 3 : 2)) {
                kernel = norm_bwd_kernel<T, kNV, kForm, kCta, true, kMost>;
                smem += stages * stage;
                ring = true;
            }
        }
        if (smem > 40 * 1024 &&
            (rc = limits[ring].raise("nb200_gated_norm_bwd", kernel, ring ? kSmShared - kCtaShared : kSlots)))
            return;
        kernel<<<(unsigned)((ch.count + per - 1) / per), dim3(s.threads, per), smem, st>>>(
            dy, dh, static_cast<const T*>(a.x), static_cast<const T*>(a.residual), static_cast<const T*>(a.gate),
            static_cast<const T*>(a.post_weight), static_cast<const T*>(a.pre_weight), rstd, n, ch, stages, dx, dres,
            dgate,
            p1, p2, pg);
    });
    if (rc) return rc;
    count_launch();
    if (p1 || p2 || pg) {
        const Sums<T> sums = {{p1, p2, pg}, {dw1, dw2, dgate}, ch.count, ch.per_group, n.width};
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)((n.width + kSumCols - 1) / kSumCols),
                           (unsigned)(2 + (pg ? ch.count / ch.per_group : 0)));
        cfg.blockDim = dim3(kSumCols, kSumRows);
        cfg.stream = st;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        cudaLaunchKernelEx(&cfg, norm_sum_kernel<T>, sums);
        count_launch();
    }
    return finish_launch("nb200_gated_norm_bwd");
}

}  // namespace

int norm_fault_take(unsigned int* bits) {
    unsigned int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_stream_fault, sizeof(v)) != cudaSuccess ||
        cudaMemcpyToSymbol(g_stream_fault, &zero, sizeof(zero)) != cudaSuccess) {
        set_error("cannot read the gated norm's fault word: %s", cudaGetErrorString(cudaGetLastError()));
        return NB200_ERR_LAUNCH;
    }
    *bits = v;
    return NB200_OK;
}

int launch_norm_fwd(const nb200_norm_args& a, int dtype, void* y, void* h, float* rstd, cudaStream_t st) {
    const int rc = check_width("nb200_gated_norm", a.width);
    if (rc) return rc;
    if (dtype == NB200_F32) return norm_fwd(a, static_cast<float*>(y), static_cast<float*>(h), rstd, st);
    if (dtype == NB200_BF16)
        return norm_fwd(a, static_cast<__nv_bfloat16*>(y), static_cast<__nv_bfloat16*>(h), rstd, st);
    return norm_fwd(a, static_cast<__half*>(y), static_cast<__half*>(h), rstd, st);
}

int64_t norm_bwd_work_bytes(const nb200_norm_args& a) {
    // The form depends on the pointers: room for the form that cuts finest.
    const Norm n = make_norm(a);
    int64_t count = bwd_chunks(n, make_shape(n.width, ALIGNED), 1).count;
    for (int64_t step = 1; step <= 8; step *= 2)
        if (lined_pays(n, step)) count = std::max(count, bwd_chunks(n, make_shape(n.width, LINED), step).count);
    return 3 * count * n.width * (int64_t)sizeof(float);
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
