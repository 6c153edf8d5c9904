// Attention's backward pass, probabilities recomputed from the saved log-sum-exp:
//
//   P_ij = exp(scale q_i k_j - lse_i), 0 where masked      delta_i = sum_d dO_id O_id
//   dV = P^T dO     dS = P * (dO V^T - delta)     dQ = scale dS K     dK = scale dS^T Q
//
// A key/value head shared by several query heads sums over them.
#include "attn.cuh"

namespace nb200 {
namespace {

struct BwdArgs {
    nb200_attn_args n;
    nb200_attn_strides s[8];  // q, k, v, o, grad_o, dq, dk, dv
    const __nv_bfloat16 *q, *k, *v, *o, *go;
    const float* lse;
    __nv_bfloat16 *dq, *dk, *dv;
    float* delta;  // [batch, heads, seq]
};

__device__ __forceinline__ int64_t at(const nb200_attn_strides& s, int64_t b, int64_t h, int64_t i) {
    return b * s.batch + h * s.head + i * s.seq;
}

// Four consecutive elements of a row of 128: lane l holds 4 l .. 4 l + 3.
struct Four {
    float v[4];
    __device__ __forceinline__ void load(const __nv_bfloat16* row) {
        const uint2 u = *reinterpret_cast<const uint2*>(row + 4 * (threadIdx.x & 31));
        Elem<__nv_bfloat16>::unpack_word(u.x, v);
        Elem<__nv_bfloat16>::unpack_word(u.y, v + 2);
    }
    __device__ __forceinline__ void store(__nv_bfloat16* row) const {
        *reinterpret_cast<uint2*>(row + 4 * (threadIdx.x & 31)) = make_uint2(
            Elem<__nv_bfloat16>::pack_word(v[0], v[1]), Elem<__nv_bfloat16>::pack_word(v[2], v[3]));
    }
    __device__ __forceinline__ void fma(float a, const Four& o) {
        for (int i = 0; i < 4; ++i) v[i] = fmaf(a, o.v[i], v[i]);
    }
    __device__ __forceinline__ float dot(const Four& o) const {
        return warp_sum(v[0] * o.v[0] + v[1] * o.v[1] + v[2] * o.v[2] + v[3] * o.v[3]);
    }
};

constexpr int kRowsPerCta = 8;  // one warp per row

__global__ void __launch_bounds__(32 * kRowsPerCta) bwd_dq_kernel(BwdArgs a) {
    const int64_t row = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5);
    if (row >= a.n.batch * a.n.heads * a.n.seq) return;
    const int64_t i = row % a.n.seq, h = row / a.n.seq % a.n.heads, b = row / a.n.seq / a.n.heads;
    const int64_t hk = h / (a.n.heads / a.n.kv_heads);
    const int len = tokens_of(a.n.seq_lens, (int)b, (int)a.n.seq);
    Four dq = {};
    if (i < len) {
        Four q, go, o;
        q.load(a.q + at(a.s[0], b, h, i));
        o.load(a.o + at(a.s[3], b, h, i));
        go.load(a.go + at(a.s[4], b, h, i));
        const float delta = go.dot(o), lse = a.lse[row];
        if ((threadIdx.x & 31) == 0) a.delta[row] = delta;
        const int64_t end = a.n.causal ? i + 1 : len;
        for (int64_t j = 0; j < end; ++j) {
            Four k, v;
            k.load(a.k + at(a.s[1], b, hk, j));
            v.load(a.v + at(a.s[2], b, hk, j));
            const float p = lse == -NB200_INF ? 0.f : expf(a.n.scale * q.dot(k) - lse);
            dq.fma(a.n.scale * p * (go.dot(v) - delta), k);
        }
    }
    dq.store(a.dq + at(a.s[5], b, h, i));
}

__global__ void __launch_bounds__(32 * kRowsPerCta) bwd_dkv_kernel(BwdArgs a) {
    const int64_t row = (int64_t)blockIdx.x * kRowsPerCta + (threadIdx.x >> 5);
    if (row >= a.n.batch * a.n.kv_heads * a.n.seq) return;
    const int64_t j = row % a.n.seq, hk = row / a.n.seq % a.n.kv_heads, b = row / a.n.seq / a.n.kv_heads;
    const int64_t group = a.n.heads / a.n.kv_heads;
    const int len = tokens_of(a.n.seq_lens, (int)b, (int)a.n.seq);
    Four dk = {}, dv = {};
    if (j < len) {
        Four k, v;
        k.load(a.k + at(a.s[1], b, hk, j));
        v.load(a.v + at(a.s[2], b, hk, j));
        for (int64_t h = hk * group; h < (hk + 1) * group; ++h)
            for (int64_t i = a.n.causal ? j : 0; i < len; ++i) {
                Four q, go;
                q.load(a.q + at(a.s[0], b, h, i));
                go.load(a.go + at(a.s[4], b, h, i));
                const int64_t r = (b * a.n.heads + h) * a.n.seq + i;
                const float lse = a.lse[r];
                const float p = lse == -NB200_INF ? 0.f : expf(a.n.scale * q.dot(k) - lse);
                dv.fma(p, go);
                dk.fma(a.n.scale * p * (go.dot(v) - a.delta[r]), q);
            }
    }
    dk.store(a.dk + at(a.s[6], b, hk, j));
    dv.store(a.dv + at(a.s[7], b, hk, j));
}

}  // namespace

int attn_bwd_fault_take(unsigned int* bits) { return take_attn_fault(bits); }

int64_t attention_bwd_work_bytes(const nb200_attn_args& n) { return n.batch * n.heads * n.seq * (int64_t)sizeof(float); }

int launch_attention_bwd(const nb200_attn_args& n, const nb200_attn_strides* strides, const void* q, const void* k,
                         const void* v, const void* o, const float* lse, const void* grad_o, void* dq, void* dk,
                         void* dv, void* work, cudaStream_t st) {
    using B = __nv_bfloat16;
    BwdArgs a;
    a.n = n;
    for (int i = 0; i < 8; ++i) a.s[i] = strides[i];
    a.q = static_cast<const B*>(q);
    a.k = static_cast<const B*>(k);
    a.v = static_cast<const B*>(v);
    a.o = static_cast<const B*>(o);
    a.go = static_cast<const B*>(grad_o);
    a.lse = lse;
    a.dq = static_cast<B*>(dq);
    a.dk = static_cast<B*>(dk);
    a.dv = static_cast<B*>(dv);
    a.delta = static_cast<float*>(work);
    const int64_t rows = n.batch * n.heads * n.seq, kv_rows = n.batch * n.kv_heads * n.seq;
    bwd_dq_kernel<<<(unsigned)((rows + kRowsPerCta - 1) / kRowsPerCta), 32 * kRowsPerCta, 0, st>>>(a);
    bwd_dkv_kernel<<<(unsigned)((kv_rows + kRowsPerCta - 1) / kRowsPerCta), 32 * kRowsPerCta, 0, st>>>(a);
    count_launch(2);
    return finish_launch("nb200_attention_bwd");
}

}  // namespace nb200
