// What the kernels of attention behind a shared prefix agree on: query rows, the keys of a part and where its
// result goes (prefix_attention.cu has the mathematics).
#pragma once

#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "fastmath.cuh"
#include "launch.h"

namespace nb200 {
namespace prefix {

struct Query {
    const void* q;
    int64_t qb, qh, qt;  // strides in elements
    int group, tokens;   // query heads per key/value head, new tokens per sequence
};  // row r = (b group + g) tokens + t of key/value head `head` is q[b, head group + g, t]

// Probabilities are rounded to the inputs' type for the product with the values, whose two operands are of one type: half a
// step of it beside the same half step of the values and of the result (bf16 2-norms of 0.0022 for 0.0017 with probabilities of
// 32 bits; the sums that divide take them unrounded). What the rounding leaves off could go into a second product; on the
// tensor cores the softmax, which bounds a tile there, would convert and store twice. They are at most 2^8 (the
// running maximum may lag behind by that much), so fp16 has room for 2^6 more: that keeps the probabilities of very
// many unlikely keys above fp16's smallest value.
constexpr float kSlack = 8.f;
template <typename T> constexpr float kLift = std::is_same<T, __half>::value ? 6.f : 0.f;

// A running maximum m is kept as the score it is, before scale and log2(e), and subtracted before they come in, 2^((s - m) sl2):
// so no finite score leaves fp32 on the way, and scores that are all alike weigh alike however far from 0 they are. (As
// 2^(s sl2 - m sl2) in one multiply-add, the rounding of m sl2 was left over: scores of -1e19 came out as NaN, or as no weight.)
// 2^(m sl2 - top sl2): what a sum behind maximum m weighs beside one behind `top`. Without a score but -inf the sum l is 0, or
// NaN, and weighs that.
__device__ __forceinline__ float weight_of(float m, float l, float top, float sl2) {
    return m == -NB200_INF ? l : ex2((m - top) * sl2);
}
// The natural log-sum-exp of a row.
template <typename T>
__device__ __forceinline__ float natural_lse(float m, float l, float scale) {
    return l == 0.f ? -NB200_INF : fmaf(m, scale, (log2f(l) - kLift<T>) * 0.69314718055994531f);
}

// The prefix on the tensor cores (prefix_attention_tc.cu): query rows of a key/value head in blocks of 256, the
// prefix's tiles of 128 keys in `splits` nearly equal ranges. Results as of any part: o [splits][kv_heads][rows][D],
// ml [splits][kv_heads][rows].
struct TensorPart {
    Query query;
    int kv_heads, rows, keys, splits;
    float sl2, slack;  // scale * log2(e), and kSlack in scores
    float* o;
    float2* ml;
};
// kSlack as a difference of scores; where scores count for next to nothing, still one that can be added to them.
inline float slack_of(float sl2) { return std::min(kSlack / sl2, 1e30f); }
// [batch, heads, keys, D] as a tensor map with a {64, box_keys} box and 128-byte swizzle. The stride of a dimension of one
// element is never used and may be anything.
int encode_keys(CUtensorMap* map, const char* what, const void* base, int dtype, int64_t d, int64_t keys, int64_t heads,
                int64_t batch, const nb200_attn_strides& s, uint32_t box_keys);

// `other_bytes`: what the kernel beside it reads.
int tensor_splits(int64_t kv_heads, int64_t rows, int64_t keys, int64_t other_bytes);
int launch_tensor_part(const TensorPart& a, int dtype, int64_t head_dim, const void* k, const nb200_attn_strides& ks,
                       const void* v, const nb200_attn_strides& vs, cudaStream_t st);

}  // namespace prefix
}  // namespace nb200
