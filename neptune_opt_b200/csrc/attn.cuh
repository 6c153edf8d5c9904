// What the attention kernels share: bounded barrier waits, the stage ring, the masked tail of a tile and
// the tensor maps of strided [batch, heads, seq, 128] bf16 tensors.
#pragma once

#include <cudaTypedefs.h>

#include "common.cuh"
#include "launch.h"
#include "fastmath.cuh"
#include "tcgen05.cuh"

namespace nb200 {

constexpr int kDim = 128;  // head dimension
constexpr long long kWaitCycles = 1ll << 31;

// Bit 1 is set by a wait that ran out; one word per kernel file, read and cleared by the host.
static __device__ unsigned int g_attn_fault = 0u;

// Bounded wait on phase `parity` of `bar`. Gives up early when another role has aborted the CTA.
// (Inline on purpose: a called function would need one register budget for roles that run under
// different setmaxnreg limits.)
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (uint32_t i = 1; i < (1u << 30); ++i) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((i & 255u) == 0) {
            if (*abort) return false;
            if (clock64() - t0 > kWaitCycles) break;
        }
    }
    atomicOr(&g_attn_fault, 2u);
    *abort = 1;
    return false;
}

// Bounded wait used while shutting down: ignores the abort flag (outstanding copies and MMAs
// must land before the CTA exits) but still gives up after the same limit.
__device__ __forceinline__ void drain_bar(uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return;
    const long long t0 = clock64();
    for (uint32_t i = 1; i < (1u << 30); ++i) {
        if (mbar_try_wait(bar, parity)) return;
        if ((i & 255u) == 0 && clock64() - t0 > kWaitCycles) break;
    }
    atomicOr(&g_attn_fault, 2u);
}

// Position in a ring of kStages stages: stage index and the parity of its current fill.
template <int kStages>
struct Ring {
    int s = 0;
    uint32_t ph = 0;
    __device__ __forceinline__ void next() {
        if (++s == kStages) {
            s = 0;
            ph ^= 1u;
        }
    }
};

// Tokens of batch element b, clamped to [0, seq].
__device__ __forceinline__ int tokens_of(const int* seq_lens, int b, int seq) {
    return seq_lens ? max(0, min(seq_lens[b], seq)) : seq;
}

// Zeroes rows [row, rows) of a staged tile of two 64-column halves (a whole warp calls it). The swizzle
// permutes 16-byte chunks inside a row's 128 bytes, so a range of rows is a range of bytes in each half.
__device__ __forceinline__ void zero_tail(uint8_t* tile, int rows, int row, int lane) {
    const uint4 z = make_uint4(0u, 0u, 0u, 0u);
    for (int i = row * 8 + lane; i < rows * 8; i += 32) {
        reinterpret_cast<uint4*>(tile)[i] = z;
        reinterpret_cast<uint4*>(tile + rows * 128)[i] = z;
    }
    fence_proxy_async();
}

// ------------------------------------------------------------------ host side
// cuTensorMapEncodeTiled, or null with an error recorded.
PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder(const char* what);

// A [batch, heads, seq, 128] bf16 tensor as a 4-D tensor map with a {64, box_rows, 1, 1} box and
// 128-byte swizzle. The stride of a dimension of one element is never used and may be anything.
inline int encode_rows(CUtensorMap* map, const char* op, const char* what, const void* base, int64_t batch,
                       int64_t heads, int64_t seq, const nb200_attn_strides& s, uint32_t box_rows) {
    const auto encode = tensor_map_encoder(op);
    if (!encode) return NB200_ERR_LAUNCH;
    auto bytes = [](int64_t stride, int64_t size) { return (cuuint64_t)(size > 1 ? stride * 2 : kDim * 2); };
    const cuuint64_t dims[4] = {(cuuint64_t)kDim, (cuuint64_t)seq, (cuuint64_t)heads, (cuuint64_t)batch};
    const cuuint64_t strides[3] = {bytes(s.seq, seq), bytes(s.head, heads), bytes(s.batch, batch)};
    const cuuint32_t box[4] = {kDim / 2, box_rows, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult rc =
        encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (rc != CUDA_SUCCESS) {
        set_error("%s: cannot describe %s as a tensor map (CUresult %d)", op, what, (int)rc);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

inline int take_attn_fault(unsigned int* bits) {
    unsigned int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_attn_fault, sizeof(v)) != cudaSuccess ||
        cudaMemcpyToSymbol(g_attn_fault, &zero, sizeof(zero)) != cudaSuccess) {
        set_error("cannot read the attention fault word: %s", cudaGetErrorString(cudaGetLastError()));
        return NB200_ERR_LAUNCH;
    }
    *bits = v;
    return NB200_OK;
}

}  // namespace nb200
