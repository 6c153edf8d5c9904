// The extern "C" boundary: argument validation, error reporting and launch bookkeeping.
// Nothing here allocates device memory; every pointer is caller-owned.
#include <cudaTypedefs.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "common.cuh"
#include "fold.cuh"
#include "launch.h"

namespace nb200 {

namespace {
thread_local char g_error[512] = "";
std::atomic<uint64_t> g_launches{0};
std::mutex g_sm_mutex;
int g_sm_count[64] = {0};
}  // namespace

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
}

int sm_count() {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
    std::lock_guard<std::mutex> lock(g_sm_mutex);
    if (g_sm_count[dev] == 0) {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
        g_sm_count[dev] = n;
    }
    return g_sm_count[dev];
}

void count_launch(int n) { g_launches.fetch_add((uint64_t)n, std::memory_order_relaxed); }

int finish_launch(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) {
        set_error("%s: CUDA launch failed: %s", what, cudaGetErrorString(e));
        return NB200_ERR_LAUNCH;
    }
    return NB200_OK;
}

}  // namespace nb200

using namespace nb200;

namespace {

bool valid_dtype(int d) { return d == NB200_F32 || d == NB200_BF16 || d == NB200_F16; }

// Sizes, scale and the strides of `count` tensors in the order q, k, v, o, grad_o, dq, dk, dv.
int check_attention(const char* what, const nb200_attn_args* a, const nb200_attn_strides* s, int count) {
    if (!a || !s) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
    if (a->batch < 0 || a->heads < 0 || a->seq < 0) { set_error("%s: negative size", what); return NB200_ERR_ARG; }
    if (a->batch == 0 || a->heads == 0 || a->seq == 0) return NB200_OK;
    if (a->kv_heads < 1 || a->heads % a->kv_heads) {
        set_error("%s: %lld query heads cannot share %lld key/value heads", what, (long long)a->heads,
                  (long long)a->kv_heads);
        return NB200_ERR_ARG;
    }
    if (!std::isfinite(a->scale)) { set_error("%s: scale must be finite", what); return NB200_ERR_ARG; }
    if (a->head_dim != 128) {
        set_error("%s: head_dim %lld is not supported (the kernels are built for 128)", what, (long long)a->head_dim);
        return NB200_ERR_UNSUPPORTED;
    }
    if (!(a->scale > 0.f)) { set_error("%s: scale must be positive", what); return NB200_ERR_ARG; }
    const int64_t most = (int64_t)1 << 30;
    if (a->seq > most || a->batch > most || a->heads > most || a->batch * a->heads > most) {
        set_error("%s: batch*heads=%lld*%lld, seq=%lld exceed the kernel's index range", what, (long long)a->batch,
                  (long long)a->heads, (long long)a->seq);
        return NB200_ERR_CAPACITY;
    }
    // The copies' limits: multiples of 16 bytes, below 2^40 bytes.
    auto bad = [](int64_t stride, int64_t size) { return size > 1 && (stride < 8 || stride % 8 || stride >= (int64_t)1 << 39); };
    for (int i = 0; i < count; ++i) {
        const bool kv = i == 1 || i == 2 || i >= 6;
        if (bad(s[i].batch, a->batch) || bad(s[i].head, kv ? a->kv_heads : a->heads) || bad(s[i].seq, a->seq)) {
            set_error("%s: strides must be positive multiples of 8 elements (tensor %d)", what, i);
            return NB200_ERR_ARG;
        }
    }
    return NB200_OK;
}

int check_attention_pointers(const char* what, const void* const* tensors, int count, const float* lse,
                             const int32_t* seq_lens) {
    for (int i = 0; i < count; ++i) {
        if (!tensors[i]) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
        if (!aligned16(tensors[i])) { set_error("%s: tensors must be 16-byte aligned", what); return NB200_ERR_ARG; }
    }
    if (((uintptr_t)lse | (uintptr_t)seq_lens) & 3u) {
        set_error("%s: lse and seq_lens must be 4-byte aligned", what);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

int check_norm(const char* what, const nb200_norm_args* a, int dtype, bool with_eps) {
    if (!a) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
    if (!valid_dtype(dtype)) { set_error("%s: unsupported dtype %d", what, dtype); return NB200_ERR_ARG; }
    if (a->rows < 0 || a->width < 1) { set_error("%s: need rows >= 0 and width >= 1", what); return NB200_ERR_ARG; }
    if (a->rows > 0x7fffffffLL) { set_error("%s: too many rows", what); return NB200_ERR_CAPACITY; }
    if (a->gate && (a->rows_per_gate < 1 || a->rows % a->rows_per_gate)) {
        set_error("%s: %lld rows are not whole groups of %lld", what, (long long)a->rows, (long long)a->rows_per_gate);
        return NB200_ERR_ARG;
    }
    if (a->gate_act < NB200_GATE_NONE || a->gate_act > NB200_GATE_SIGMOID || !std::isfinite(a->scale) ||
        (with_eps && !(std::isfinite(a->eps) && a->eps > 0))) {
        set_error("%s: unknown gate activation, or scale or eps out of range", what);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

int check_distill(const char* what, const nb200_distill_args* a) {
    if (!a) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
    if (!valid_dtype(a->dtype) || !valid_dtype(a->teacher_dtype) ||
        (a->index_dtype != NB200_I32 && a->index_dtype != NB200_I64)) {
        set_error("%s: unsupported dtype", what);
        return NB200_ERR_ARG;
    }
    if (a->rows < 0 || a->vocab < 1 || a->top < 0) {
        set_error("%s: need rows >= 0, vocab >= 1 and top >= 0", what);
        return NB200_ERR_ARG;
    }
    if (!(std::isfinite(a->temperature) && a->temperature > 0)) {
        set_error("%s: temperature must be finite and positive", what);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

int check_prefix_attention(const char* what, const nb200_prefix_attn_args* a, const nb200_attn_strides* s) {
    if (!a || !s) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
    if (a->dtype != NB200_BF16 && a->dtype != NB200_F16) {
        set_error("%s: dtype must be bfloat16 or float16", what);
        return NB200_ERR_ARG;
    }
    if (a->batch < 0 || a->heads < 0 || a->tokens < 0 || a->prefix < 0 || a->cache < 0) {
        set_error("%s: negative size", what);
        return NB200_ERR_ARG;
    }
    if (a->batch == 0 || a->heads == 0 || a->tokens == 0) return NB200_OK;
    if (a->kv_heads < 1 || a->heads % a->kv_heads) {
        set_error("%s: %lld query heads cannot share %lld key/value heads", what, (long long)a->heads,
                  (long long)a->kv_heads);
        return NB200_ERR_ARG;
    }
    if (a->head_dim != 64 && a->head_dim != 128) {
        set_error("%s: head_dim %lld is not supported (the kernels are built for 64 and 128)", what,
                  (long long)a->head_dim);
        return NB200_ERR_UNSUPPORTED;
    }
    if (!std::isfinite(a->scale) || !(a->scale > 0.f)) {
        set_error("%s: scale must be finite and positive", what);
        return NB200_ERR_ARG;
    }
    const int64_t most = (int64_t)1 << 30;
    if (a->batch > most || a->heads > most || a->tokens > most || a->prefix > most || a->cache > most ||
        a->batch * a->heads > most || a->batch * a->heads * a->tokens > most) {
        set_error("%s: batch=%lld, heads=%lld, tokens=%lld, prefix=%lld, cache=%lld exceed the kernel's index range", what,
                  (long long)a->batch, (long long)a->heads, (long long)a->tokens, (long long)a->prefix,
                  (long long)a->cache);
        return NB200_ERR_CAPACITY;
    }
    // The steps of 16 keys that the tiles of 8 query rows take, which the kernels count in 32 bits for a worker, and for
    // one tile of every sequence. (Only tensors whose rows overlap get this far.)
    const int64_t own_tiles = a->heads / a->kv_heads * a->tokens / 8 + 1, tiles = a->batch * own_tiles;
    const int64_t own_steps = a->batch * (a->cache / 16 + 3), prefix_steps = a->prefix / 16 + 3;
    if (own_steps > most || (double)a->kv_heads * ((double)own_tiles * own_steps + (double)tiles * prefix_steps) > 0x1p40) {
        set_error("%s: batch=%lld, prefix=%lld, cache=%lld exceed the kernel's index range", what, (long long)a->batch,
                  (long long)a->prefix, (long long)a->cache);
        return NB200_ERR_CAPACITY;
    }
    // The copies' limits: multiples of 16 bytes, below 2^40 bytes.
    auto bad = [](int64_t stride, int64_t size) { return size > 1 && (stride < 8 || stride % 8 || stride >= (int64_t)1 << 39); };
    for (int i = 0; i < 5; ++i) {
        const bool shared = i == 1 || i == 2;
        const int64_t seq = i == 0 ? a->tokens : shared ? a->prefix : a->cache;
        if (seq == 0) continue;
        if ((!shared && bad(s[i].batch, a->batch)) || bad(s[i].head, i ? a->kv_heads : a->heads) || bad(s[i].seq, seq)) {
            set_error("%s: strides must be positive multiples of 8 elements (tensor %d)", what, i);
            return NB200_ERR_ARG;
        }
    }
    return NB200_OK;
}

int check_norm8(const char* what, const nb200_norm8_args* a) {
    if (!a) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
    if (!valid_dtype(a->dtype)) { set_error("%s: unsupported dtype %d", what, a->dtype); return NB200_ERR_ARG; }
    if (a->kind < NB200_E4M3 || a->kind > NB200_I8) {
        set_error("%s: unknown 8-bit type %d", what, a->kind);
        return NB200_ERR_ARG;
    }
    if (a->rows < 0 || a->width < 1) { set_error("%s: need rows >= 0 and width >= 1", what); return NB200_ERR_ARG; }
    if (a->group != 0 && a->group != 16 && a->group != 32 && a->group != 64 && a->group != 128) {
        set_error("%s: group must be 0, 16, 32, 64 or 128, got %lld", what, (long long)a->group);
        return NB200_ERR_ARG;
    }
    if (a->group && a->width % a->group) {
        set_error("%s: width %lld is not whole groups of %lld", what, (long long)a->width, (long long)a->group);
        return NB200_ERR_ARG;
    }
    if (!std::isfinite(a->eps) || !((float)a->eps > 0.f) || !std::isfinite((float)a->eps)) {
        set_error("%s: eps must be finite and positive in fp32", what);
        return NB200_ERR_ARG;
    }
    if (a->width > 16384) {
        set_error("%s: width %lld exceeds 16384", what, (long long)a->width);
        return NB200_ERR_CAPACITY;
    }
    if (a->rows > 1 && (a->stride_x < 0 || (a->residual && a->stride_residual < 0))) {
        set_error("%s: negative stride", what);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

int check_logits(const char* what, const nb200_logits_args* a) {
    if (!a) { set_error("%s: null pointer", what); return NB200_ERR_ARG; }
    auto index = [](int32_t d) { return d == NB200_I32 || d == NB200_I64; };
    if (!valid_dtype(a->dtype) || (a->history && !index(a->token_dtype)) || (a->biases && !index(a->bias_dtype))) {
        set_error("%s: unsupported dtype", what);
        return NB200_ERR_ARG;
    }
    if (a->rows < 0 || a->vocab < 1 || a->history < 0 || a->biases < 0) {
        set_error("%s: need rows >= 0, vocab >= 1, history >= 0 and biases >= 0", what);
        return NB200_ERR_ARG;
    }
    const int64_t most = (int64_t)1 << 30;
    if (a->rows > most || a->vocab > most || a->history >= most / 2 || a->biases > 1024) {
        set_error("%s: rows=%lld, vocab=%lld, history=%lld or biases=%lld (at most 1024) exceed the kernel's range", what,
                  (long long)a->rows, (long long)a->vocab, (long long)a->history, (long long)a->biases);
        return NB200_ERR_CAPACITY;
    }
    if (a->rows > 1 && (a->stride_logits < 0 || a->stride_tokens < 0 || a->stride_bias_index < 0 ||
                        a->stride_bias_value < 0 || a->stride_allowed < 0)) {
        set_error("%s: negative stride", what);
        return NB200_ERR_ARG;
    }
    return NB200_OK;
}

// Declared-parameter checks of the reference's certificate (algebra.py:285-302): every declared
// scalar finite, T/beta/N/eps strictly positive, tiny nonnegative.
int check_params(int sk, const nb200_params* q, nb200_params* out) {
    nb200_params p{};
    if (q) p = *q;
    *out = p;
    auto finite = [](double v) { return std::isfinite(v); };
    switch (sk) {
        case NB200_LOGSUMEXP:
            if (!finite(p.tiny) || p.tiny < 0) { set_error("parameter 'tiny' must be finite and nonnegative"); return NB200_ERR_ARG; }
            return NB200_OK;
        case NB200_LSE_BIASED:
            if (!finite(p.tiny) || p.tiny < 0) { set_error("parameter 'tiny' must be finite and nonnegative"); return NB200_ERR_ARG; }
            if (!finite(p.alpha)) { set_error("parameter 'alpha' must be finite"); return NB200_ERR_ARG; }
            return NB200_OK;
        case NB200_LSE_SCALED:
            if (!finite(p.tiny) || p.tiny < 0) { set_error("parameter 'tiny' must be finite and nonnegative"); return NB200_ERR_ARG; }
            if (!finite(p.T) || p.T <= 0) { set_error("parameter 'T' must be finite and positive"); return NB200_ERR_ARG; }
            return NB200_OK;
        case NB200_SOFTCAP_LSE:
            if (!finite(p.tiny) || p.tiny < 0) { set_error("parameter 'tiny' must be finite and nonnegative"); return NB200_ERR_ARG; }
            if (!finite(p.beta) || p.beta <= 0) { set_error("parameter 'beta' must be finite and positive"); return NB200_ERR_ARG; }
            return NB200_OK;
        case NB200_DECAY_RENORM:
            if (!finite(p.N) || p.N <= 0) { set_error("parameter 'N' must be finite and positive"); return NB200_ERR_ARG; }
            return NB200_OK;
        case NB200_RMSNORM_MAX:
            if (!finite(p.eps) || p.eps <= 0) { set_error("parameter 'eps' must be finite and positive"); return NB200_ERR_ARG; }
            return NB200_OK;
        case NB200_STABLE_L2: case NB200_LINEAR_ATTN: case NB200_SUMSQ_DIV:
        case NB200_VARIANCE: case NB200_STD:
            return NB200_OK;
    }
    set_error("unknown skeleton %d", sk);
    return NB200_ERR_ARG;
}

int check_rows(const void* x, int dtype, int64_t rows, int64_t ncols, const void* out, const char* what) {
    if (!valid_dtype(dtype)) { set_error("%s: unsupported dtype %d; expected float16/bfloat16/float32", what, dtype); return NB200_ERR_ARG; }
    if (rows < 0) { set_error("%s: negative row count", what); return NB200_ERR_ARG; }
    if (ncols <= 0) { set_error("%s: Neptune requires positive last-dimension width", what); return NB200_ERR_ARG; }
    if (rows > 0 && (x == nullptr || out == nullptr)) { set_error("%s: null data pointer", what); return NB200_ERR_ARG; }
    return NB200_OK;
}

int check_launch(const nb200_launch* L) {
    if (!L) return NB200_OK;
    if (L->variant < 0 || L->variant > NB200_VARIANT_CLUSTER) { set_error("unknown launch variant %d", L->variant); return NB200_ERR_ARG; }
    if (L->threads && (L->threads < 64 || L->threads > 512 || L->threads % 32)) {
        set_error("launch threads must be a multiple of 32 in [64, 512]"); return NB200_ERR_ARG;
    }
    if (L->ctas_per_sm < 0 || L->ctas_per_sm > 32) { set_error("ctas_per_sm must be in [0, 32]"); return NB200_ERR_ARG; }
    if (L->variant == NB200_VARIANT_CLUSTER) {
        if (L->stages != 0 && (L->stages < 2 || L->stages > 16)) {
            set_error("cluster launches take 2..16 CTAs per row (stages field), or 0 to choose");
            return NB200_ERR_ARG;
        }
    } else if (L->stages < 0 || L->stages > 8) { set_error("stages must be in [0, 8]"); return NB200_ERR_ARG; }
    return NB200_OK;
}

}  // namespace

extern "C" {

const char* nb200_last_error(void) { return g_error; }
const char* nb200_version(void) { return "neptune_b200 0.1 (sm_100a)"; }
uint64_t nb200_launch_count(void) { return g_launches.load(std::memory_order_relaxed); }

int nb200_stream_fault(uint32_t* bits) {
    if (!bits) { set_error("nb200_stream_fault: null pointer"); return NB200_ERR_ARG; }
    unsigned int v = 0, w = 0, x = 0, y = 0, z = 0, p = 0, q = 0;
    int rc = stream_fault_take(&v);
    if (rc == NB200_OK) rc = attn_fault_take(&w);
    if (rc == NB200_OK) rc = peer_fault_take(&x);
    if (rc == NB200_OK) rc = attn_bwd_fault_take(&y);
    if (rc == NB200_OK) rc = norm_fault_take(&z);
    if (rc == NB200_OK) rc = prefix_fault_take(&p);
    if (rc == NB200_OK) rc = prefix_stream_fault_take(&q);
    *bits = v | w | x | y | z | p | q;
    return rc;
}

int nb200_fold(int skeleton, const nb200_params* params, const void* x, int dtype, int64_t rows,
               int64_t ncols, int64_t stride_row, int64_t stride_col, void* out,
               const nb200_launch* launch, void* stream) {
    nb200_params q;
    int rc = check_params(skeleton, params, &q);
    if (rc) return rc;
    if ((rc = check_rows(x, dtype, rows, ncols, out, "nb200_fold"))) return rc;
    if ((rc = check_launch(launch))) return rc;
    if (rows == 0) return NB200_OK;
    return launch_fold(skeleton, make_params(q, ncols), x, dtype, rows, ncols, stride_row, stride_col,
                       out, launch, (cudaStream_t)stream);
}

int nb200_softmax(int mode, const void* x, int dtype, int64_t rows, int64_t ncols, int64_t stride_row,
                  int64_t stride_col, void* y, void* lse, const nb200_launch* launch, void* stream) {
    if (mode != 0 && mode != 1) { set_error("nb200_softmax: mode must be 0 (softmax) or 1 (log_softmax)"); return NB200_ERR_ARG; }
    int rc = check_rows(x, dtype, rows, ncols, y, "nb200_softmax");
    if (rc) return rc;
    if ((rc = check_launch(launch))) return rc;
    if (rows == 0) return NB200_OK;
    return launch_softmax(mode, x, dtype, rows, ncols, stride_row, stride_col, y, lse, launch,
                          (cudaStream_t)stream);
}

int nb200_l2_normalize(const void* x, int dtype, int64_t rows, int64_t ncols, int64_t stride_row,
                       int64_t stride_col, void* y, void* norm, const nb200_launch* launch, void* stream) {
    int rc = check_rows(x, dtype, rows, ncols, y, "nb200_l2_normalize");
    if (rc) return rc;
    if ((rc = check_launch(launch))) return rc;
    if (rows == 0) return NB200_OK;
    return launch_l2(x, dtype, rows, ncols, stride_row, stride_col, y, norm, launch, (cudaStream_t)stream);
}

int64_t nb200_fold_split_scratch_bytes(int64_t rows, int64_t nparts) {
    if (rows < 0 || nparts < 0) return -1;
    return rows * nparts * (int64_t)sizeof(nb200_state);
}

int nb200_fold_partial(int skeleton, const nb200_params* params, const void* x, int dtype, int64_t rows,
                       int64_t ncols_total, int64_t col_begin, int64_t ncols_shard, int64_t stride_row,
                       int64_t stride_col, int64_t chunk_cols, nb200_state* states, const nb200_launch* launch,
                       void* stream) {
    nb200_params q;
    int rc = check_params(skeleton, params, &q);
    if (rc) return rc;
    if ((rc = check_rows(x, dtype, rows, ncols_total, states, "nb200_fold_partial"))) return rc;
    if (col_begin < 0 || ncols_shard <= 0 || col_begin + ncols_shard > ncols_total) {
        set_error("nb200_fold_partial: column shard [%lld, %lld) outside [0, %lld)", (long long)col_begin,
                  (long long)(col_begin + ncols_shard), (long long)ncols_total);
        return NB200_ERR_ARG;
    }
    if (chunk_cols <= 0) { set_error("nb200_fold_partial: chunk_cols must be positive"); return NB200_ERR_ARG; }
    if ((rc = check_launch(launch))) return rc;
    if (rows > 0 && !aligned16(states)) { set_error("nb200_fold_partial: states must be 16-byte aligned"); return NB200_ERR_ARG; }
    if (rows == 0) return NB200_OK;
    const int64_t nparts = (ncols_shard + chunk_cols - 1) / chunk_cols;
    return launch_partial(skeleton, make_params(q, ncols_total), x, dtype, rows, col_begin, ncols_shard,
                          stride_row, stride_col, chunk_cols, nparts, states, launch, (cudaStream_t)stream);
}

int nb200_fold_merge(int skeleton, const nb200_params* params, const nb200_state* states, int64_t rows,
                     int64_t nparts, int64_t row_stride, int64_t part_stride, void* out, int dtype,
                     void* stream) {
    nb200_params q;
    int rc = check_params(skeleton, params, &q);
    if (rc) return rc;
    if (!valid_dtype(dtype)) { set_error("nb200_fold_merge: unsupported dtype %d", dtype); return NB200_ERR_ARG; }
    if (rows < 0 || nparts <= 0) { set_error("nb200_fold_merge: need rows >= 0 and nparts > 0"); return NB200_ERR_ARG; }
    if (rows == 0) return NB200_OK;
    if (!states || !out) { set_error("nb200_fold_merge: null pointer"); return NB200_ERR_ARG; }
    return launch_merge(skeleton, make_params(q, 0), states, rows, nparts, row_stride, part_stride, out,
                        dtype, (cudaStream_t)stream);
}

int nb200_fold_split(int skeleton, const nb200_params* params, const void* x, int dtype, int64_t rows,
                     int64_t ncols, int64_t stride_row, int64_t stride_col, int64_t chunk_cols,
                     void* scratch, int64_t scratch_bytes, void* out, const nb200_launch* launch, void* stream) {
    nb200_params q;
    int rc = check_params(skeleton, params, &q);
    if (rc) return rc;
    if ((rc = check_rows(x, dtype, rows, ncols, out, "nb200_fold_split"))) return rc;
    if (skeleton == NB200_VARIANCE || skeleton == NB200_STD) {
        set_error("two_pass needs extended carried state; split refused");
        return NB200_ERR_UNSUPPORTED;
    }
    if (chunk_cols <= 0) { set_error("nb200_fold_split: chunk_cols must be positive"); return NB200_ERR_ARG; }
    if ((rc = check_launch(launch))) return rc;
    const int64_t nparts = (ncols + chunk_cols - 1) / chunk_cols;
    if (nparts > 4096) {
        set_error("split needs %lld partials, exceeding capacity 4096; use serial", (long long)nparts);
        return NB200_ERR_CAPACITY;
    }
    if (rows == 0) return NB200_OK;
    const int64_t need = nb200_fold_split_scratch_bytes(rows, nparts);
    if (!scratch || scratch_bytes < need || !aligned16(scratch)) {
        set_error("nb200_fold_split: scratch needs %lld bytes, 16-byte aligned (got %lld)", (long long)need,
                  (long long)scratch_bytes);
        return NB200_ERR_ARG;
    }
    nb200_state* states = (nb200_state*)scratch;
    const Params p = make_params(q, ncols);
    rc = launch_partial(skeleton, p, x, dtype, rows, 0, ncols, stride_row, stride_col, chunk_cols, nparts,
                        states, launch, (cudaStream_t)stream);
    if (rc) return rc;
    return launch_merge(skeleton, p, states, rows, nparts, nparts, 1, out, dtype, (cudaStream_t)stream);
}

int nb200_rms_norm(const void* x, const void* gamma, int dtype, int64_t rows, int64_t ncols,
                   int64_t stride_row, int64_t stride_col, int64_t stride_gamma, double eps, void* out,
                   const nb200_launch* launch, void* stream) {
    int rc = check_rows(x, dtype, rows, ncols, out, "nb200_rms_norm");
    if (rc) return rc;
    if ((rc = check_launch(launch))) return rc;
    if (!std::isfinite(eps) || eps <= 0) { set_error("RMSNorm requires an explicit finite positive eps"); return NB200_ERR_ARG; }
    if (rows == 0) return NB200_OK;
    if (!gamma) { set_error("nb200_rms_norm: null gamma"); return NB200_ERR_ARG; }
    return launch_rms(x, gamma, dtype, rows, ncols, stride_row, stride_col, stride_gamma, (float)eps, out,
                      launch, (cudaStream_t)stream);
}

int nb200_segment_spans(const void* lengths, int index_dtype, int64_t nsegments, int64_t length_stride,
                        int unsafe, int64_t nrows, int64_t* spans, uint32_t* status, void* stream) {
    if (index_dtype != NB200_I32 && index_dtype != NB200_I64) {
        set_error("segment index dtype must be int32/int64"); return NB200_ERR_ARG;
    }
    if (nsegments < 0 || nrows < 0) { set_error("nb200_segment_spans: negative size"); return NB200_ERR_ARG; }
    if (!spans || (nsegments > 0 && !lengths)) { set_error("nb200_segment_spans: null pointer"); return NB200_ERR_ARG; }
    return launch_spans(lengths, index_dtype, nsegments, length_stride, unsafe, nrows, spans, status,
                        (cudaStream_t)stream);
}

int nb200_segment_pool(const void* data, int dtype, int64_t nrows, int64_t channels, int64_t stride_row,
                       int64_t stride_channel, const void* bounds, int index_dtype, int64_t bound_stride,
                       int64_t nsegments, int reduce, int has_initial, uint32_t initial_bits, void* out,
                       uint32_t* status, void* stream) {
    if (!valid_dtype(dtype)) { set_error("segment data dtype must be float16/bfloat16/float32"); return NB200_ERR_ARG; }
    if (index_dtype != NB200_I32 && index_dtype != NB200_I64) {
        set_error("segment index dtype must be int32/int64"); return NB200_ERR_ARG;
    }
    if (reduce != 0 && reduce != 1) { set_error("segment reduce must be 0 (sum) or 1 (mean)"); return NB200_ERR_ARG; }
    if (nrows < 0 || channels < 0 || nsegments < 0) { set_error("nb200_segment_pool: negative size"); return NB200_ERR_ARG; }
    if (nsegments == 0 || channels == 0) return NB200_OK;
    if (!bounds || !out || (nrows > 0 && !data)) { set_error("nb200_segment_pool: null pointer"); return NB200_ERR_ARG; }
    return launch_segment_pool(data, dtype, nrows, channels, stride_row, stride_channel, bounds, index_dtype,
                               bound_stride, nsegments, reduce, has_initial, initial_bits, out, status,
                               (cudaStream_t)stream);
}

int64_t nb200_peer_buffer_bytes(int64_t rows, int64_t world, int64_t nparts) {
    if (rows < 0 || world < 1 || world > peer_max_world() || nparts < 1) return -1;
    return peer_buffer_bytes(rows, world, nparts);
}

int nb200_peer_init(void* buffer, int64_t rows, int world, int64_t nparts, void* stream) {
    if (world < 1 || world > peer_max_world() || rows < 0 || nparts < 1) {
        set_error("nb200_peer_init: need 1 <= world <= %d, rows >= 0, nparts >= 1", peer_max_world());
        return NB200_ERR_ARG;
    }
    if (!buffer || (reinterpret_cast<uintptr_t>(buffer) & 255u)) {
        set_error("nb200_peer_init: null or unaligned buffer");
        return NB200_ERR_ARG;
    }
    return launch_peer_init(buffer, rows, nparts, world, (cudaStream_t)stream);
}

int nb200_peer_push(const nb200_state* states, int64_t rows, int64_t nlocal, int64_t nparts, void* const* peers,
                    int world, int rank, void* buffer, void* stream) {
    if (world < 1 || world > peer_max_world() || rank < 0 || rank >= world) {
        set_error("nb200_peer_push: need 1 <= world <= %d and 0 <= rank < world", peer_max_world());
        return NB200_ERR_ARG;
    }
    if (rows < 0 || nlocal < 0 || nparts < 1 || nlocal > nparts) {
        set_error("nb200_peer_push: need rows >= 0 and 0 <= nlocal <= nparts, nparts >= 1");
        return NB200_ERR_ARG;
    }
    if (!peers || !buffer || (rows > 0 && nlocal > 0 && !states)) {
        set_error("nb200_peer_push: null pointer");
        return NB200_ERR_ARG;
    }
    for (int r = 0; r < world; ++r)
        if (!peers[r] || (reinterpret_cast<uintptr_t>(peers[r]) & 255u)) {
            set_error("nb200_peer_push: exchange buffer of rank %d is null or not 256-byte aligned", r);
            return NB200_ERR_ARG;
        }
    if (peers[rank] != buffer) {
        set_error("nb200_peer_push: peers[rank] must be this rank's own buffer");
        return NB200_ERR_ARG;
    }
    return launch_peer_push(states, rows, nlocal, nparts, peers, world, rank, buffer, (cudaStream_t)stream);
}

int nb200_peer_fold(int skeleton, const nb200_params* params, const void* x, int dtype, int64_t rows,
                    int64_t ncols_total, int64_t ncols_shard, int64_t stride_row, int64_t chunk_cols, int64_t nparts,
                    void* const* peers, int world, int rank, void* buffer, void* out, void* stream) {
    nb200_params q;
    int rc = check_params(skeleton, params, &q);
    if (rc) return rc;
    if (!valid_dtype(dtype)) { set_error("nb200_peer_fold: unsupported dtype %d", dtype); return NB200_ERR_ARG; }
    if (world < 1 || world > peer_max_world() || rank < 0 || rank >= world) {
        set_error("nb200_peer_fold: need 1 <= world <= %d and 0 <= rank < world", peer_max_world());
        return NB200_ERR_ARG;
    }
    if (rows < 0 || ncols_shard < 1 || ncols_total < ncols_shard || chunk_cols < 1 || nparts < 1 || stride_row < 0) {
        set_error("nb200_peer_fold: need rows >= 0, 1 <= ncols_shard <= ncols_total, chunk_cols >= 1, nparts >= 1");
        return NB200_ERR_ARG;
    }
    if (!peers || !buffer || (rows > 0 && (!x || !out))) {
        set_error("nb200_peer_fold: null pointer");
        return NB200_ERR_ARG;
    }
    for (int r = 0; r < world; ++r)
        if (!peers[r] || (reinterpret_cast<uintptr_t>(peers[r]) & 255u)) {
            set_error("nb200_peer_fold: exchange buffer of rank %d is null or not 256-byte aligned", r);
            return NB200_ERR_ARG;
        }
    if (peers[rank] != buffer) {
        set_error("nb200_peer_fold: peers[rank] must be this rank's own buffer");
        return NB200_ERR_ARG;
    }
    if (rows == 0) return NB200_OK;
    return launch_peer_fold(skeleton, make_params(q, ncols_total), x, dtype, rows, ncols_shard, stride_row, chunk_cols,
                            nparts, peers, world, rank, buffer, out, (cudaStream_t)stream);
}

int nb200_peer_merge(int skeleton, const nb200_params* params, void* buffer, int64_t rows, int64_t nparts,
                     int world, void* out, int dtype, void* stream) {
    nb200_params q;
    int rc = check_params(skeleton, params, &q);
    if (rc) return rc;
    if (!valid_dtype(dtype)) { set_error("nb200_peer_merge: unsupported dtype %d", dtype); return NB200_ERR_ARG; }
    if (world < 1 || world > peer_max_world() || rows < 0 || nparts < 1) {
        set_error("nb200_peer_merge: need 1 <= world <= %d, rows >= 0, nparts >= 1", peer_max_world());
        return NB200_ERR_ARG;
    }
    if (!buffer || (rows > 0 && !out) || (reinterpret_cast<uintptr_t>(buffer) & 255u)) {
        set_error("nb200_peer_merge: null or unaligned pointer");
        return NB200_ERR_ARG;
    }
    return launch_peer_merge(skeleton, make_params(q, 0), buffer, rows, nparts, world, out, dtype,
                             (cudaStream_t)stream);
}

int nb200_ipc_handle(const void* ptr, void* handle, int64_t* offset) {
    if (!ptr || !handle || !offset) { set_error("nb200_ipc_handle: null pointer"); return NB200_ERR_ARG; }
    static PFN_cuMemGetAddressRange_v3020 range = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &fn, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            range = reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(fn);
        cudaGetLastError();
    });
    CUdeviceptr base = 0;
    size_t size = 0;
    if (!range || range(&base, &size, reinterpret_cast<CUdeviceptr>(ptr)) != CUDA_SUCCESS) {
        set_error("nb200_ipc_handle: %p is not device memory this process allocated", ptr);
        return NB200_ERR_ARG;
    }
    cudaIpcMemHandle_t h;
    if (cudaIpcGetMemHandle(&h, reinterpret_cast<void*>(base)) != cudaSuccess) {
        set_error("nb200_ipc_handle: %s", cudaGetErrorString(cudaGetLastError()));
        return NB200_ERR_LAUNCH;
    }
    std::memcpy(handle, &h, sizeof(h));
    *offset = (int64_t)(reinterpret_cast<uintptr_t>(ptr) - (uintptr_t)base);
    return NB200_OK;
}

int nb200_ipc_open(const void* handle, void** base) {
    if (!handle || !base) { set_error("nb200_ipc_open: null pointer"); return NB200_ERR_ARG; }
    cudaIpcMemHandle_t h;
    std::memcpy(&h, handle, sizeof(h));
    if (cudaIpcOpenMemHandle(base, h, cudaIpcMemLazyEnablePeerAccess) != cudaSuccess) {
        set_error("nb200_ipc_open: %s", cudaGetErrorString(cudaGetLastError()));
        return NB200_ERR_LAUNCH;
    }
    return NB200_OK;
}

int nb200_ipc_close(void* base) {
    if (!base) { set_error("nb200_ipc_close: null pointer"); return NB200_ERR_ARG; }
    if (cudaIpcCloseMemHandle(base) != cudaSuccess) {
        set_error("nb200_ipc_close: %s", cudaGetErrorString(cudaGetLastError()));
        return NB200_ERR_LAUNCH;
    }
    return NB200_OK;
}

int nb200_attention(const void* q, const void* k, const void* v, void* o, float* lse, int64_t batch,
                    int64_t heads, int64_t seq, int64_t head_dim, int causal, float scale, void* stream) {
    const nb200_attn_args a = {batch, heads, heads, seq, head_dim, nullptr, causal, scale};
    const nb200_attn_strides s = {heads * seq * head_dim, seq * head_dim, head_dim};
    const nb200_attn_strides all[4] = {s, s, s, s};
    return nb200_attention_fwd(&a, all, q, k, v, o, lse, stream);
}

int nb200_attention_fwd(const nb200_attn_args* args, const nb200_attn_strides* strides, const void* q, const void* k,
                        const void* v, void* o, float* lse, void* stream) {
    int rc = check_attention("nb200_attention", args, strides, 4);
    if (rc) return rc;
    if (args->batch * args->heads * args->seq == 0) return NB200_OK;
    const void* tensors[4] = {q, k, v, o};
    if ((rc = check_attention_pointers("nb200_attention", tensors, 4, lse, args->seq_lens))) return rc;
    return launch_attention(*args, strides, q, k, v, o, lse, (cudaStream_t)stream);
}

int64_t nb200_attention_bwd_work_bytes(const nb200_attn_args* args) {
    const nb200_attn_strides none[8] = {};
    const int rc = check_attention("nb200_attention_bwd", args, none, 0);
    if (rc) return rc;
    return args->batch * args->heads * args->seq ? attention_bwd_work_bytes(*args) : 0;
}

int nb200_attention_bwd(const nb200_attn_args* args, const nb200_attn_strides* strides, const void* q, const void* k,
                        const void* v, const void* o, const float* lse, const void* grad_o, void* dq, void* dk,
                        void* dv, void* work, int64_t work_bytes, void* stream) {
    int rc = check_attention("nb200_attention_bwd", args, strides, 8);
    if (rc) return rc;
    if (args->batch * args->heads * args->seq == 0) return NB200_OK;
    const void* tensors[8] = {q, k, v, o, grad_o, dq, dk, dv};
    if ((rc = check_attention_pointers("nb200_attention_bwd", tensors, 8, lse, args->seq_lens))) return rc;
    if (!lse) { set_error("nb200_attention_bwd: null pointer"); return NB200_ERR_ARG; }
    if (!work || !aligned16(work) || work_bytes < attention_bwd_work_bytes(*args)) {
        set_error("nb200_attention_bwd: work must hold %lld bytes, 16-byte aligned",
                  (long long)attention_bwd_work_bytes(*args));
        return NB200_ERR_ARG;
    }
    return launch_attention_bwd(*args, strides, q, k, v, o, lse, grad_o, dq, dk, dv, work, (cudaStream_t)stream);
}

int nb200_gated_norm(const nb200_norm_args* args, int dtype, void* y, void* h, float* rstd, void* stream) {
    const int rc = check_norm("nb200_gated_norm", args, dtype, true);
    if (rc) return rc;
    if (args->rows == 0) return NB200_OK;
    if (!args->x || !args->residual || !y || !rstd || (args->pre_weight && !h) || ((uintptr_t)rstd & 7u)) {
        set_error("nb200_gated_norm: null pointer, or rstd not 8-byte aligned");
        return NB200_ERR_ARG;
    }
    return launch_norm_fwd(*args, dtype, y, h, rstd, (cudaStream_t)stream);
}

int64_t nb200_gated_norm_bwd_work_bytes(const nb200_norm_args* args) {
    const int rc = check_norm("nb200_gated_norm_bwd", args, NB200_F32, false);
    if (rc) return rc;
    return args->rows ? norm_bwd_work_bytes(*args) : 0;
}

int nb200_gated_norm_bwd(const nb200_norm_args* args, int dtype, const float* rstd, const void* grad_y,
                         const void* grad_h, void* dx, void* dresidual, void* dgate, void* dpost, void* dpre,
                         void* work, int64_t work_bytes, void* stream) {
    const int rc = check_norm("nb200_gated_norm_bwd", args, dtype, false);
    if (rc) return rc;
    if (args->rows == 0) return NB200_OK;
    if (!args->x || !args->residual || !rstd || !dx || !dresidual || ((uintptr_t)rstd & 7u)) {
        set_error("nb200_gated_norm_bwd: null pointer, or rstd not 8-byte aligned");
        return NB200_ERR_ARG;
    }
    if ((dgate && !args->gate) || (dpost && !args->post_weight) || (dpre && !args->pre_weight) ||
        (grad_h && !args->pre_weight)) {
        set_error("nb200_gated_norm_bwd: a gradient of an input that is absent");
        return NB200_ERR_ARG;
    }
    if (!work || !aligned16(work) || work_bytes < norm_bwd_work_bytes(*args)) {
        set_error("nb200_gated_norm_bwd: work must hold %lld bytes, 16-byte aligned",
                  (long long)norm_bwd_work_bytes(*args));
        return NB200_ERR_ARG;
    }
    return launch_norm_bwd(*args, dtype, rstd, grad_y, grad_h, dx, dresidual, dgate, dpost, dpre,
                           static_cast<float*>(work), (cudaStream_t)stream);
}

int nb200_distill_loss(const nb200_distill_args* args, const float* teacher_lse, float* loss, float* stats,
                       void* stream) {
    const int rc = check_distill("nb200_distill_loss", args);
    if (rc) return rc;
    if (args->rows == 0) return NB200_OK;
    if (!args->x || (args->top && (!args->teacher || !args->index)) || !loss || !stats) {
        set_error("nb200_distill_loss: null pointer");
        return NB200_ERR_ARG;
    }
    return launch_distill_fwd(*args, teacher_lse, loss, stats, (cudaStream_t)stream);
}

int nb200_distill_loss_bwd(const nb200_distill_args* args, const float* grad, int64_t stride_grad, const float* stats,
                           void* dx, void* stream) {
    const int rc = check_distill("nb200_distill_loss_bwd", args);
    if (rc) return rc;
    if (args->rows == 0) return NB200_OK;
    if (!args->x || (args->top && (!args->teacher || !args->index)) || !grad || !stats || !dx || stride_grad < 0) {
        set_error("nb200_distill_loss_bwd: null pointer or negative stride");
        return NB200_ERR_ARG;
    }
    return launch_distill_bwd(*args, grad, stride_grad, stats, dx, (cudaStream_t)stream);
}

int64_t nb200_prefix_attention_work_bytes(const nb200_prefix_attn_args* args) {
    const nb200_attn_strides any = {8, 8, 8};
    const nb200_attn_strides strides[5] = {any, any, any, any, any};
    const int rc = check_prefix_attention("nb200_prefix_attention", args, strides);
    if (rc) return rc;
    return args->batch * args->heads * args->tokens ? prefix_attention_work_bytes(*args) : 0;
}

int nb200_prefix_attention(const nb200_prefix_attn_args* args, const nb200_attn_strides* strides, const void* q,
                           const void* prefix_k, const void* prefix_v, const void* k, const void* v, void* o, float* lse,
                           void* work, int64_t work_bytes, void* stream) {
    const char* what = "nb200_prefix_attention";
    const int rc = check_prefix_attention(what, args, strides);
    if (rc) return rc;
    if (args->batch * args->heads * args->tokens == 0) return NB200_OK;
    const void* tensors[6] = {q, o, prefix_k, prefix_v, k, v};
    for (int i = 0; i < 6; ++i) {
        if ((i == 2 || i == 3) ? args->prefix == 0 : i > 3 && args->cache == 0) continue;
        if (!tensors[i] || !aligned16(tensors[i])) {
            set_error("%s: null pointer, or a tensor is not 16-byte aligned", what);
            return NB200_ERR_ARG;
        }
    }
    if (((uintptr_t)lse | (uintptr_t)args->seq_lens) & 3u) {
        set_error("%s: lse and seq_lens must be 4-byte aligned", what);
        return NB200_ERR_ARG;
    }
    const int64_t need = prefix_attention_work_bytes(*args);
    if (need && (!work || !aligned16(work) || work_bytes < need)) {
        set_error("%s: work must hold %lld bytes, 16-byte aligned", what, (long long)need);
        return NB200_ERR_ARG;
    }
    return launch_prefix_attention(*args, strides, q, prefix_k, prefix_v, k, v, o, lse, work, (cudaStream_t)stream);
}

int nb200_norm8(const nb200_norm8_args* args, void* q, float* scale, void* y, void* stream) {
    const int rc = check_norm8("nb200_norm8", args);
    if (rc) return rc;
    if (args->rows == 0) return NB200_OK;
    if (!args->x || !args->weight || !q || !scale || (args->residual && !y)) {
        set_error("nb200_norm8: null pointer");
        return NB200_ERR_ARG;
    }
    const uintptr_t values = (uintptr_t)args->x | (uintptr_t)args->residual | (uintptr_t)args->weight |
                             (args->residual ? (uintptr_t)y : 0);
    if (values & (args->dtype == NB200_F32 ? 3u : 1u) || (uintptr_t)scale & 3u) {
        set_error("nb200_norm8: a tensor is not aligned to its elements");
        return NB200_ERR_ARG;
    }
    return launch_norm8(*args, q, scale, y, (cudaStream_t)stream);
}

int64_t nb200_penalize_logits_work_bytes(const nb200_logits_args* args) {
    const int rc = check_logits("nb200_penalize_logits", args);
    return rc ? rc : logits_work_bytes(*args);
}

int nb200_penalize_logits(const nb200_logits_args* args, void* out, void* work, int64_t work_bytes, void* stream) {
    const int rc = check_logits("nb200_penalize_logits", args);
    if (rc) return rc;
    if (args->rows == 0) return NB200_OK;
    if (!args->logits || !out || (args->history && !args->tokens) ||
        (args->biases && (!args->bias_index || !args->bias_value))) {
        set_error("nb200_penalize_logits: null pointer");
        return NB200_ERR_ARG;
    }
    uintptr_t words = (uintptr_t)args->token_lens | (uintptr_t)args->prompt_lens | (uintptr_t)args->allowed |
                      (uintptr_t)args->repetition | (uintptr_t)args->presence | (uintptr_t)args->frequency |
                      (uintptr_t)args->temperature;
    if (args->biases) words |= (uintptr_t)args->bias_value;
    auto off = [](const void* p, int32_t index) { return ((uintptr_t)p & (index == NB200_I64 ? 7u : 3u)) != 0; };
    if (((uintptr_t)args->logits | (uintptr_t)out) & (args->dtype == NB200_F32 ? 3u : 1u) || words & 3u ||
        (args->history && off(args->tokens, args->token_dtype)) || (args->biases && off(args->bias_index, args->bias_dtype))) {
        set_error("nb200_penalize_logits: a tensor is not aligned to its elements");
        return NB200_ERR_ARG;
    }
    // A named token's logit is read once more after its tile is written.
    const uintptr_t size = args->dtype == NB200_F32 ? 4 : 2, in = (uintptr_t)args->logits, to = (uintptr_t)out;
    if (in < to + (uintptr_t)(args->rows * args->vocab) * size &&
        to < in + (uintptr_t)((args->rows - 1) * args->stride_logits + args->vocab) * size) {
        set_error("nb200_penalize_logits: out must not overlap logits");
        return NB200_ERR_ARG;
    }
    const int64_t need = logits_work_bytes(*args);
    if (need < 0) return (int)need;
    if (need && (!work || !aligned16(work) || work_bytes < need)) {
        set_error("nb200_penalize_logits: work must hold %lld bytes, 16-byte aligned", (long long)need);
        return NB200_ERR_ARG;
    }
    return launch_logits(*args, out, work, (cudaStream_t)stream);
}

}  // extern "C"
