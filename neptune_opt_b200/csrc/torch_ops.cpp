// The region ops registered with the PyTorch dispatcher from C++ (namespace `nb200`), so that a
// graph holding them can be compiled by AOTInductor into a package whose calls reach the CUDA
// kernels without any Python: the package's generated code calls the op by name through the
// dispatcher, and this library -- loaded into the process that runs the package -- answers with a
// C++ kernel that calls the C ABI of libneptune_b200.so (include/neptune_b200.h).
//
// Ops (CUDA kernels + Meta kernels that compute shapes only, for export and fake tensors):
//   fold(Tensor x, int skeleton, float[] params, bool keepdim, int plan, int block,
//        int num_warps=0) -> Tensor
//       params = [tiny, alpha, T, beta, N, eps]; plan 0 serial, 1 split (block-column chunks);
//       serial launch from num_warps as the host launch policy maps (block, num_warps): 0 the
//       library's own choice, 1 one warp per row, 2..16 one CTA of 32 n threads per row, 32 one
//       thread-block cluster per row
//   softmax(Tensor x, int mode) -> (Tensor y, Tensor lse)           mode 0 softmax, 1 log_softmax
//   l2_normalize(Tensor x) -> (Tensor y, Tensor norm)
//   rms_norm(Tensor x, Tensor gamma, float eps) -> Tensor
//   segment_pool(Tensor data, Tensor segments, bool offsets, int reduce, float? initial,
//                bool unsafe) -> Tensor                              reduce 0 sum, 1 mean
//   segment_status(int device, bool clear) -> int
//   segment_status_word(int device) -> Tensor      the per-device int32 word itself, for launches
//                                                  made through the C ABI by other host code
//   attention(Tensor q, Tensor k, Tensor v, bool causal, float scale) -> (Tensor o, Tensor lse)
//                                                  (k and v may have fewer heads, a divisor of q's)
// The training operators (their CUDA kernels check the whole contract of the Python functions; an absent
// result is a tensor without elements, which graphs and packages can hold):
//   attention_fwd(Tensor q, Tensor k, Tensor v, Tensor? seq_lens, bool causal, float scale, bool with_lse)
//              -> (Tensor o, Tensor lse)
//   attention_bwd(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor grad_o, Tensor? seq_lens,
//                 bool causal, float scale) -> (Tensor dq, Tensor dk, Tensor dv)
//   gated_norm(Tensor x, Tensor residual, Tensor? gate, Tensor? post, Tensor? pre, int act, float scale,
//              float eps) -> (Tensor y, Tensor h, Tensor rstd)
//   gated_norm_bwd(Tensor? grad_y, Tensor? grad_h, Tensor x, Tensor residual, Tensor? gate, Tensor rstd,
//                  Tensor? post, Tensor? pre, int act, float scale, bool want_gate=True, bool want_post=True,
//                  bool want_pre=True)
//              -> (Tensor dx, Tensor dresidual, Tensor dgate, Tensor dpost, Tensor dpre)
//   distill_loss(Tensor x, Tensor teacher, Tensor index, float temperature, Tensor? teacher_lse)
//              -> (Tensor loss, Tensor stats)
//   distill_loss_bwd(Tensor grad, Tensor x, Tensor teacher, Tensor index, Tensor stats,
//                    float temperature) -> Tensor
// The serving operators (the same, but without a gradient: one that is asked for is refused):
//   prefix_attention(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor k, Tensor v, Tensor? seq_lens, float scale,
//                    bool with_lse) -> (Tensor o, Tensor lse)
//   norm8(Tensor x, Tensor weight, Tensor? residual, int group, int kind, float eps)
//              -> (Tensor q, Tensor scale, Tensor y)          kind 0 float8_e4m3fn, 1 float8_e5m2, 2 int8 (packages
//                                                            hand a dtype on by another number)
//   penalize_logits(Tensor logits, Tensor? tokens, Tensor? token_lens, Tensor? prompt_lens, Tensor? repetition,
//                   Tensor? presence, Tensor? frequency, Tensor? bias_index, Tensor? bias_value, Tensor? allowed,
//                   Tensor? temperature) -> Tensor
//
// libneptune_b200.so is opened at the first call from the directory this library lives in, so
// the two files only need to sit side by side.
#include <dlfcn.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/inductor/aoti_torch/utils.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <initializer_list>
#include <map>
#include <mutex>
#include <string>

#include "../../include/neptune_b200.h"

namespace {

struct Api {
    decltype(&nb200_last_error) last_error;
    decltype(&nb200_fold) fold;
    decltype(&nb200_fold_split_scratch_bytes) split_scratch_bytes;
    decltype(&nb200_fold_split) fold_split;
    decltype(&nb200_softmax) softmax;
    decltype(&nb200_l2_normalize) l2_normalize;
    decltype(&nb200_rms_norm) rms_norm;
    decltype(&nb200_segment_spans) segment_spans;
    decltype(&nb200_segment_pool) segment_pool;
    decltype(&nb200_attention_fwd) attention_fwd;
    decltype(&nb200_attention_bwd_work_bytes) attention_bwd_work_bytes;
    decltype(&nb200_attention_bwd) attention_bwd;
    decltype(&nb200_gated_norm) gated_norm;
    decltype(&nb200_gated_norm_bwd_work_bytes) gated_norm_bwd_work_bytes;
    decltype(&nb200_gated_norm_bwd) gated_norm_bwd;
    decltype(&nb200_distill_loss) distill_loss;
    decltype(&nb200_distill_loss_bwd) distill_loss_bwd;
    decltype(&nb200_prefix_attention_work_bytes) prefix_attention_work_bytes;
    decltype(&nb200_prefix_attention) prefix_attention;
    decltype(&nb200_norm8) norm8;
    decltype(&nb200_penalize_logits_work_bytes) penalize_logits_work_bytes;
    decltype(&nb200_penalize_logits) penalize_logits;
};

std::string own_directory() {
    Dl_info info;
    if (dladdr(reinterpret_cast<void*>(&own_directory), &info) && info.dli_fname) {
        std::string p(info.dli_fname);
        const auto slash = p.rfind('/');
        if (slash != std::string::npos) return p.substr(0, slash);
    }
    return ".";
}

template <typename F>
void bind(void* h, const char* name, F& f) {
    f = reinterpret_cast<F>(dlsym(h, name));
    TORCH_CHECK(f != nullptr, "nb200: libneptune_b200.so does not export ", name);
}

const Api& api() {
    static Api a;
    static std::once_flag once;
    std::call_once(once, [] {
        const std::string path = own_directory() + "/libneptune_b200.so";
        void* h = dlopen(path.c_str(), RTLD_NOW | RTLD_GLOBAL);
        TORCH_CHECK(h != nullptr, "nb200: cannot load ", path, ": ", dlerror());
        bind(h, "nb200_last_error", a.last_error);
        bind(h, "nb200_fold", a.fold);
        bind(h, "nb200_fold_split_scratch_bytes", a.split_scratch_bytes);
        bind(h, "nb200_fold_split", a.fold_split);
        bind(h, "nb200_softmax", a.softmax);
        bind(h, "nb200_l2_normalize", a.l2_normalize);
        bind(h, "nb200_rms_norm", a.rms_norm);
        bind(h, "nb200_segment_spans", a.segment_spans);
        bind(h, "nb200_segment_pool", a.segment_pool);
        bind(h, "nb200_attention_fwd", a.attention_fwd);
        bind(h, "nb200_attention_bwd_work_bytes", a.attention_bwd_work_bytes);
        bind(h, "nb200_attention_bwd", a.attention_bwd);
        bind(h, "nb200_gated_norm", a.gated_norm);
        bind(h, "nb200_gated_norm_bwd_work_bytes", a.gated_norm_bwd_work_bytes);
        bind(h, "nb200_gated_norm_bwd", a.gated_norm_bwd);
        bind(h, "nb200_distill_loss", a.distill_loss);
        bind(h, "nb200_distill_loss_bwd", a.distill_loss_bwd);
        bind(h, "nb200_prefix_attention_work_bytes", a.prefix_attention_work_bytes);
        bind(h, "nb200_prefix_attention", a.prefix_attention);
        bind(h, "nb200_norm8", a.norm8);
        bind(h, "nb200_penalize_logits_work_bytes", a.penalize_logits_work_bytes);
        bind(h, "nb200_penalize_logits", a.penalize_logits);
    });
    return a;
}

// Status codes to the exception types the Python layer raises for the same conditions.
void check(int rc, const char* what) {
    if (rc == NB200_OK) return;
    const char* msg = api().last_error();
    TORCH_CHECK_VALUE(rc != NB200_ERR_ARG, what, ": ", msg);
    TORCH_CHECK_NOT_IMPLEMENTED(rc != NB200_ERR_CAPACITY && rc != NB200_ERR_UNSUPPORTED, what, ": ", msg);
    TORCH_CHECK(false, what, ": ", msg);
}

int dtype_code(const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return NB200_F32;
        case at::kBFloat16: return NB200_BF16;
        case at::kHalf: return NB200_F16;
        default: TORCH_CHECK_TYPE(false, "nb200: dtype must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
    return -1;
}

void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// Rows of the last dimension: [..., n] viewed as [rows, n] (a copy only when no view exists).
at::Tensor rows_view(const at::Tensor& x) {
    TORCH_CHECK_VALUE(x.dim() >= 1, "nb200: input needs at least one dimension");
    TORCH_CHECK(x.size(-1) > 0, "nb200: the reduced width must be positive");
    return x.reshape({-1, x.size(-1)});
}

std::vector<int64_t> lead_shape(const at::Tensor& x, bool keepdim) {
    std::vector<int64_t> s(x.sizes().begin(), x.sizes().end() - 1);
    if (keepdim) s.push_back(1);
    return s;
}

nb200_params params_of(at::ArrayRef<double> p) {
    TORCH_CHECK_VALUE(p.size() == 6, "nb200.fold: params must be [tiny, alpha, T, beta, N, eps]");
    return nb200_params{p[0], p[1], p[2], p[3], p[4], p[5]};
}

void check_cuda(const at::Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.is_cuda(), what, ": inputs must be CUDA tensors, got ", t.device());
}

// ------------------------------------------------------------------ CUDA kernels
// The launch a (block, num_warps) pair selects for the serial plan (nullptr: library default).
const nb200_launch* serial_launch(int64_t num_warps, nb200_launch* storage) {
    if (num_warps <= 0) return nullptr;
    if (num_warps == 1) {
        *storage = nb200_launch{NB200_VARIANT_WARP_ROW, 0, 0, 0};
    } else if (num_warps == 32) {
        *storage = nb200_launch{NB200_VARIANT_CLUSTER, 0, 0, 0};
    } else {
        TORCH_CHECK_VALUE(num_warps <= 16, "nb200.fold: num_warps must be in 0..16 or 32, got ", num_warps);
        *storage = nb200_launch{NB200_VARIANT_CTA_ROW, (int32_t)(32 * num_warps), 0, 0};
    }
    return storage;
}

at::Tensor fold_cuda(const at::Tensor& x, int64_t skeleton, at::ArrayRef<double> params, bool keepdim, int64_t plan,
                     int64_t block, int64_t num_warps) {
    check_cuda(x, "nb200.fold");
    const int dt = dtype_code(x);
    c10::cuda::CUDAGuard guard(x.device());
    const nb200_params p = params_of(params);
    at::Tensor out = at::empty(lead_shape(x, keepdim), x.options());
    if (out.numel() == 0) return out;
    const at::Tensor x2 = rows_view(x);
    if (plan == 0) {
        nb200_launch storage;
        check(api().fold((int)skeleton, &p, x2.data_ptr(), dt, x2.size(0), x2.size(1), x2.stride(0), x2.stride(1),
                         out.data_ptr(), serial_launch(num_warps, &storage), stream_of(x)),
              "nb200.fold");
    } else {
        const int64_t chunk = block > 0 ? block : 16384;
        const int64_t nparts = (x2.size(1) + chunk - 1) / chunk;
        const int64_t bytes = api().split_scratch_bytes(x2.size(0), nparts);
        TORCH_CHECK_NOT_IMPLEMENTED(bytes >= 0, "nb200.fold: split plan capacity: ", api().last_error());
        at::Tensor scratch = at::empty({std::max<int64_t>(bytes, 1)}, x.options().dtype(at::kByte));
        check(api().fold_split((int)skeleton, &p, x2.data_ptr(), dt, x2.size(0), x2.size(1), x2.stride(0),
                               x2.stride(1), chunk, scratch.data_ptr(), bytes, out.data_ptr(), nullptr, stream_of(x)),
              "nb200.fold");
    }
    return out;
}

std::tuple<at::Tensor, at::Tensor> softmax_cuda(const at::Tensor& x, int64_t mode) {
    check_cuda(x, "nb200.softmax");
    const int dt = dtype_code(x);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor lse = at::empty(lead_shape(x, false), x.options());
    if (x.numel() == 0) return {y, lse};
    const at::Tensor x2 = rows_view(x);
    check(api().softmax((int)mode, x2.data_ptr(), dt, x2.size(0), x2.size(1), x2.stride(0), x2.stride(1),
                        y.data_ptr(), lse.data_ptr(), nullptr, stream_of(x)),
          "nb200.softmax");
    return {y, lse};
}

std::tuple<at::Tensor, at::Tensor> l2_cuda(const at::Tensor& x) {
    check_cuda(x, "nb200.l2_normalize");
    const int dt = dtype_code(x);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor norm = at::empty(lead_shape(x, false), x.options());
    if (x.numel() == 0) return {y, norm};
    const at::Tensor x2 = rows_view(x);
    check(api().l2_normalize(x2.data_ptr(), dt, x2.size(0), x2.size(1), x2.stride(0), x2.stride(1), y.data_ptr(),
                             norm.data_ptr(), nullptr, stream_of(x)),
          "nb200.l2_normalize");
    return {y, norm};
}

at::Tensor rms_cuda(const at::Tensor& x, const at::Tensor& gamma, double eps) {
    check_cuda(x, "nb200.rms_norm");
    check_cuda(gamma, "nb200.rms_norm");
    const int dt = dtype_code(x);
    TORCH_CHECK_TYPE(gamma.scalar_type() == x.scalar_type(), "nb200.rms_norm: gamma must have x's dtype");
    TORCH_CHECK_VALUE(gamma.dim() == 1 && x.dim() >= 1 && gamma.size(0) == x.size(-1),
                      "nb200.rms_norm: gamma must be 1-D with x's last dimension");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty(x.sizes(), x.options());
    if (x.numel() == 0) return y;
    const at::Tensor x2 = rows_view(x);
    check(api().rms_norm(x2.data_ptr(), gamma.data_ptr(), dt, x2.size(0), x2.size(1), x2.stride(0), x2.stride(1),
                         gamma.stride(0), eps, y.data_ptr(), nullptr, stream_of(x)),
          "nb200.rms_norm");
    return y;
}

// Per-device descriptor-status words of the C++ ops (same bits as the Python layer's:
// 1 negative or oversized length, 2 lengths not covering the rows, 4 boundary out of range,
// 8 boundaries decreasing). Malformed segments pool to NaN; the word records why.
std::mutex g_status_mutex;
std::map<int, at::Tensor> g_status;

at::Tensor status_word(const at::Device& dev) {
    std::lock_guard<std::mutex> lock(g_status_mutex);
    auto it = g_status.find(dev.index());
    if (it != g_status.end()) return it->second;
    at::Tensor w = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(dev));
    g_status.emplace(dev.index(), w);
    return w;
}

int index_code(const at::Tensor& t) {
    if (t.scalar_type() == at::kInt) return NB200_I32;
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong, "nb200.segment_pool: segments must be int32 or int64");
    return NB200_I64;
}

at::Tensor segment_cuda(const at::Tensor& data, const at::Tensor& segments, bool offsets, int64_t reduce,
                        std::optional<double> initial, bool unsafe) {
    check_cuda(data, "nb200.segment_pool");
    check_cuda(segments, "nb200.segment_pool");
    const int dt = dtype_code(data);
    const int idt = index_code(segments);
    TORCH_CHECK_VALUE(data.dim() >= 1 && segments.dim() == 1, "nb200.segment_pool: data [T, ...], segments 1-D");
    TORCH_CHECK_VALUE(reduce == 0 || reduce == 1, "nb200.segment_pool: reduce must be 0 (sum) or 1 (mean)");
    TORCH_CHECK_VALUE(!offsets || segments.size(0) >= 1, "nb200.segment_pool: offsets need at least one boundary");
    c10::cuda::CUDAGuard guard(data.device());
    const int64_t nseg = offsets ? segments.size(0) - 1 : segments.size(0);
    std::vector<int64_t> shape{nseg};
    int64_t channels = 1;
    for (int64_t d = 1; d < data.dim(); ++d) {
        shape.push_back(data.size(d));
        channels *= data.size(d);
    }
    at::Tensor out = at::empty(shape, data.options());
    if (nseg == 0 || channels == 0) return out;
    at::Tensor status = status_word(data.device());
    void* st = stream_of(data);
    at::Tensor bounds = segments;
    int bidx = idt;
    int64_t bstride = segments.numel() ? segments.stride(0) : 1;
    if (!offsets) {
        bounds = at::empty({nseg + 1}, segments.options().dtype(at::kLong));
        check(api().segment_spans(segments.data_ptr(), idt, nseg, bstride, unsafe ? 1 : 0, data.size(0),
                                  bounds.data_ptr<int64_t>(), reinterpret_cast<uint32_t*>(status.data_ptr()), st),
              "nb200.segment_pool");
        bidx = NB200_I64;
        bstride = 1;
    }
    const at::Tensor flat = data.reshape({data.size(0), channels});
    uint32_t bits = 0;
    if (initial.has_value()) {
        const float f = static_cast<float>(*initial);
        std::memcpy(&bits, &f, sizeof(bits));
    }
    check(api().segment_pool(flat.data_ptr(), dt, flat.size(0), channels, flat.stride(0), flat.stride(1),
                             bounds.data_ptr(), bidx, bstride, nseg, (int)reduce, initial.has_value() ? 1 : 0, bits,
                             out.data_ptr(), reinterpret_cast<uint32_t*>(status.data_ptr()), st),
          "nb200.segment_pool");
    return out;
}

at::Tensor segment_status_word(int64_t device) { return status_word(at::Device(at::kCUDA, (c10::DeviceIndex)device)); }

int64_t segment_status(int64_t device, bool clear) {
    at::Tensor w = status_word(at::Device(at::kCUDA, (c10::DeviceIndex)device));
    const int64_t bits = w.item<int32_t>();
    if (clear && bits) w.zero_();
    return bits;
}

// ------------------------------------------------------------------ attention and the training operators
using OptTensor = std::optional<at::Tensor>;

void check_strided(const at::Tensor& t, const char* what) {
    TORCH_CHECK_TYPE(t.layout() == at::kStrided, what, ": tensors must be strided");
}

bool present(const OptTensor& t) { return t.has_value() && t->defined(); }
// The result in the place of something absent.
at::Tensor none_like(const at::Tensor& x) { return at::empty({0}, x.options()); }

// Whether the attention kernels' copies can read rows of t's strides (unit stride in a row, positive 16-byte
// multiples between rows, heads and batch elements); symbolic sizes too.
bool rows_fit(const at::Tensor& t) {
    const auto sizes = t.sym_sizes(), strides = t.sym_strides();
    if (strides[3] != 1) return false;
    for (int i = 0; i < 3; ++i)
        if (sizes[i] > 1 && (strides[i] <= 0 || strides[i] % 8 != 0)) return false;
    return true;
}
// t itself when the copies can read its rows (16-byte aligned base), else a contiguous copy.
at::Tensor attn_rows(const at::Tensor& t) {
    const bool ok = rows_fit(t) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
// A gradient keeps the memory layout of its input.
at::Tensor attn_grad(const at::Tensor& t) {
    return rows_fit(t) ? at::empty_like(t) : at::empty_symint(t.sym_sizes(), t.options());
}

nb200_attn_strides attn_strides(const at::Tensor& t) { return {t.stride(0), t.stride(1), t.stride(2)}; }

// What the attention ops ask of q, k, v, symbolic sizes too: [batch, heads, seq, head_dim], k and v with a divisor of
// q's heads.
void check_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const char* what) {
    for (const at::Tensor* t : {&q, &k, &v}) {
        check_strided(*t, what);
        TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16, what, ": q, k, v must be bfloat16");
        TORCH_CHECK_VALUE(t->dim() == 4 && t->device() == q.device(), what, ": q, k, v must be 4-D on one device");
    }
    const auto qs = q.sym_sizes(), ks = k.sym_sizes();
    TORCH_CHECK_VALUE(ks == v.sym_sizes() && qs[0] == ks[0] && qs[2] == ks[2] && qs[3] == ks[3], what,
                      ": the shapes of q, k, v differ");
    TORCH_CHECK_VALUE(qs[1] == ks[1] || (ks[1] > 0 && qs[1] % ks[1] == 0), what, ": ", qs[1],
                      " query heads cannot share ", ks[1], " key/value heads");
}

void check_seq_lens(const OptTensor& seq_lens, const at::Tensor& q, const char* what) {
    if (!present(seq_lens)) return;
    TORCH_CHECK_TYPE(seq_lens->scalar_type() == at::kInt, what, ": seq_lens must be int32");
    TORCH_CHECK_VALUE(seq_lens->device() == q.device() && seq_lens->dim() == 1 && seq_lens->is_contiguous() &&
                          seq_lens->sym_size(0) == q.sym_size(0),
                      what, ": seq_lens must be contiguous [batch] on the device of q");
}

std::tuple<at::Tensor, at::Tensor> attention_fwd_cuda(const at::Tensor& q_, const at::Tensor& k_, const at::Tensor& v_,
                                                      const OptTensor& seq_lens, bool causal, double scale,
                                                      bool with_lse) {
    const char* what = "nb200.attention_fwd";
    check_cuda(q_, what);
    check_attention(q_, k_, v_, what);
    check_seq_lens(seq_lens, q_, what);
    c10::cuda::CUDAGuard guard(q_.device());
    const at::Tensor q = attn_rows(q_), k = attn_rows(k_), v = attn_rows(v_);
    at::Tensor o = at::empty(q.sizes(), q.options());
    const auto f32 = q.options().dtype(at::kFloat);
    at::Tensor lse = with_lse ? at::empty(q.sizes().slice(0, 3), f32) : at::empty({0}, f32);
    const nb200_attn_args a = {q.size(0), q.size(1), k.size(1), q.size(2), q.size(3),
                               present(seq_lens) ? seq_lens->data_ptr<int32_t>() : nullptr, causal ? 1 : 0, (float)scale};
    const nb200_attn_strides strides[4] = {attn_strides(q), attn_strides(k), attn_strides(v), attn_strides(o)};
    check(api().attention_fwd(&a, strides, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                              with_lse ? lse.data_ptr<float>() : nullptr, stream_of(q)),
          what);
    return {o, lse};
}
std::tuple<at::Tensor, at::Tensor> attention_cuda(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                  bool causal, double scale) {
    return attention_fwd_cuda(q, k, v, std::nullopt, causal, scale, true);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_bwd_cuda(const at::Tensor& q_, const at::Tensor& k_,
                                                                  const at::Tensor& v_, const at::Tensor& o_,
                                                                  const at::Tensor& lse_, const at::Tensor& go_,
                                                                  const OptTensor& seq_lens, bool causal,
                                                                  double scale) {
    const char* what = "nb200.attention_bwd";
    check_cuda(q_, what);
    check_attention(q_, k_, v_, what);
    for (const at::Tensor* t : {&o_, &go_}) {
        check_strided(*t, what);
        TORCH_CHECK_TYPE(t->scalar_type() == at::kBFloat16, what, ": o, grad_o must be bfloat16");
        TORCH_CHECK_VALUE(t->device() == q_.device() && t->sizes() == q_.sizes(), what,
                          ": o, grad_o must have the shape and device of q");
    }
    TORCH_CHECK_TYPE(lse_.scalar_type() == at::kFloat, what, ": lse must be float32");
    TORCH_CHECK_VALUE(lse_.device() == q_.device() && lse_.sizes() == q_.sizes().slice(0, 3), what,
                      ": lse must be [batch, heads, seq]");
    check_seq_lens(seq_lens, q_, what);
    c10::cuda::CUDAGuard guard(q_.device());
    const at::Tensor q = attn_rows(q_), k = attn_rows(k_), v = attn_rows(v_), o = attn_rows(o_), go = attn_rows(go_);
    const at::Tensor lse = lse_.contiguous();
    at::Tensor dq = attn_grad(q_), dk = attn_grad(k_), dv = attn_grad(v_);
    nb200_attn_args a = {q.size(0), q.size(1), k.size(1), q.size(2), q.size(3), nullptr, causal ? 1 : 0, (float)scale};
    if (present(seq_lens)) a.seq_lens = seq_lens->data_ptr<int32_t>();
    const nb200_attn_strides strides[8] = {attn_strides(q),  attn_strides(k),  attn_strides(v),  attn_strides(o),
                                           attn_strides(go), attn_strides(dq), attn_strides(dk), attn_strides(dv)};
    const int64_t bytes = api().attention_bwd_work_bytes(&a);
    if (bytes < 0) check((int)bytes, what);
    at::Tensor work = at::empty({std::max<int64_t>(bytes, 16)}, q.options().dtype(at::kByte));
    check(api().attention_bwd(&a, strides, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(),
                              lse.data_ptr<float>(), go.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(),
                              work.data_ptr(), work.numel(), stream_of(q)),
          what);
    return {dq, dk, dv};
}

// [rows, last] of t with unit column stride: a copy only when no such view exists.
at::Tensor unit_rows(const at::Tensor& t, int64_t rows) {
    at::Tensor f = t.dim() == 2 ? t : t.reshape({rows, t.size(-1)});
    return (f.stride(1) == 1 || f.size(1) == 1) && f.stride(0) >= 0 ? f : f.contiguous();
}

// Consecutive rows of x that share one row of the gate: all of them for a 1-D gate, otherwise those under the
// gate's trailing ones (its leading dimensions are x's).
int64_t rows_per_gate(const at::Tensor& x, const at::Tensor& gate, const char* what) {
    const int64_t lead = x.dim() - 1;
    int64_t n = 0, rows = 1;
    if (gate.dim() != 1) {
        TORCH_CHECK_VALUE(gate.dim() == x.dim(), what, ": gate does not broadcast over the rows of x");
        while (n < lead && gate.size(n) == x.size(n)) ++n;
        for (int64_t d = n; d < lead; ++d)
            TORCH_CHECK_VALUE(gate.size(d) == 1, what, ": gate does not broadcast over the rows of x");
    }
    for (int64_t d = n; d < lead; ++d) rows *= x.size(d);
    return rows;
}

// The descriptor of a gated norm's inputs and the tensors whose memory it names.
struct NormInputs {
    nb200_norm_args a = {};
    int dtype;
    int64_t rows;
    std::vector<at::Tensor> keep;
    static void same_kind(const at::Tensor& t, const at::Tensor& like, const char* what) {
        check_strided(t, what);
        TORCH_CHECK_TYPE(t.scalar_type() == like.scalar_type(), what, ": tensors must share one dtype");
        TORCH_CHECK_VALUE(t.device() == like.device(), what, ": tensors must be on one CUDA device");
    }
    const void* row_input(const at::Tensor& t, int64_t n, int64_t* stride) {
        if (t.is_contiguous()) {
            *stride = t.size(-1);
            return t.data_ptr();
        }
        keep.push_back(unit_rows(t, n));
        *stride = keep.back().stride(0);
        return keep.back().data_ptr();
    }
    const void* like_x(const at::Tensor& t, const at::Tensor& x, int64_t* stride, const char* what) {
        same_kind(t, x, what);
        TORCH_CHECK_VALUE(t.sizes() == x.sizes(), what, ": residual and gradients must have x's shape");
        return row_input(t, rows, stride);
    }
    const void* weight(const OptTensor& t, const at::Tensor& x, const char* what) {
        if (!present(t)) return nullptr;
        same_kind(*t, x, what);
        TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == x.size(-1), what,
                          ": weights must be 1-D with x's last dimension");
        if (t->is_contiguous()) return t->data_ptr();
        keep.push_back(t->contiguous());
        return keep.back().data_ptr();
    }
    NormInputs(const at::Tensor& x, const at::Tensor& residual, const OptTensor& gate, const OptTensor& post,
               const OptTensor& pre, int64_t act, double scale, double eps, const char* what) {
        check_strided(x, what);
        check_cuda(x, what);
        dtype = dtype_code(x);
        TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, what, ": x must be [..., width]");
        TORCH_CHECK_VALUE(present(post) || present(pre), what, ": neither weight is given");
        rows = x.numel() / x.size(-1);
        keep.reserve(7);
        a.rows = rows;
        a.width = x.size(-1);
        a.x = row_input(x, rows, &a.stride_x);
        a.residual = like_x(residual, x, &a.stride_residual, what);
        a.rows_per_gate = 1;
        if (present(gate)) {
            same_kind(*gate, x, what);
            TORCH_CHECK_VALUE(gate->dim() >= 1 && gate->size(-1) == x.size(-1), what, ": gate must be [..., width]");
            a.rows_per_gate = std::max<int64_t>(rows_per_gate(x, *gate, what), 1);  // x may have no rows
            a.gate = row_input(*gate, gate->numel() / gate->size(-1), &a.stride_gate);
        }
        a.post_weight = weight(post, x, what);
        a.pre_weight = weight(pre, x, what);
        a.gate_act = (int32_t)act;
        a.scale = scale;
        a.eps = eps;
    }
};

std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_norm_cuda(const at::Tensor& x, const at::Tensor& residual,
                                                               const OptTensor& gate, const OptTensor& post,
                                                               const OptTensor& pre, int64_t act, double scale,
                                                               double eps) {
    const char* what = "nb200.gated_norm";
    const NormInputs in(x, residual, gate, post, pre, act, scale, eps, what);
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor h = present(pre) ? at::empty(x.sizes(), x.options()) : none_like(x);
    std::vector<int64_t> shape = lead_shape(x, false);
    shape.push_back(2);
    at::Tensor rstd = at::empty(shape, x.options().dtype(at::kFloat));
    check(api().gated_norm(&in.a, in.dtype, y.data_ptr(), present(pre) ? h.data_ptr() : nullptr, rstd.data_ptr<float>(),
                           stream_of(x)),
          what);
    return {y, h, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> gated_norm_bwd_cuda(
    const OptTensor& gy, const OptTensor& gh, const at::Tensor& x, const at::Tensor& residual, const OptTensor& gate,
    const at::Tensor& rstd_, const OptTensor& post, const OptTensor& pre, int64_t act, double scale, bool want_gate,
    bool want_post, bool want_pre) {
    const char* what = "nb200.gated_norm_bwd";
    NormInputs in(x, residual, gate, post, pre, act, scale, 1.0, what);
    c10::cuda::CUDAGuard guard(x.device());
    TORCH_CHECK_TYPE(rstd_.scalar_type() == at::kFloat, what, ": rstd must be float32");
    TORCH_CHECK_VALUE(rstd_.device() == x.device() && rstd_.dim() == x.dim() && rstd_.size(-1) == 2 &&
                          rstd_.sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                      what, ": rstd must be [..., 2]");
    const bool whole = rstd_.is_contiguous() && reinterpret_cast<uintptr_t>(rstd_.data_ptr()) % 8 == 0;
    const at::Tensor rstd = whole ? rstd_ : rstd_.clone(at::MemoryFormat::Contiguous);
    const void* dy = present(gy) ? in.like_x(*gy, x, &in.a.stride_grad_y, what) : nullptr;
    const void* dh = present(gh) ? in.like_x(*gh, x, &in.a.stride_grad_h, what) : nullptr;
    auto fresh = [&](const OptTensor& t, bool want) {  // sums over no rows are zero
        if (!present(t) || !want) return none_like(x);
        return in.rows ? at::empty(t->sizes(), t->options()) : at::zeros(t->sizes(), t->options());
    };
    at::Tensor dx = at::empty(x.sizes(), x.options()), dr = at::empty(x.sizes(), x.options());
    at::Tensor dgate = fresh(gate, want_gate), dpost = fresh(post, want_post), dpre = fresh(pre, want_pre);
    auto ptr = [](const OptTensor& t, bool want, const at::Tensor& d) {
        return present(t) && want ? d.data_ptr() : nullptr;
    };
    const int64_t bytes = api().gated_norm_bwd_work_bytes(&in.a);
    if (bytes < 0) check((int)bytes, what);
    at::Tensor work = at::empty({std::max<int64_t>(bytes, 16)}, x.options().dtype(at::kByte));
    check(api().gated_norm_bwd(&in.a, in.dtype, rstd.data_ptr<float>(), dy, dh, dx.data_ptr(), dr.data_ptr(),
                               ptr(gate, want_gate, dgate), ptr(post, want_post, dpost), ptr(pre, want_pre, dpre), work.data_ptr(), work.numel(), stream_of(x)),
          what);
    return {dx, dr, dgate, dpost, dpre};
}

// The descriptor of a distillation loss's inputs and the tensors whose memory it names.
struct DistillInputs {
    nb200_distill_args a = {};
    at::Tensor x, teacher, index;
    DistillInputs(const at::Tensor& x_, const at::Tensor& teacher_, const at::Tensor& index_, double temperature,
                  const char* what) {
        for (const at::Tensor* t : {&x_, &teacher_, &index_}) check_strided(*t, what);
        check_cuda(x_, what);
        a.dtype = dtype_code(x_);
        a.teacher_dtype = dtype_code(teacher_);
        a.index_dtype = index_code(index_);
        TORCH_CHECK_VALUE(x_.dim() >= 1 && x_.size(-1) >= 1 && teacher_.sizes() == index_.sizes() &&
                              teacher_.dim() == x_.dim() &&
                              teacher_.sizes().slice(0, x_.dim() - 1) == x_.sizes().slice(0, x_.dim() - 1),
                          what, ": logits must be [..., vocab], teacher and index [..., top] over the same rows");
        TORCH_CHECK_VALUE(teacher_.device() == x_.device() && index_.device() == x_.device(), what,
                          ": tensors must be on one CUDA device");
        a.rows = x_.numel() / x_.size(-1);
        a.vocab = x_.size(-1);
        a.top = teacher_.size(-1);
        x = unit_rows(x_, a.rows);
        teacher = unit_rows(teacher_, a.rows);
        index = unit_rows(index_, a.rows);
        a.x = x.data_ptr();
        a.teacher = teacher.data_ptr();
        a.index = index.data_ptr();
        a.stride_x = x.stride(0);
        a.stride_teacher = teacher.stride(0);
        a.stride_index = index.stride(0);
        a.temperature = temperature;
    }
};

std::tuple<at::Tensor, at::Tensor> distill_loss_cuda(const at::Tensor& x, const at::Tensor& teacher,
                                                     const at::Tensor& index, double temperature,
                                                     const OptTensor& teacher_lse) {
    const char* what = "nb200.distill_loss";
    const DistillInputs in(x, teacher, index, temperature, what);
    c10::cuda::CUDAGuard guard(x.device());
    std::vector<int64_t> shape = lead_shape(x, false);
    const auto f32 = x.options().dtype(at::kFloat);
    at::Tensor loss = at::empty(shape, f32), z;
    shape.push_back(3);
    at::Tensor stats = at::empty(shape, f32);
    if (present(teacher_lse)) {
        TORCH_CHECK_TYPE(teacher_lse->scalar_type() == at::kFloat, what, ": teacher_lse must be float32");
        TORCH_CHECK_VALUE(teacher_lse->device() == x.device() && teacher_lse->sizes() == loss.sizes(), what,
                          ": teacher_lse must be [...] over the logits' rows");
        z = teacher_lse->contiguous();
    }
    check(api().distill_loss(&in.a, z.defined() ? z.data_ptr<float>() : nullptr, loss.data_ptr<float>(),
                             stats.data_ptr<float>(), stream_of(x)),
          what);
    return {loss, stats};
}

at::Tensor distill_loss_bwd_cuda(const at::Tensor& grad_, const at::Tensor& x, const at::Tensor& teacher,
                                 const at::Tensor& index, const at::Tensor& stats_, double temperature) {
    const char* what = "nb200.distill_loss_bwd";
    const DistillInputs in(x, teacher, index, temperature, what);
    c10::cuda::CUDAGuard guard(x.device());
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    TORCH_CHECK_TYPE(grad_.scalar_type() == at::kFloat && stats_.scalar_type() == at::kFloat, what,
                     ": grad and stats must be float32");
    TORCH_CHECK_VALUE(grad_.sizes() == lead && stats_.dim() == x.dim() && stats_.size(-1) == 3 &&
                          stats_.sizes().slice(0, x.dim() - 1) == lead && grad_.device() == x.device() &&
                          stats_.device() == x.device(),
                      what, ": grad must be [...], stats [..., 3] over the logits' rows");
    at::Tensor grad = grad_.reshape({-1});
    if (grad.stride(0) < 0) grad = grad.contiguous();
    const at::Tensor stats = stats_.contiguous();
    at::Tensor dx = at::empty(x.sizes(), x.options());
    check(api().distill_loss_bwd(&in.a, grad.data_ptr<float>(), grad.stride(0), stats.data_ptr<float>(), dx.data_ptr(),
                                 stream_of(x)),
          what);
    return dx;
}

// ------------------------------------------------------------------ the serving operators
// A contiguous tensor on x's device, without the dispatcher's way to it: single-token calls are bound by the host.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& x) {
    return at::detail::empty_cuda(sizes, dtype, x.device(), std::nullopt);
}

// What prefix_attention asks of its tensors, symbolic sizes too.
void check_prefix_attention(const at::Tensor& q, const at::Tensor& pk, const at::Tensor& pv, const at::Tensor& k,
                            const at::Tensor& v, const OptTensor& seq_lens, double scale, const char* what) {
    for (const at::Tensor* t : {&q, &pk, &pv, &k, &v}) {
        check_strided(*t, what);
        TORCH_CHECK_TYPE(t->scalar_type() == q.scalar_type() &&
                             (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf),
                         what, ": tensors must all be bfloat16 or all float16");
        TORCH_CHECK_VALUE(t->device() == q.device(), what, ": tensors must be on one device");
    }
    TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4 && pk.dim() == 3 && pv.dim() == 3, what,
                      ": q, k, v must be 4-D, prefix_k, prefix_v 3-D");
    const auto qs = q.sym_sizes(), ks = k.sym_sizes(), ps = pk.sym_sizes();
    TORCH_CHECK_VALUE(ks == v.sym_sizes() && ps == pv.sym_sizes() && qs[0] == ks[0] && qs[3] == ks[3] &&
                          qs[3] == ps[2] && ks[1] == ps[0],
                      what, ": the shapes differ");
    TORCH_CHECK_VALUE(qs[1] == ks[1] || (ks[1] > 0 && qs[1] % ks[1] == 0), what, ": ", qs[1],
                      " query heads cannot share ", ks[1], " key/value heads");
    check_seq_lens(seq_lens, q, what);
    TORCH_CHECK_VALUE(std::isfinite((float)scale) && (float)scale > 0.f, what, ": scale must be finite and positive");
    TORCH_CHECK_NOT_IMPLEMENTED(qs[3] == 64 || qs[3] == 128, what, ": head_dim ", qs[3],
                                " is not supported (the kernels are built for 64 and 128)");
}

// As attn_rows, for [kv_heads, prefix, head_dim].
at::Tensor prefix_rows(const at::Tensor& t) {
    bool ok = t.stride(2) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
    for (int i = 0; i < 2; ++i) ok = ok && (t.size(i) <= 1 || (t.stride(i) > 0 && t.stride(i) % 8 == 0));
    return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}

std::tuple<at::Tensor, at::Tensor> prefix_attention_cuda(const at::Tensor& q_, const at::Tensor& pk_,
                                                         const at::Tensor& pv_, const at::Tensor& k_,
                                                         const at::Tensor& v_, const OptTensor& seq_lens, double scale,
                                                         bool with_lse) {
    const char* what = "nb200.prefix_attention";
    check_cuda(q_, what);
    check_prefix_attention(q_, pk_, pv_, k_, v_, seq_lens, scale, what);
    c10::cuda::CUDAGuard guard(q_.device());
    const at::Tensor q = attn_rows(q_), k = attn_rows(k_), v = attn_rows(v_), pk = prefix_rows(pk_), pv = prefix_rows(pv_);
    at::Tensor o = fresh(q.sizes(), q.scalar_type(), q);
    at::Tensor lse = fresh(with_lse ? q.sizes().slice(0, 3) : at::IntArrayRef{0}, at::kFloat, q);
    const nb200_prefix_attn_args a = {q.size(0), q.size(1), k.size(1), q.size(2), q.size(3), pk.size(1), k.size(2),
                                      present(seq_lens) ? seq_lens->data_ptr<int32_t>() : nullptr, dtype_code(q),
                                      (float)scale};
    const nb200_attn_strides strides[5] = {attn_strides(q), {0, pk.stride(0), pk.stride(1)}, {0, pv.stride(0), pv.stride(1)},
                                           attn_strides(k), attn_strides(v)};
    const int64_t bytes = api().prefix_attention_work_bytes(&a);
    if (bytes < 0) check((int)bytes, what);
    at::Tensor work = fresh({std::max<int64_t>(bytes, 16)}, at::kByte, q);
    check(api().prefix_attention(&a, strides, q.data_ptr(), pk.data_ptr(), pv.data_ptr(), k.data_ptr(), v.data_ptr(),
                                 o.data_ptr(), with_lse ? lse.data_ptr<float>() : nullptr, work.data_ptr(), bytes,
                                 stream_of(q)),
          what);
    return {o, lse};
}

at::ScalarType byte_dtype(int64_t kind, const char* what) {
    TORCH_CHECK_TYPE(kind >= NB200_E4M3 && kind <= NB200_I8, what, ": dtype must be float8_e4m3fn, float8_e5m2 or int8");
    return kind == NB200_E4M3 ? at::kFloat8_e4m3fn : kind == NB200_E5M2 ? at::kFloat8_e5m2 : at::kChar;
}

// What norm8 asks of its arguments, symbolic sizes too.
void check_norm8(const at::Tensor& x, const at::Tensor& weight, const OptTensor& residual, int64_t group, double eps,
                 const char* what) {
    check_strided(x, what);
    dtype_code(x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.sym_size(-1) >= 1, what, ": x must be [..., width]");
    const c10::SymInt width = x.sym_size(-1);
    NormInputs::same_kind(weight, x, what);
    TORCH_CHECK_VALUE(weight.dim() == 1 && weight.sym_size(0) == width, what, ": weight must be 1-D with x's last dimension");
    if (present(residual)) {
        NormInputs::same_kind(*residual, x, what);
        TORCH_CHECK_VALUE(residual->sym_sizes() == x.sym_sizes(), what, ": residual must have x's shape");
    }
    TORCH_CHECK_VALUE(group == 0 || group == 16 || group == 32 || group == 64 || group == 128, what,
                      ": group must be 0, 16, 32, 64 or 128, got ", group);
    TORCH_CHECK_VALUE(group == 0 || width % group == 0, what, ": width ", width, " is not whole groups of ", group);
    TORCH_CHECK_VALUE(std::isfinite((float)eps) && (float)eps > 0.f, what, ": eps must be finite and positive in fp32");
    TORCH_CHECK_NOT_IMPLEMENTED(width <= 16384, what, ": width ", width, " exceeds 16384");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> norm8_cuda(const at::Tensor& x_, const at::Tensor& weight_,
                                                          const OptTensor& residual_, int64_t group, int64_t kind,
                                                          double eps) {
    const char* what = "nb200.norm8";
    const at::ScalarType dtype = byte_dtype(kind, what);
    check_cuda(x_, what);
    check_norm8(x_, weight_, residual_, group, eps, what);
    nb200_norm8_args a = {};
    a.dtype = dtype_code(x_);
    a.kind = (int32_t)kind;
    a.width = x_.size(-1);
    a.rows = x_.numel() / a.width;
    a.group = group;
    a.eps = eps;
    c10::cuda::CUDAGuard guard(x_.device());
    const at::Tensor x = unit_rows(x_, a.rows), weight = weight_.contiguous();
    at::Tensor residual, y;
    a.x = x.data_ptr();
    a.stride_x = x.stride(0);
    a.weight = weight.data_ptr();
    if (present(residual_)) {
        residual = unit_rows(*residual_, a.rows);
        a.residual = residual.data_ptr();
        a.stride_residual = residual.stride(0);
        y = fresh(x_.sizes(), x_.scalar_type(), x_);
    } else {
        y = fresh({0}, x_.scalar_type(), x_);
    }
    at::Tensor q = fresh(x_.sizes(), dtype, x_);
    std::vector<int64_t> shape = lead_shape(x_, false);
    shape.push_back(group ? a.width / group : 1);
    at::Tensor scale = fresh(shape, at::kFloat, x_);
    check(api().norm8(&a, q.data_ptr(), scale.data_ptr<float>(), a.residual ? y.data_ptr() : nullptr, stream_of(x_)),
          what);
    return {q, scale, y};
}

// A tensor beside the logits: of one of the types, with a row (dims 2) or a value (dims 1) for each of theirs.
void check_beside(const OptTensor& t, const char* name, int64_t dims, std::initializer_list<at::ScalarType> dtypes,
                  const at::Tensor& logits, const char* what) {
    if (!present(t)) return;
    check_strided(*t, what);
    TORCH_CHECK_TYPE(std::find(dtypes.begin(), dtypes.end(), t->scalar_type()) != dtypes.end(), what, ": ", name, " must be ",
                     *dtypes.begin(), dtypes.size() > 1 ? " or int64" : "", ", got ", t->scalar_type());
    TORCH_CHECK_VALUE(t->device() == logits.device() && t->dim() == dims && t->sym_size(0) == logits.sym_size(0), what, ": ",
                      name, dims == 1 ? " must be [rows]" : " must be [rows, ...]", " on the device of logits");
}

// What penalize_logits asks of its tensors, symbolic sizes too.
void check_logits(const at::Tensor& logits, const OptTensor& tokens, const OptTensor& token_lens,
                  const OptTensor& prompt_lens, const OptTensor& repetition, const OptTensor& presence,
                  const OptTensor& frequency, const OptTensor& bias_index, const OptTensor& bias_value,
                  const OptTensor& allowed, const OptTensor& temperature, const char* what) {
    check_strided(logits, what);
    dtype_code(logits);
    TORCH_CHECK_VALUE(logits.dim() == 2 && logits.sym_size(1) >= 1, what, ": logits must be [rows, vocab]");
    const auto beside = [&](const OptTensor& t, const char* name, int64_t dims, std::initializer_list<at::ScalarType> dtypes) {
        check_beside(t, name, dims, dtypes, logits, what);
    };
    beside(tokens, "tokens", 2, {at::kInt, at::kLong});
    beside(token_lens, "token_lens", 1, {at::kInt});
    beside(prompt_lens, "prompt_lens", 1, {at::kInt});
    beside(repetition, "repetition", 1, {at::kFloat});
    beside(presence, "presence", 1, {at::kFloat});
    beside(frequency, "frequency", 1, {at::kFloat});
    beside(temperature, "temperature", 1, {at::kFloat});
    beside(bias_index, "bias_index", 2, {at::kInt, at::kLong});
    beside(bias_value, "bias_value", 2, {at::kFloat});
    beside(allowed, "allowed", 2, {at::kInt});
    TORCH_CHECK_VALUE(present(tokens) || !(present(token_lens) || present(prompt_lens) || present(repetition) ||
                                           present(presence) || present(frequency)),
                      what, ": lengths or penalties without tokens");
    TORCH_CHECK_VALUE(present(bias_index) == present(bias_value), what, ": bias_index and bias_value go together");
    if (present(bias_index)) {
        TORCH_CHECK_VALUE(bias_index->sym_sizes() == bias_value->sym_sizes(), what, ": the shapes of the biases differ");
        TORCH_CHECK_NOT_IMPLEMENTED(bias_index->sym_size(1) <= 1024, what, ": ", bias_index->sym_size(1),
                                    " biases per row exceed 1024");
    }
    if (present(allowed)) {
        const c10::SymInt words = (logits.sym_size(1) + 31) / 32;
        TORCH_CHECK_VALUE(allowed->sym_size(1) == words, what, ": allowed must hold ", words, " words a row, got ",
                          allowed->sym_size(1));
    }
}

// The descriptor of the logits' inputs and the tensors whose memory it names.
struct LogitsInputs {
    nb200_logits_args a = {};
    std::vector<at::Tensor> keep;
    // A tensor with a row for each of the logits', or null.
    const void* rows_of(const OptTensor& t, int64_t* columns, int64_t* stride) {
        if (!present(t)) return nullptr;
        keep.push_back(unit_rows(*t, a.rows));
        *columns = t->size(1);
        *stride = keep.back().stride(0);
        return keep.back().data_ptr();
    }
    template <typename T>
    const T* per_row(const OptTensor& t) {
        if (!present(t)) return nullptr;
        if (t->is_contiguous()) return t->data_ptr<T>();
        keep.push_back(t->contiguous());
        return keep.back().data_ptr<T>();
    }
    explicit LogitsInputs(const at::Tensor& x) {
        a.dtype = dtype_code(x);
        a.rows = x.size(0);
        a.vocab = x.size(1);
        keep.reserve(16);
    }
};

at::Tensor penalize_logits_cuda(const at::Tensor& logits, const OptTensor& tokens, const OptTensor& token_lens,
                                const OptTensor& prompt_lens, const OptTensor& repetition, const OptTensor& presence,
                                const OptTensor& frequency, const OptTensor& bias_index, const OptTensor& bias_value,
                                const OptTensor& allowed, const OptTensor& temperature) {
    const char* what = "nb200.penalize_logits";
    check_cuda(logits, what);
    check_logits(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, bias_index, bias_value, allowed,
                 temperature, what);
    LogitsInputs in(logits);
    nb200_logits_args& a = in.a;
    c10::cuda::CUDAGuard guard(logits.device());
    int64_t columns = 0;
    a.logits = in.rows_of(logits, &columns, &a.stride_logits);
    if (present(tokens)) a.token_dtype = index_code(*tokens);
    a.tokens = in.rows_of(tokens, &a.history, &a.stride_tokens);
    a.token_lens = in.per_row<int32_t>(token_lens);
    a.prompt_lens = in.per_row<int32_t>(prompt_lens);
    a.repetition = in.per_row<float>(repetition);
    a.presence = in.per_row<float>(presence);
    a.frequency = in.per_row<float>(frequency);
    a.temperature = in.per_row<float>(temperature);
    if (present(bias_index)) a.bias_dtype = index_code(*bias_index);
    a.bias_index = in.rows_of(bias_index, &a.biases, &a.stride_bias_index);
    a.bias_value = static_cast<const float*>(in.rows_of(bias_value, &columns, &a.stride_bias_value));
    a.allowed = static_cast<const int32_t*>(in.rows_of(allowed, &columns, &a.stride_allowed));
    at::Tensor out = fresh(logits.sizes(), logits.scalar_type(), logits);
    const int64_t bytes = api().penalize_logits_work_bytes(&a);
    if (bytes < 0) check((int)bytes, what);
    at::Tensor work;
    if (bytes) work = fresh({bytes}, at::kByte, logits);
    check(api().penalize_logits(&a, out.data_ptr(), bytes ? work.data_ptr() : nullptr, bytes, stream_of(logits)), what);
    return out;
}

// ------------------------------------------------------------------ Meta kernels (shapes only)
// Symbolic sizes throughout, so graphs exported with dynamic dimensions trace through these ops.
std::vector<c10::SymInt> lead_sym_shape(const at::Tensor& x, bool keepdim) {
    const auto s = x.sym_sizes();
    std::vector<c10::SymInt> v(s.begin(), s.end() - 1);
    if (keepdim) v.emplace_back(1);
    return v;
}
at::Tensor fold_meta(const at::Tensor& x, int64_t, at::ArrayRef<double>, bool keepdim, int64_t, int64_t, int64_t) {
    return at::empty_symint(lead_sym_shape(x, keepdim), x.options());
}
std::tuple<at::Tensor, at::Tensor> softmax_meta(const at::Tensor& x, int64_t) {
    return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint(lead_sym_shape(x, false), x.options())};
}
std::tuple<at::Tensor, at::Tensor> l2_meta(const at::Tensor& x) {
    return {at::empty_symint(x.sym_sizes(), x.options()), at::empty_symint(lead_sym_shape(x, false), x.options())};
}
at::Tensor rms_meta(const at::Tensor& x, const at::Tensor&, double) {
    return at::empty_symint(x.sym_sizes(), x.options());
}
at::Tensor segment_meta(const at::Tensor& data, const at::Tensor& segments, bool offsets, int64_t,
                        std::optional<double>, bool) {
    std::vector<c10::SymInt> shape{offsets ? segments.sym_size(0) - 1 : segments.sym_size(0)};
    const auto ds = data.sym_sizes();
    for (size_t d = 1; d < ds.size(); ++d) shape.push_back(ds[d]);
    return at::empty_symint(shape, data.options());
}
std::tuple<at::Tensor, at::Tensor> attention_fwd_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                      const OptTensor& seq_lens, bool, double, bool with_lse) {
    check_attention(q, k, v, "nb200.attention_fwd");
    check_seq_lens(seq_lens, q, "nb200.attention_fwd");
    const auto qs = q.sym_sizes();
    const auto f32 = q.options().dtype(at::kFloat);
    return {at::empty_symint(qs, q.options()),
            with_lse ? at::empty_symint(std::vector<c10::SymInt>(qs.begin(), qs.end() - 1), f32) : at::empty({0}, f32)};
}
std::tuple<at::Tensor, at::Tensor> attention_meta(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                  bool causal, double scale) {
    return attention_fwd_meta(q, k, v, std::nullopt, causal, scale, true);
}
// Of the training operators: the Python functions check the contract before a graph is traced.
std::vector<c10::SymInt> lead_sym_shape_with(const at::Tensor& x, int64_t last) {
    std::vector<c10::SymInt> v = lead_sym_shape(x, false);
    v.emplace_back(last);
    return v;
}
at::Tensor like_meta(const at::Tensor& x) { return at::empty_symint(x.sym_sizes(), x.options()); }
at::Tensor like_meta(const OptTensor& t, const at::Tensor& x) { return present(t) ? like_meta(*t) : none_like(x); }
std::tuple<at::Tensor, at::Tensor, at::Tensor> attention_bwd_meta(const at::Tensor& q, const at::Tensor& k,
                                                                  const at::Tensor& v, const at::Tensor&,
                                                                  const at::Tensor&, const at::Tensor&,
                                                                  const OptTensor&, bool, double) {
    return {attn_grad(q), attn_grad(k), attn_grad(v)};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> gated_norm_meta(const at::Tensor& x, const at::Tensor&,
                                                               const OptTensor&, const OptTensor&,
                                                               const OptTensor& pre, int64_t, double, double) {
    return {like_meta(x), present(pre) ? like_meta(x) : none_like(x),
            at::empty_symint(lead_sym_shape_with(x, 2), x.options().dtype(at::kFloat))};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> gated_norm_bwd_meta(
    const OptTensor&, const OptTensor&, const at::Tensor& x, const at::Tensor&, const OptTensor& gate,
    const at::Tensor&, const OptTensor& post, const OptTensor& pre, int64_t, double, bool want_gate, bool want_post,
    bool want_pre) {
    return {like_meta(x), like_meta(x), want_gate ? like_meta(gate, x) : none_like(x),
            want_post ? like_meta(post, x) : none_like(x), want_pre ? like_meta(pre, x) : none_like(x)};
}
std::tuple<at::Tensor, at::Tensor> distill_loss_meta(const at::Tensor& x, const at::Tensor&, const at::Tensor&, double,
                                                     const OptTensor&) {
    const auto f32 = x.options().dtype(at::kFloat);
    return {at::empty_symint(lead_sym_shape(x, false), f32), at::empty_symint(lead_sym_shape_with(x, 3), f32)};
}
at::Tensor distill_loss_bwd_meta(const at::Tensor&, const at::Tensor& x, const at::Tensor&, const at::Tensor&,
                                 const at::Tensor&, double) {
    return like_meta(x);
}
std::tuple<at::Tensor, at::Tensor> prefix_attention_meta(const at::Tensor& q, const at::Tensor& pk,
                                                         const at::Tensor& pv, const at::Tensor& k,
                                                         const at::Tensor& v, const OptTensor& seq_lens, double scale,
                                                         bool with_lse) {
    check_prefix_attention(q, pk, pv, k, v, seq_lens, scale, "nb200.prefix_attention");
    const auto qs = q.sym_sizes();
    const auto f32 = q.options().dtype(at::kFloat);
    return {at::empty_symint(qs, q.options()),
            with_lse ? at::empty_symint(std::vector<c10::SymInt>(qs.begin(), qs.end() - 1), f32) : at::empty({0}, f32)};
}
std::tuple<at::Tensor, at::Tensor, at::Tensor> norm8_meta(const at::Tensor& x, const at::Tensor& weight,
                                                          const OptTensor& residual, int64_t group, int64_t kind,
                                                          double eps) {
    check_norm8(x, weight, residual, group, eps, "nb200.norm8");
    std::vector<c10::SymInt> shape = lead_sym_shape(x, false);
    shape.emplace_back(group > 0 ? x.sym_size(-1) / group : c10::SymInt(1));
    return {at::empty_symint(x.sym_sizes(), x.options().dtype(byte_dtype(kind, "nb200.norm8"))),
            at::empty_symint(shape, x.options().dtype(at::kFloat)),
            present(residual) ? like_meta(x) : none_like(x)};
}
at::Tensor penalize_logits_meta(const at::Tensor& logits, const OptTensor& tokens, const OptTensor& token_lens,
                                const OptTensor& prompt_lens, const OptTensor& repetition, const OptTensor& presence,
                                const OptTensor& frequency, const OptTensor& bias_index, const OptTensor& bias_value,
                                const OptTensor& allowed, const OptTensor& temperature) {
    check_logits(logits, tokens, token_lens, prompt_lens, repetition, presence, frequency, bias_index, bias_value, allowed,
                 temperature, "nb200.penalize_logits");
    return like_meta(logits);
}

}  // namespace

// ------------------------------------------------------------------ AOTInductor C shims
// Direct C entry points for AOTInductor packages (torch._inductor.config.aot_inductor.
// custom_ops_to_c_shims): a package compiled with them calls these functions instead of going
// through the proxy executor's boxed dispatcher call, which costs microseconds per region call.
// Argument conventions are AOTInductor's generated C shims': tensors as AtenTensorHandle, int as
// int64_t, bool as int32_t, float as double, float? as double* (nullptr = None), float[] as pointer
// + length, results as AtenTensorHandle* out-parameters. The process that runs such a package
// must make these symbols visible (load this library with RTLD_GLOBAL, as aot.load() does).
namespace {
at::Tensor& tensor_of(AtenTensorHandle h) { return *torch::aot_inductor::tensor_handle_to_tensor_pointer(h); }
}  // namespace

extern "C" {
AOTITorchError aoti_torch_cuda_fold(AtenTensorHandle x, int64_t skeleton, const double* params, int64_t params_len_,
                                    int32_t keepdim, int64_t plan, int64_t block, int64_t num_warps,
                                    AtenTensorHandle* ret0) {
    AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
        *ret0 = torch::aot_inductor::new_tensor_handle(fold_cuda(tensor_of(x), skeleton,
                                                                 at::ArrayRef<double>(params, params_len_),
                                                                 keepdim != 0, plan, block, num_warps));
    });
}
AOTITorchError aoti_torch_cuda_softmax(AtenTensorHandle x, int64_t mode, AtenTensorHandle* ret0,
                                       AtenTensorHandle* ret1) {
    AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
        auto r = softmax_cuda(tensor_of(x), mode);
        *ret0 = torch::aot_inductor::new_tensor_handle(std::move(std::get<0>(r)));
        *ret1 = torch::aot_inductor::new_tensor_handle(std::move(std::get<1>(r)));
    });
}
AOTITorchError aoti_torch_cuda_l2_normalize(AtenTensorHandle x, AtenTensorHandle* ret0, AtenTensorHandle* ret1) {
    AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
        auto r = l2_cuda(tensor_of(x));
        *ret0 = torch::aot_inductor::new_tensor_handle(std::move(std::get<0>(r)));
        *ret1 = torch::aot_inductor::new_tensor_handle(std::move(std::get<1>(r)));
    });
}
AOTITorchError aoti_torch_cuda_rms_norm(AtenTensorHandle x, AtenTensorHandle gamma, double eps,
                                        AtenTensorHandle* ret0) {
    AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
        *ret0 = torch::aot_inductor::new_tensor_handle(rms_cuda(tensor_of(x), tensor_of(gamma), eps));
    });
}
AOTITorchError aoti_torch_cuda_segment_pool(AtenTensorHandle data, AtenTensorHandle segments, int32_t offsets,
                                            int64_t reduce, double* initial, int32_t unsafe, AtenTensorHandle* ret0) {
    AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
        const std::optional<double> init = initial ? std::optional<double>(*initial) : std::nullopt;
        *ret0 = torch::aot_inductor::new_tensor_handle(
            segment_cuda(tensor_of(data), tensor_of(segments), offsets != 0, reduce, init, unsafe != 0));
    });
}
AOTITorchError aoti_torch_cuda_attention(AtenTensorHandle q, AtenTensorHandle k, AtenTensorHandle v, int32_t causal,
                                         double scale, AtenTensorHandle* ret0, AtenTensorHandle* ret1) {
    AOTI_TORCH_CONVERT_EXCEPTION_TO_ERROR_CODE({
        auto r = attention_cuda(tensor_of(q), tensor_of(k), tensor_of(v), causal != 0, scale);
        *ret0 = torch::aot_inductor::new_tensor_handle(std::move(std::get<0>(r)));
        *ret1 = torch::aot_inductor::new_tensor_handle(std::move(std::get<1>(r)));
    });
}
}  // extern "C"

TORCH_LIBRARY(nb200, m) {
    m.def("fold(Tensor x, int skeleton, float[] params, bool keepdim, int plan, int block, int num_warps=0) -> Tensor");
    m.def("softmax(Tensor x, int mode) -> (Tensor, Tensor)");
    m.def("l2_normalize(Tensor x) -> (Tensor, Tensor)");
    m.def("rms_norm(Tensor x, Tensor gamma, float eps) -> Tensor");
    m.def("segment_pool(Tensor data, Tensor segments, bool offsets, int reduce, float? initial, bool unsafe) -> Tensor");
    m.def("segment_status(int device, bool clear) -> int", &segment_status);
    m.def("segment_status_word(int device) -> Tensor", &segment_status_word);
    m.def("attention(Tensor q, Tensor k, Tensor v, bool causal, float scale) -> (Tensor, Tensor)");
    m.def("attention_fwd(Tensor q, Tensor k, Tensor v, Tensor? seq_lens, bool causal, float scale, bool with_lse) "
          "-> (Tensor, Tensor)");
    m.def("attention_bwd(Tensor q, Tensor k, Tensor v, Tensor o, Tensor lse, Tensor grad_o, Tensor? seq_lens, "
          "bool causal, float scale) -> (Tensor, Tensor, Tensor)");
    m.def("gated_norm(Tensor x, Tensor residual, Tensor? gate, Tensor? post, Tensor? pre, int act, "
          "float scale, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("gated_norm_bwd(Tensor? grad_y, Tensor? grad_h, Tensor x, Tensor residual, Tensor? gate, Tensor rstd, "
          "Tensor? post, Tensor? pre, int act, float scale, bool want_gate=True, bool want_post=True, "
          "bool want_pre=True) "
          "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
    m.def("distill_loss(Tensor x, Tensor teacher, Tensor index, float temperature, Tensor? teacher_lse) "
          "-> (Tensor, Tensor)");
    m.def("distill_loss_bwd(Tensor grad, Tensor x, Tensor teacher, Tensor index, Tensor stats, float temperature) "
          "-> Tensor");
    m.def("prefix_attention(Tensor q, Tensor prefix_k, Tensor prefix_v, Tensor k, Tensor v, Tensor? seq_lens, "
          "float scale, bool with_lse) -> (Tensor, Tensor)");
    m.def("norm8(Tensor x, Tensor weight, Tensor? residual, int group, int kind, float eps) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("penalize_logits(Tensor logits, Tensor? tokens, Tensor? token_lens, Tensor? prompt_lens, "
          "Tensor? repetition, Tensor? presence, Tensor? frequency, Tensor? bias_index, Tensor? bias_value, "
          "Tensor? allowed, Tensor? temperature) -> Tensor");
}

// The training operators are their own gradients' building blocks: autograd records nothing for them (the
// Python layer's autograd functions call them). A tangent of forward mode would be lost that way: it is refused.
static void below_autograd(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
    for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size()))
        TORCH_CHECK_NOT_IMPLEMENTED(!v.isTensor() || !torch::autograd::isFwGradDefined(v.toTensor()),
                                    op.schema().name(), " has no forward-mode derivative");
    at::AutoDispatchBelowADInplaceOrView guard;
    op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
}
// The serving operators have no gradient; one that autograd would have to record is refused, not dropped.
static void without_gradient(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
    for (const c10::IValue& v : torch::jit::last(*stack, op.schema().arguments().size()))
        TORCH_CHECK_NOT_IMPLEMENTED(!v.isTensor() || !(at::GradMode::is_enabled() && v.toTensor().requires_grad()),
                                    op.schema().name(), " has no gradient: call it under torch.no_grad()");
    below_autograd(op, keys, stack);
}
TORCH_LIBRARY_IMPL(nb200, Autograd, m) {
    for (const char* op : {"prefix_attention", "norm8", "penalize_logits"})
        m.impl(op, torch::CppFunction::makeFromBoxedFunction<&without_gradient>());
    for (const char* op : {"attention_fwd", "attention_bwd", "gated_norm", "gated_norm_bwd", "distill_loss",
                           "distill_loss_bwd"})
        m.impl(op, torch::CppFunction::makeFromBoxedFunction<&below_autograd>());
}

TORCH_LIBRARY_IMPL(nb200, CUDA, m) {
    m.impl("fold", &fold_cuda);
    m.impl("softmax", &softmax_cuda);
    m.impl("l2_normalize", &l2_cuda);
    m.impl("rms_norm", &rms_cuda);
    m.impl("segment_pool", &segment_cuda);
    m.impl("attention", &attention_cuda);
    m.impl("attention_fwd", &attention_fwd_cuda);
    m.impl("attention_bwd", &attention_bwd_cuda);
    m.impl("gated_norm", &gated_norm_cuda);
    m.impl("gated_norm_bwd", &gated_norm_bwd_cuda);
    m.impl("distill_loss", &distill_loss_cuda);
    m.impl("distill_loss_bwd", &distill_loss_bwd_cuda);
    m.impl("prefix_attention", &prefix_attention_cuda);
    m.impl("norm8", &norm8_cuda);
    m.impl("penalize_logits", &penalize_logits_cuda);
}

TORCH_LIBRARY_IMPL(nb200, Meta, m) {
    m.impl("fold", &fold_meta);
    m.impl("softmax", &softmax_meta);
    m.impl("l2_normalize", &l2_meta);
    m.impl("rms_norm", &rms_meta);
    m.impl("segment_pool", &segment_meta);
    m.impl("attention", &attention_meta);
    m.impl("attention_fwd", &attention_fwd_meta);
    m.impl("attention_bwd", &attention_bwd_meta);
    m.impl("gated_norm", &gated_norm_meta);
    m.impl("gated_norm_bwd", &gated_norm_bwd_meta);
    m.impl("distill_loss", &distill_loss_meta);
    m.impl("distill_loss_bwd", &distill_loss_bwd_meta);
    m.impl("prefix_attention", &prefix_attention_meta);
    m.impl("norm8", &norm8_meta);
    m.impl("penalize_logits", &penalize_logits_meta);
}
