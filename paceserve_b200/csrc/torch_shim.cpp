// Thin torch extension over the C ABI (include/pace_b200.h).  It recreates
// the reference's four pybind modules with their exact signatures
// (csrc/layernorm.cpp:3-14, csrc/pos_encoding.cpp:3-16,
// csrc/activation.cpp:3-28, csrc/moe.cpp:3-28) as submodules
// layernorm_ops / pos_encoding_ops / activation_ops / moe_ops of
// paceserve_b200._C, adds the new ops (fused_add_rms_norm, gelu_and_mul,
// gelu_tanh_and_mul) in the same style, a kv_transfer_ops submodule for the
// paged-KV block copy, append, quantised cache and step tables, an attention_ops
// submodule for paged attention and an int8_ops submodule for 8-bit projections.
// Tensors are validated here; every launch goes through the C ABI on the current
// stream of the tensors' device, and a non-zero status becomes a RuntimeError
// carrying pace_last_error().
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAEvent.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <map>
#include <mutex>
#include <string>
#include <vector>

#include "pace_b200.h"

namespace {

using torch::Tensor;

int pace_dtype(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PACE_F32;
    case at::kHalf: return PACE_F16;
    case at::kBFloat16: return PACE_BF16;
    case at::kByte: return PACE_U8;
    case at::kChar: return PACE_I8;
    case at::kShort: return PACE_I16;
    case at::kInt: return PACE_I32;
    case at::kLong: return PACE_I64;
    default: return -1;
  }
}

void check_status(int rc, const char* op) {
  TORCH_CHECK(rc == PACE_OK, op, " failed (", pace_status_string(rc), "): ", pace_last_error());
}

cudaStream_t stream_of(const Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

void check_cuda(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor");
}

void check_same_device(const Tensor& a, const Tensor& b, const char* op) {
  TORCH_CHECK(a.device() == b.device(), op, ": tensors on different devices (", a.device(), " vs ",
              b.device(), ")");
}

// Device pointer of an optional int32 counter the kernel adds to, or null.  It
// must live on the launching device: a host pointer would reach the kernel.
int32_t* counter_ptr(const c10::optional<Tensor>& t, const at::Device& dev, const char* op,
                     const char* name) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->is_cuda() && t->device() == dev && t->scalar_type() == at::kInt &&
                  t->numel() >= 1,
              op, ": ", name, " must be an int32 tensor with at least one element on ", dev);
  return t->data_ptr<int32_t>();
}

bool is_float_type(const Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf ||
         t.scalar_type() == at::kBFloat16;
}

// Row view of a tensor whose last dimension is contiguous: (rows, width,
// row_stride).  2-D tensors may have any row stride; higher ranks must be
// collapsible into rows with a single stride.
struct Rows {
  int64_t rows, width, stride;
};

Rows rows_of(const Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.dim() >= 1, op, ": ", name, " must have at least one dimension");
  const int64_t w = t.size(-1);
  TORCH_CHECK(t.numel() == 0 || w == 1 || t.stride(-1) == 1, op, ": ", name,
              " must be contiguous in its last dimension");
  if (t.dim() == 1) return {1, w, w};
  if (t.dim() == 2) return {t.size(0), w, t.size(0) <= 1 ? w : t.stride(0)};
  TORCH_CHECK(t.is_contiguous(), op, ": ", name, " of rank > 2 must be contiguous");
  return {w == 0 ? 0 : t.numel() / w, w, w};
}

// ------------------------------------------------------------- layernorm --
void rms_norm(Tensor& out, Tensor& input, Tensor& weight, double epsilon) {
  const char* op = "rms_norm";
  check_cuda(input, op, "input");
  check_same_device(out, input, op);
  check_same_device(weight, input, op);
  TORCH_CHECK(is_float_type(input), op, ": input dtype must be float32, float16 or bfloat16");
  TORCH_CHECK(out.scalar_type() == input.scalar_type() && weight.scalar_type() == input.scalar_type(),
              op, ": out, input and weight must share a dtype");
  const Rows in = rows_of(input, op, "input");
  const Rows o = rows_of(out, op, "out");
  TORCH_CHECK(o.rows == in.rows && o.width == in.width, op, ": out shape ", out.sizes(),
              " does not match input ", input.sizes());
  TORCH_CHECK(weight.is_contiguous() && weight.numel() == in.width, op, ": weight must be [",
              in.width, "] and contiguous");
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_rms_norm(out.data_ptr(), input.data_ptr(), weight.data_ptr(), (float)epsilon,
                             in.rows, in.width, in.stride, o.stride, pace_dtype(input),
                             stream_of(input)),
               op);
}

void fused_add_rms_norm(Tensor& input, Tensor& residual, Tensor& weight, double epsilon) {
  const char* op = "fused_add_rms_norm";
  check_cuda(input, op, "input");
  check_same_device(residual, input, op);
  check_same_device(weight, input, op);
  TORCH_CHECK(is_float_type(input), op, ": input dtype must be float32, float16 or bfloat16");
  TORCH_CHECK(residual.scalar_type() == input.scalar_type() &&
                  weight.scalar_type() == input.scalar_type(),
              op, ": input, residual and weight must share a dtype");
  const Rows in = rows_of(input, op, "input");
  const Rows r = rows_of(residual, op, "residual");
  TORCH_CHECK(r.rows == in.rows && r.width == in.width, op, ": residual shape ", residual.sizes(),
              " does not match input ", input.sizes());
  TORCH_CHECK(weight.is_contiguous() && weight.numel() == in.width, op, ": weight must be [",
              in.width, "] and contiguous");
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_fused_add_rms_norm(input.data_ptr(), residual.data_ptr(), weight.data_ptr(),
                                       (float)epsilon, in.rows, in.width, in.stride, r.stride,
                                       pace_dtype(input), stream_of(input)),
               op);
}

// ---------------------------------------------------------- pos encoding --
// q/k as [T, heads * head_size] (any row stride) or [T, heads, head_size].
Rows qk_rows(const Tensor& t, int64_t head_size, const char* op, const char* name) {
  TORCH_CHECK(t.dim() == 2 || t.dim() == 3, op, ": ", name, " must be 2-D or 3-D");
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, op, ": ", name,
              " must be contiguous in its last dimension");
  if (t.dim() == 3) {
    TORCH_CHECK(t.size(2) == head_size, op, ": ", name, " last dim must equal head_size");
    TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == head_size, op, ": ", name,
                " heads must be contiguous");
    return {t.size(0), t.size(1) * head_size, t.size(0) <= 1 ? t.size(1) * head_size : t.stride(0)};
  }
  TORCH_CHECK(t.size(1) % head_size == 0, op, ": ", name, " width ", t.size(1),
              " is not a multiple of head_size ", head_size);
  return {t.size(0), t.size(1), t.size(0) <= 1 ? t.size(1) : t.stride(0)};
}

void rotary_embedding(Tensor& positions, Tensor& query, Tensor& key, int64_t head_size,
                      Tensor& cos_sin_cache, bool is_neox) {
  const char* op = "rotary_embedding";
  check_cuda(query, op, "query");
  check_same_device(positions, query, op);
  check_same_device(key, query, op);
  check_same_device(cos_sin_cache, query, op);
  TORCH_CHECK(head_size > 0, op, ": head_size must be positive");
  TORCH_CHECK(is_float_type(query) && key.scalar_type() == query.scalar_type(), op,
              ": query and key must share a float dtype");
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.is_contiguous(), op,
              ": positions must be a contiguous int64 tensor");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), op,
              ": cos_sin_cache must be a contiguous [max_position, rot_dim] tensor");
  TORCH_CHECK(cos_sin_cache.scalar_type() == at::kFloat ||
                  cos_sin_cache.scalar_type() == query.scalar_type(),
              op, ": cos_sin_cache must be float32 or the query dtype");
  const Rows q = qk_rows(query, head_size, op, "query");
  const Rows k = qk_rows(key, head_size, op, "key");
  TORCH_CHECK(k.rows == q.rows, op, ": query and key token counts differ");
  TORCH_CHECK(positions.numel() >= q.rows, op, ": positions has ", positions.numel(),
              " entries for ", q.rows, " tokens");
  const at::cuda::CUDAGuard guard(query.device());
  check_status(pace_rotary_embedding(
                   positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(), q.rows,
                   (int)(q.width / head_size), (int)(k.width / head_size), (int)head_size,
                   q.stride, k.stride, cos_sin_cache.data_ptr(), pace_dtype(cos_sin_cache),
                   (int)cos_sin_cache.size(1), cos_sin_cache.size(0), is_neox ? 1 : 0,
                   pace_dtype(query), stream_of(query)),
               op);
}

// qkv = hidden @ weight^T with the rotary embedding of the q and k heads
// applied before the output is rounded (tcgen05 GEMM + rope epilogue).  It
// replaces qkv_proj followed by rotary_embedding
// (paceserve/model_executor/models/llama.py:176-178); `qkv` is the [T, (nq +
// 2 nkv) * head_size] output the split into q, k, v views reads.
// The stream-K workspace of the fused projection, kept per (device, stream):
// zero-filled once on that stream, and left zeroed by every call, so calls on
// one stream can share it; calls on different streams never do.
Tensor qkv_workspace(const at::Device& dev, cudaStream_t stream, size_t bytes) {
  static std::mutex mu;
  static std::map<std::pair<int, cudaStream_t>, Tensor> cache;
  std::lock_guard<std::mutex> lock(mu);
  Tensor& ws = cache[{dev.index(), stream}];
  if (!ws.defined() || (size_t)ws.numel() < bytes)
    ws = at::zeros({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(dev));
  return ws;
}

// A workspace tensor as the C ABI takes it (an undefined tensor: none).
void* ws_ptr(const Tensor& ws) { return ws.defined() ? ws.data_ptr() : nullptr; }
size_t ws_bytes(const Tensor& ws) { return ws.defined() ? (size_t)ws.nbytes() : 0; }

void qkv_proj_rotary_embedding(Tensor& qkv, Tensor& hidden, Tensor& weight, Tensor& positions,
                               int64_t head_size, int64_t num_heads, int64_t num_kv_heads,
                               Tensor& cos_sin_cache, bool is_neox,
                               const c10::optional<Tensor>& fault_flags,
                               const c10::optional<Tensor>& workspace) {
  const char* op = "qkv_proj_rotary_embedding";
  check_cuda(hidden, op, "hidden");
  check_same_device(qkv, hidden, op);
  check_same_device(weight, hidden, op);
  check_same_device(positions, hidden, op);
  check_same_device(cos_sin_cache, hidden, op);
  TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf, op,
              ": hidden must be bfloat16 or float16");
  TORCH_CHECK(qkv.scalar_type() == hidden.scalar_type() &&
                  weight.scalar_type() == hidden.scalar_type(),
              op, ": qkv, hidden and weight must share a dtype");
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.is_contiguous(), op,
              ": positions must be a contiguous int64 tensor");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), op,
              ": cos_sin_cache must be a contiguous [max_position, rot_dim] tensor");
  TORCH_CHECK(num_heads >= 0 && num_kv_heads >= 0 && head_size > 0, op, ": bad head counts");
  const Rows h = rows_of(hidden, op, "hidden");
  TORCH_CHECK(hidden.dim() == 2, op, ": hidden must be [T, hidden_size]");
  TORCH_CHECK(qkv.dim() == 2 && qkv.size(0) == h.rows, op, ": qkv must be [T, ",
              (num_heads + 2 * num_kv_heads) * head_size, "]");
  const Rows o = rows_of(qkv, op, "qkv");
  const int64_t n = (num_heads + 2 * num_kv_heads) * head_size;
  TORCH_CHECK(o.width == n, op, ": qkv width ", o.width, " != (num_heads + 2 * num_kv_heads) * head_size = ", n);
  TORCH_CHECK(weight.dim() == 2 && weight.is_contiguous() && weight.size(0) == n &&
                  weight.size(1) == h.width,
              op, ": weight must be a contiguous [", n, ", ", h.width, "] tensor");
  TORCH_CHECK(positions.numel() >= h.rows, op, ": positions has ", positions.numel(),
              " entries for ", h.rows, " tokens");
  const at::cuda::CUDAGuard guard(hidden.device());
  int32_t* fault = counter_ptr(fault_flags, hidden.device(), op, "fault_flags");
  if (h.rows == 0) return;
  const cudaStream_t stream = stream_of(hidden);
  const size_t need = pace_qkv_proj_rope_workspace_size(h.rows, h.width, (int)num_heads,
                                                        (int)num_kv_heads, hidden.device().index());
  Tensor ws;
  if (workspace.has_value()) {
    ws = *workspace;
    TORCH_CHECK(ws.is_cuda() && ws.device() == hidden.device() && ws.is_contiguous() &&
                    (size_t)ws.nbytes() >= need,
                op, ": workspace must be a contiguous tensor of at least ", need, " bytes on ",
                hidden.device());
  } else if (need > 0) {  // none at decode sizes
    ws = qkv_workspace(hidden.device(), stream, need);
  }
  check_status(pace_qkv_proj_rope(qkv.data_ptr(), hidden.data_ptr(), weight.data_ptr(),
                                  positions.data_ptr<int64_t>(), h.rows, h.width, (int)num_heads,
                                  (int)num_kv_heads, (int)head_size, h.stride, o.stride,
                                  cos_sin_cache.data_ptr(), pace_dtype(cos_sin_cache),
                                  (int)cos_sin_cache.size(1), cos_sin_cache.size(0),
                                  is_neox ? 1 : 0, pace_dtype(hidden), ws_ptr(ws),
                                  ws_bytes(ws), fault, stream),
               op);
}

// Workspace for the tensor-core GEMMs (caller's, or the per-stream cache).
Tensor gemm_workspace(const c10::optional<Tensor>& workspace, const at::Device& dev,
                      cudaStream_t stream, size_t need, const char* op) {
  if (workspace.has_value()) {
    const Tensor& ws = *workspace;
    TORCH_CHECK(ws.is_cuda() && ws.device() == dev && ws.is_contiguous() &&
                    (size_t)ws.nbytes() >= need,
                op, ": workspace must be a contiguous tensor of at least ", need, " bytes on ",
                dev);
    return ws;
  }
  if (need == 0) return Tensor();  // the call needs none
  return qkv_workspace(dev, stream, need);
}


// residual <- residual + input @ weight^T (o_proj / down_proj with the residual
// add in the epilogue); row_sumsq (optional, float32 [T, n / 32]) receives the
// new residual's sum-of-squares partials for the next RMSNorm.
void linear_residual(Tensor& residual, Tensor& input, Tensor& weight,
                     const c10::optional<Tensor>& row_sumsq,
                     const c10::optional<Tensor>& workspace,
                     const c10::optional<Tensor>& fault_flags) {
  const char* op = "linear_residual";
  check_cuda(input, op, "input");
  check_same_device(residual, input, op);
  check_same_device(weight, input, op);
  TORCH_CHECK(input.scalar_type() == at::kBFloat16 || input.scalar_type() == at::kHalf, op,
              ": input must be bfloat16 or float16");
  TORCH_CHECK(residual.scalar_type() == input.scalar_type() &&
                  weight.scalar_type() == input.scalar_type(),
              op, ": residual, input and weight must share a dtype");
  TORCH_CHECK(input.dim() == 2 && residual.dim() == 2 && weight.dim() == 2 &&
                  weight.is_contiguous(),
              op, ": input [T, k], residual [T, n] and a contiguous weight [n, k] expected");
  const Rows a = rows_of(input, op, "input");
  const Rows r = rows_of(residual, op, "residual");
  TORCH_CHECK(r.rows == a.rows && weight.size(0) == r.width && weight.size(1) == a.width, op,
              ": shapes do not match: input ", input.sizes(), ", residual ", residual.sizes(),
              ", weight ", weight.sizes());
  float* ss = nullptr;
  if (row_sumsq.has_value()) {
    const Tensor& t = *row_sumsq;
    check_same_device(t, input, op);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() &&
                    t.numel() >= a.rows * (r.width / 32),
                op, ": row_sumsq must be a contiguous float32 tensor of T * n / 32 entries");
    ss = t.data_ptr<float>();
  }
  const at::cuda::CUDAGuard guard(input.device());
  if (a.rows == 0) return;
  const cudaStream_t stream = stream_of(input);
  const size_t need = pace_linear_residual_workspace_size(a.rows, r.width, a.width,
                                                          input.device().index());
  Tensor ws = gemm_workspace(workspace, input.device(), stream, need, op);
  int32_t* fault = counter_ptr(fault_flags, input.device(), op, "fault_flags");
  check_status(pace_linear_residual(residual.data_ptr(), input.data_ptr(), weight.data_ptr(), ss,
                                    a.rows, r.width, a.width, a.stride, r.stride,
                                    pace_dtype(input), ws_ptr(ws), ws_bytes(ws), fault,
                                    stream),
               op);
}

void row_sumsq(Tensor& out, Tensor& input) {
  const char* op = "row_sumsq";
  check_cuda(input, op, "input");
  check_same_device(out, input, op);
  const Rows a = rows_of(input, op, "input");
  TORCH_CHECK(out.scalar_type() == at::kFloat && out.is_contiguous() &&
                  out.numel() >= a.rows * (a.width / 32),
              op, ": out must be a contiguous float32 tensor of T * hidden / 32 entries");
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_row_sumsq(out.data_ptr<float>(), input.data_ptr(), a.rows, a.width,
                              a.stride, pace_dtype(input), stream_of(input)),
               op);
}

// qkv = rope(inv * (hidden @ folded_weight^T)), inv the rows' RMSNorm factor
// from row_sumsq: input RMSNorm + qkv_proj + rotary_embedding in one GEMM.
void qkv_proj_rmsnorm_rotary_embedding(Tensor& qkv, Tensor& hidden, Tensor& folded_weight,
                                       Tensor& row_sumsq, double epsilon, Tensor& positions,
                                       int64_t head_size, int64_t num_heads,
                                       int64_t num_kv_heads, Tensor& cos_sin_cache,
                                       bool is_neox, const c10::optional<Tensor>& fault_flags,
                                       const c10::optional<Tensor>& workspace) {
  const char* op = "qkv_proj_rmsnorm_rotary_embedding";
  check_cuda(hidden, op, "hidden");
  for (const Tensor* t : {&qkv, &folded_weight, &row_sumsq, &positions, &cos_sin_cache})
    check_same_device(*t, hidden, op);
  TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf, op,
              ": hidden must be bfloat16 or float16");
  TORCH_CHECK(qkv.scalar_type() == hidden.scalar_type() &&
                  folded_weight.scalar_type() == hidden.scalar_type(),
              op, ": qkv, hidden and weight must share a dtype");
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.is_contiguous(), op,
              ": positions must be a contiguous int64 tensor");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), op,
              ": cos_sin_cache must be a contiguous [max_position, rot_dim] tensor");
  TORCH_CHECK(hidden.dim() == 2 && qkv.dim() == 2, op, ": hidden and qkv must be 2-D");
  const Rows h = rows_of(hidden, op, "hidden");
  const Rows o = rows_of(qkv, op, "qkv");
  const int64_t n = (num_heads + 2 * num_kv_heads) * head_size;
  TORCH_CHECK(o.rows == h.rows && o.width == n, op, ": qkv must be [T, ", n, "]");
  TORCH_CHECK(folded_weight.dim() == 2 && folded_weight.is_contiguous() &&
                  folded_weight.size(0) == n && folded_weight.size(1) == h.width,
              op, ": weight must be a contiguous [", n, ", ", h.width, "] tensor");
  TORCH_CHECK(row_sumsq.scalar_type() == at::kFloat && row_sumsq.is_contiguous() &&
                  row_sumsq.numel() >= h.rows * (h.width / 32),
              op, ": row_sumsq must be a contiguous float32 tensor of T * hidden / 32 entries");
  TORCH_CHECK(positions.numel() >= h.rows, op, ": positions has too few entries");
  const at::cuda::CUDAGuard guard(hidden.device());
  if (h.rows == 0) return;
  const cudaStream_t stream = stream_of(hidden);
  const size_t need = pace_qkv_proj_rope_workspace_size(h.rows, h.width, (int)num_heads,
                                                        (int)num_kv_heads, hidden.device().index());
  Tensor ws = gemm_workspace(workspace, hidden.device(), stream, need, op);
  int32_t* fault = counter_ptr(fault_flags, hidden.device(), op, "fault_flags");
  check_status(pace_qkv_proj_rmsnorm_rope(
                   qkv.data_ptr(), hidden.data_ptr(), folded_weight.data_ptr(),
                   row_sumsq.data_ptr<float>(), h.width / 32, (float)epsilon,
                   positions.data_ptr<int64_t>(), h.rows, h.width, (int)num_heads,
                   (int)num_kv_heads, (int)head_size, h.stride, o.stride,
                   cos_sin_cache.data_ptr(), pace_dtype(cos_sin_cache),
                   (int)cos_sin_cache.size(1), cos_sin_cache.size(0), is_neox ? 1 : 0,
                   pace_dtype(hidden), ws_ptr(ws), ws_bytes(ws), fault, stream),
               op);
}

// out = silu(gate) * up with [gate | up] = hidden @ weight^T, weight =
// [gate rows; up rows]: gate_up_proj + silu_and_mul in one GEMM.  With
// row_sumsq the rows are RMS-normalised by a per-row factor (the norm weight
// folded into `weight`).
void gate_up_silu(Tensor& out, Tensor& hidden, Tensor& weight,
                  const c10::optional<Tensor>& row_sumsq, double epsilon,
                  const c10::optional<Tensor>& workspace,
                  const c10::optional<Tensor>& fault_flags) {
  const char* op = "gate_up_silu";
  check_cuda(hidden, op, "hidden");
  check_same_device(out, hidden, op);
  check_same_device(weight, hidden, op);
  TORCH_CHECK(hidden.scalar_type() == at::kBFloat16 || hidden.scalar_type() == at::kHalf, op,
              ": hidden must be bfloat16 or float16");
  TORCH_CHECK(out.scalar_type() == hidden.scalar_type() &&
                  weight.scalar_type() == hidden.scalar_type(),
              op, ": out, hidden and weight must share a dtype");
  TORCH_CHECK(hidden.dim() == 2 && out.dim() == 2 && weight.dim() == 2 && weight.is_contiguous(),
              op, ": hidden [T, H], out [T, I] and a contiguous weight [2 I, H] expected");
  const Rows h = rows_of(hidden, op, "hidden");
  const Rows o = rows_of(out, op, "out");
  TORCH_CHECK(o.rows == h.rows && weight.size(0) == 2 * o.width && weight.size(1) == h.width, op,
              ": shapes do not match: hidden ", hidden.sizes(), ", out ", out.sizes(),
              ", weight ", weight.sizes());
  const float* ss = nullptr;
  if (row_sumsq.has_value()) {
    const Tensor& t = *row_sumsq;
    check_same_device(t, hidden, op);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() &&
                    t.numel() >= h.rows * (h.width / 32),
                op, ": row_sumsq must be a contiguous float32 tensor of T * hidden / 32 entries");
    ss = t.data_ptr<float>();
  }
  const at::cuda::CUDAGuard guard(hidden.device());
  if (h.rows == 0) return;
  const cudaStream_t stream = stream_of(hidden);
  const size_t need = pace_gate_up_silu_workspace_size(h.rows, h.width, o.width,
                                                       hidden.device().index());
  // 0: none needed (decode sizes) or a shape the entry point rejects
  Tensor ws = gemm_workspace(workspace, hidden.device(), stream, need, op);
  int32_t* fault = counter_ptr(fault_flags, hidden.device(), op, "fault_flags");
  check_status(pace_gate_up_silu(out.data_ptr(), hidden.data_ptr(), weight.data_ptr(), ss,
                                 h.width / 32, (float)epsilon, h.rows, h.width, o.width, h.stride,
                                 o.stride, pace_dtype(hidden), ws_ptr(ws), ws_bytes(ws),
                                 fault, stream),
               op);
}

// ------------------------------------------------------------ activation --
using ActFn = int (*)(void*, const void*, int64_t, int64_t, int64_t, int64_t, int, cudaStream_t);

void activation(Tensor& out, Tensor& input, ActFn fn, bool gated, const char* op) {
  check_cuda(input, op, "input");
  check_same_device(out, input, op);
  TORCH_CHECK(is_float_type(input) && out.scalar_type() == input.scalar_type(), op,
              ": out and input must share a float dtype");
  const Rows in = rows_of(input, op, "input");
  const Rows o = rows_of(out, op, "out");
  const int64_t d = gated ? in.width / 2 : in.width;
  TORCH_CHECK(!gated || in.width % 2 == 0, op, ": input width must be even");
  TORCH_CHECK(o.rows == in.rows && o.width == d, op, ": out shape ", out.sizes(),
              " does not match input ", input.sizes());
  const at::cuda::CUDAGuard guard(input.device());
  check_status(fn(out.data_ptr(), input.data_ptr(), in.rows, d, in.stride, o.stride,
                  pace_dtype(input), stream_of(input)),
               op);
}

void silu_and_mul(Tensor& out, Tensor& input) {
  activation(out, input, pace_silu_and_mul, true, "silu_and_mul");
}
void gelu_and_mul(Tensor& out, Tensor& input) {
  activation(out, input, pace_gelu_and_mul, true, "gelu_and_mul");
}
void gelu_tanh_and_mul(Tensor& out, Tensor& input) {
  activation(out, input, pace_gelu_tanh_and_mul, true, "gelu_tanh_and_mul");
}
void gelu_new(Tensor& out, Tensor& input) {
  activation(out, input, pace_gelu_new, false, "gelu_new");
}
void gelu_fast(Tensor& out, Tensor& input) {
  activation(out, input, pace_gelu_fast, false, "gelu_fast");
}

// ------------------------------------------------------------------- moe --
void topk_softmax(Tensor& topk_weights, Tensor& topk_indices, Tensor& token_expert_indices,
                  Tensor& gating_output, bool renormalize) {
  const char* op = "topk_softmax";
  check_cuda(gating_output, op, "gating_output");
  check_same_device(topk_weights, gating_output, op);
  check_same_device(topk_indices, gating_output, op);
  check_same_device(token_expert_indices, gating_output, op);
  TORCH_CHECK(gating_output.scalar_type() == at::kFloat && gating_output.is_contiguous(), op,
              ": gating_output must be a contiguous float32 tensor");
  TORCH_CHECK(topk_weights.scalar_type() == at::kFloat && topk_weights.is_contiguous(), op,
              ": topk_weights must be a contiguous float32 tensor");
  TORCH_CHECK(topk_indices.scalar_type() == at::kInt && topk_indices.is_contiguous() &&
                  token_expert_indices.scalar_type() == at::kInt &&
                  token_expert_indices.is_contiguous(),
              op, ": topk_indices and token_expert_indices must be contiguous int32 tensors");
  const int64_t E = gating_output.size(-1);
  TORCH_CHECK(E > 0, op, ": no experts");
  const int64_t T = gating_output.numel() / E;
  const int64_t k = topk_weights.size(-1);
  TORCH_CHECK(topk_weights.numel() == T * k && topk_indices.numel() == T * k &&
                  token_expert_indices.numel() == T * k,
              op, ": outputs must hold [", T, ", ", k, "]");
  const at::cuda::CUDAGuard guard(gating_output.device());
  check_status(pace_topk_softmax(topk_weights.data_ptr<float>(), topk_indices.data_ptr<int32_t>(),
                                 token_expert_indices.data_ptr<int32_t>(),
                                 gating_output.data_ptr<float>(), T, (int)E, (int)k,
                                 renormalize ? 1 : 0, stream_of(gating_output)),
               op);
}

void moe_align_block_size(Tensor topk_ids, int64_t num_experts, int64_t block_size,
                          Tensor sorted_token_ids, Tensor experts_ids, Tensor num_tokens_post_pad,
                          bool fill_padding) {
  const char* op = "moe_align_block_size";
  check_cuda(topk_ids, op, "topk_ids");
  check_same_device(sorted_token_ids, topk_ids, op);
  check_same_device(experts_ids, topk_ids, op);
  check_same_device(num_tokens_post_pad, topk_ids, op);
  const int dt = pace_dtype(topk_ids);
  TORCH_CHECK(dt >= PACE_U8 && dt <= PACE_I64, op, ": topk_ids must have an integral dtype");
  TORCH_CHECK(topk_ids.is_contiguous(), op, ": topk_ids must be contiguous");
  for (const Tensor* t : {&sorted_token_ids, &experts_ids, &num_tokens_post_pad})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), op,
                ": outputs must be contiguous int32 tensors");
  TORCH_CHECK(num_tokens_post_pad.numel() >= 1, op, ": num_tokens_post_pad is empty");
  TORCH_CHECK(num_experts > 0 && num_experts <= INT32_MAX && block_size > 0 &&
                  block_size <= INT32_MAX,
              op, ": num_experts and block_size must be positive int32 values");
  const at::cuda::CUDAGuard guard(topk_ids.device());
  check_status(pace_moe_align_block_size(
                   topk_ids.data_ptr(), dt, topk_ids.numel(), (int)num_experts, (int)block_size,
                   sorted_token_ids.data_ptr<int32_t>(), sorted_token_ids.numel(),
                   experts_ids.data_ptr<int32_t>(), experts_ids.numel(),
                   num_tokens_post_pad.data_ptr<int32_t>(), fill_padding ? 1 : 0,
                   stream_of(topk_ids)),
               op);
}

// Rows of the routed tokens in moe_align order (block 128): out[i] =
// input[sorted_token_ids[i] / top_k], zero for padding ids (>= numel).
void moe_gather_rows(Tensor& out, Tensor& input, Tensor& sorted_token_ids,
                     Tensor& num_tokens_post_pad, int64_t numel, int64_t top_k) {
  const char* op = "moe_gather_rows";
  check_cuda(input, op, "input");
  for (const Tensor* t : {&out, &sorted_token_ids, &num_tokens_post_pad})
    check_same_device(*t, input, op);
  TORCH_CHECK(input.scalar_type() == at::kBFloat16 || input.scalar_type() == at::kHalf, op,
              ": input must be bfloat16 or float16");
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), op, ": out and input dtypes differ");
  TORCH_CHECK(sorted_token_ids.scalar_type() == at::kInt && sorted_token_ids.is_contiguous() &&
                  num_tokens_post_pad.scalar_type() == at::kInt,
              op, ": sorted_token_ids and num_tokens_post_pad must be contiguous int32");
  TORCH_CHECK(input.dim() == 2 && out.dim() == 2 && out.size(1) == input.size(1), op,
              ": input [T, H] and out [num_sorted, H] expected");
  TORCH_CHECK(out.size(0) <= sorted_token_ids.numel(), op,
              ": out has more rows than sorted_token_ids");
  const Rows in = rows_of(input, op, "input");
  const Rows o = rows_of(out, op, "out");
  TORCH_CHECK(numel <= in.rows * top_k && top_k > 0, op, ": numel exceeds the input's rows");
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_moe_gather_rows(out.data_ptr(), input.data_ptr(),
                                    sorted_token_ids.data_ptr<int32_t>(), o.rows,
                                    num_tokens_post_pad.data_ptr<int32_t>(), numel, (int)top_k,
                                    in.width, in.stride, o.stride, pace_dtype(input),
                                    stream_of(input)),
               op);
}

// One expert GEMM of fused_experts on the tensor cores.  mode 0: out
// [num_sorted, I] = silu(a @ w1[e, :I]^T) * (a @ w1[e, I:]^T), w = w1 [E, 2I, K];
// mode 1: out [numel, H] rows sorted_token_ids[i] = topk_weights * (a @ w2[e]^T),
// w = w2 [E, H, K].
void moe_expert_gemm(Tensor& out, Tensor& a, Tensor& w, Tensor& sorted_token_ids,
                     Tensor& expert_ids, Tensor& num_tokens_post_pad, int64_t numel,
                     const c10::optional<Tensor>& topk_weights, int64_t mode,
                     const c10::optional<Tensor>& fault_flags) {
  const char* op = "moe_expert_gemm";
  check_cuda(a, op, "a");
  for (const Tensor* t : {&out, &w, &sorted_token_ids, &expert_ids, &num_tokens_post_pad})
    check_same_device(*t, a, op);
  TORCH_CHECK(mode == 0 || mode == 1, op, ": mode must be 0 (gate/up + SiLU) or 1 (down)");
  TORCH_CHECK(a.scalar_type() == at::kBFloat16 || a.scalar_type() == at::kHalf, op,
              ": a must be bfloat16 or float16");
  TORCH_CHECK(out.scalar_type() == a.scalar_type() && w.scalar_type() == a.scalar_type(), op,
              ": out, a and w must share a dtype");
  for (const Tensor* t : {&sorted_token_ids, &expert_ids, &num_tokens_post_pad})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), op,
                ": routing tensors must be contiguous int32");
  TORCH_CHECK(w.dim() == 3 && w.is_contiguous(), op, ": w must be a contiguous [E, N, K] tensor");
  TORCH_CHECK(a.dim() == 2 && out.dim() == 2, op, ": a and out must be 2-D");
  const Rows ar = rows_of(a, op, "a");
  const Rows orow = rows_of(out, op, "out");
  const int64_t E = w.size(0), k = w.size(2);
  TORCH_CHECK(ar.width == k, op, ": a width ", ar.width, " != w's K ", k);
  const int64_t n = mode == 0 ? w.size(1) / 2 : w.size(1);
  TORCH_CHECK(mode == 1 || w.size(1) % 2 == 0, op, ": w1 rows must be 2 * I");
  TORCH_CHECK(orow.width == n, op, ": out width ", orow.width, " != ", n);
  TORCH_CHECK(ar.rows <= sorted_token_ids.numel(), op, ": a has more rows than sorted_token_ids");
  TORCH_CHECK(expert_ids.numel() * 128 >= ar.rows, op,
              ": expert_ids must hold one entry per 128 sorted rows (moe_align with block 128)");
  const float* tw = nullptr;
  if (mode == 0) {
    TORCH_CHECK(orow.rows >= ar.rows, op, ": out needs a row per sorted row");
  } else {
    TORCH_CHECK(topk_weights.has_value(), op, ": mode 1 needs topk_weights");
    const Tensor& twt = *topk_weights;
    check_same_device(twt, a, op);
    TORCH_CHECK(twt.scalar_type() == at::kFloat && twt.is_contiguous() && twt.numel() >= numel,
                op, ": topk_weights must be a contiguous float32 tensor of >= numel entries");
    TORCH_CHECK(orow.rows >= numel, op, ": out needs numel rows");
    tw = twt.data_ptr<float>();
  }
  const at::cuda::CUDAGuard guard(a.device());
  int32_t* fault = counter_ptr(fault_flags, a.device(), op, "fault_flags");
  check_status(pace_moe_gemm(out.data_ptr(), a.data_ptr(), w.data_ptr(), ar.rows,
                            sorted_token_ids.data_ptr<int32_t>(), expert_ids.data_ptr<int32_t>(),
                            num_tokens_post_pad.data_ptr<int32_t>(), numel, tw, (int)E, n, k,
                            ar.stride, orow.stride, (int)mode, pace_dtype(a), fault,
                            stream_of(a)),
               op);
}

// ------------------------------------------------------------ kv transfer --
struct CacheSet {
  std::vector<void*> ptrs;
  int64_t num_blocks = 0;
  int64_t block_bytes = 0;
  c10::Device device = c10::Device(c10::kCPU);
};

CacheSet cache_set(const std::vector<Tensor>& caches, const char* op, const char* name) {
  TORCH_CHECK(!caches.empty(), op, ": ", name, " is empty");
  CacheSet s;
  s.device = caches[0].device();
  for (const Tensor& c : caches) {
    TORCH_CHECK(c.is_cuda() && c.device() == s.device, op, ": ", name,
                " must be CUDA tensors on one device");
    TORCH_CHECK(c.is_contiguous() && c.dim() >= 1, op, ": ", name, " must be contiguous");
    const int64_t nb = c.size(0);
    const int64_t bb = nb == 0 ? 0 : (int64_t)(c.numel() / nb) * (int64_t)c.element_size();
    if (s.ptrs.empty()) {
      s.num_blocks = nb;
      s.block_bytes = bb;
    }
    TORCH_CHECK(nb == s.num_blocks && bb == s.block_bytes, op, ": ", name,
                " layers differ in shape");
    s.ptrs.push_back(c.data_ptr());
  }
  return s;
}

// Block ids as a contiguous int32 tensor on `dev`.  int64 ids outside
// [0, INT32_MAX] become -1 before narrowing (on the device, no synchronisation),
// so the kernel skips and counts them instead of a wrapped id selecting a
// valid block.
Tensor ids_on(const Tensor& ids, const c10::Device& dev, const char* op, const char* name) {
  TORCH_CHECK(ids.dim() == 1, op, ": ", name, " must be 1-D");
  TORCH_CHECK(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, op, ": ", name,
              " must be int32 or int64");
  if (ids.scalar_type() == at::kLong) {
    Tensor t = ids.to(dev, /*non_blocking=*/false, /*copy=*/false);
    t = at::where(t.lt(0).logical_or(t.gt((int64_t)INT32_MAX)), at::full_like(t, -1), t);
    return t.to(at::kInt).contiguous();
  }
  return ids.to(dev, at::kInt, /*non_blocking=*/false, /*copy=*/false).contiguous();
}

// Method 3 of the Python-facing copies: the copy engines (pace_kv_copy_blocks_ce).
constexpr int64_t kMethodCopyEngine = 3;

// Host int32 copy of a 1-D id tensor (a device tensor is copied to the host,
// which synchronises with its stream).  int64 ids outside int32 become -1.
std::vector<int32_t> host_ids(const Tensor& ids, const char* op, const char* name) {
  TORCH_CHECK(ids.dim() == 1, op, ": ", name, " must be 1-D");
  TORCH_CHECK(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, op, ": ", name,
              " must be int32 or int64");
  Tensor t = ids.to(at::kCPU).to(at::kLong).contiguous();
  const int64_t* p = t.data_ptr<int64_t>();
  std::vector<int32_t> out((size_t)t.numel());
  for (int64_t i = 0; i < t.numel(); ++i)
    out[(size_t)i] = (p[i] < 0 || p[i] > (int64_t)INT32_MAX) ? -1 : (int32_t)p[i];
  return out;
}

void run_kv_copy(const std::vector<void*>& src, const std::vector<void*>& dst,
                 int64_t src_blocks, int64_t dst_blocks, int64_t block_bytes,
                 const c10::Device& exec, const Tensor& src_ids, const Tensor& dst_ids,
                 int64_t method, const c10::optional<Tensor>& bad_pairs, int64_t max_ctas,
                 int64_t wait_limit_ns, const char* op) {
  TORCH_CHECK(src.size() == dst.size(), op, ": source and destination layer counts differ (",
              src.size(), " vs ", dst.size(), ")");
  const at::cuda::CUDAGuard guard(exec);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream(exec.index()).stream();
  if (method == kMethodCopyEngine) {
    std::vector<int32_t> s = host_ids(src_ids, op, "src_block_ids");
    std::vector<int32_t> d = host_ids(dst_ids, op, "dst_block_ids");
    TORCH_CHECK(s.size() == d.size(), op, ": block id lists differ in length");
    counter_ptr(bad_pairs, exec, op, "bad_pairs");  // validates the counter before any copy
    int64_t nbad = 0, issued = 0;
    int rc;
    {
      // One copy call per run of blocks can take milliseconds of host time for
      // fragmented tables: let other Python threads (the serving loop) run.
      py::gil_scoped_release no_gil;
      rc = pace_kv_copy_blocks_ce(src.data(), dst.data(), (int)src.size(), s.data(), d.data(),
                                  (int64_t)s.size(), block_bytes, src_blocks, dst_blocks, &nbad,
                                  &issued, stream);
    }
    check_status(rc, op);
    if (bad_pairs.has_value() && nbad > 0) bad_pairs->add_(nbad);  // stream-ordered, as the kernels count
    return;
  }
  Tensor s = ids_on(src_ids, exec, op, "src_block_ids");
  Tensor d = ids_on(dst_ids, exec, op, "dst_block_ids");
  TORCH_CHECK(s.numel() == d.numel(), op, ": block id lists differ in length");
  int32_t* bad = counter_ptr(bad_pairs, exec, op, "bad_pairs");
  TORCH_CHECK(method != 2 || bad != nullptr, op,
              ": method 2 reports wait timeouts through bad_pairs; pass an int32 counter");
  pace_kv_copy_opts opts = {};
  opts.method = (int)method;
  opts.max_ctas = (int)max_ctas;
  opts.wait_limit_ns = (uint64_t)wait_limit_ns;
  check_status(pace_kv_copy_blocks_ex(src.data(), dst.data(), (int)src.size(),
                                      s.data_ptr<int32_t>(), d.data_ptr<int32_t>(), s.numel(),
                                      block_bytes, src_blocks, dst_blocks, bad, &opts, stream),
               op);
  // Device copies of the ids were allocated on this same stream, so the
  // caching allocator cannot hand their memory out before the kernel ran.
}

// Copy blocks between two lists of per-layer caches (same or different GPUs).
// Runs on the destination device (pull) unless push=True.
void copy_blocks_p2p(const std::vector<Tensor>& src_caches, const std::vector<Tensor>& dst_caches,
                     const Tensor& src_block_ids, const Tensor& dst_block_ids, int64_t method,
                     bool push, const c10::optional<Tensor>& bad_pairs, int64_t max_ctas,
                     int64_t wait_limit_ns) {
  const char* op = "copy_blocks_p2p";
  CacheSet s = cache_set(src_caches, op, "src_caches");
  CacheSet d = cache_set(dst_caches, op, "dst_caches");
  TORCH_CHECK(s.block_bytes == d.block_bytes, op, ": source and destination block sizes differ");
  const c10::Device exec = push ? s.device : d.device;
  const c10::Device other = push ? d.device : s.device;
  if (exec != other)
    check_status(pace_enable_peer_access(exec.index(), other.index()), op);
  run_kv_copy(s.ptrs, d.ptrs, s.num_blocks, d.num_blocks, s.block_bytes, exec, src_block_ids,
              dst_block_ids, method, bad_pairs, max_ctas, wait_limit_ns, op);
}

// Same, with the source given as raw per-layer pointers (e.g. mapped from
// another process with ipc_open_handle) of src_num_blocks blocks each.
void copy_blocks_from_ptrs(const std::vector<int64_t>& src_ptrs, int64_t src_num_blocks,
                           const std::vector<Tensor>& dst_caches, const Tensor& src_block_ids,
                           const Tensor& dst_block_ids, int64_t method,
                           const c10::optional<Tensor>& bad_pairs, int64_t max_ctas,
                           int64_t wait_limit_ns) {
  const char* op = "copy_blocks_from_ptrs";
  CacheSet d = cache_set(dst_caches, op, "dst_caches");
  std::vector<void*> s;
  for (int64_t p : src_ptrs) s.push_back(reinterpret_cast<void*>(p));
  run_kv_copy(s, d.ptrs, src_num_blocks, d.num_blocks, d.block_bytes, d.device, src_block_ids,
              dst_block_ids, method, bad_pairs, max_ctas, wait_limit_ns, op);
}

// Destination given as raw pointers (push into another process's cache).
void copy_blocks_to_ptrs(const std::vector<Tensor>& src_caches, const std::vector<int64_t>& dst_ptrs,
                         int64_t dst_num_blocks, const Tensor& src_block_ids,
                         const Tensor& dst_block_ids, int64_t method,
                         const c10::optional<Tensor>& bad_pairs, int64_t max_ctas,
                         int64_t wait_limit_ns) {
  const char* op = "copy_blocks_to_ptrs";
  CacheSet s = cache_set(src_caches, op, "src_caches");
  std::vector<void*> d;
  for (int64_t p : dst_ptrs) d.push_back(reinterpret_cast<void*>(p));
  run_kv_copy(s.ptrs, d, s.num_blocks, dst_num_blocks, s.block_bytes, s.device, src_block_ids,
              dst_block_ids, method, bad_pairs, max_ctas, wait_limit_ns, op);
}

// out[l, j] = caches[l][block_ids[j]]; out is [L, n, ...] on the caches'
// device or pinned host memory.
void gather_blocks(const std::vector<Tensor>& caches, const Tensor& block_ids, Tensor& out,
                   const c10::optional<Tensor>& bad_ids) {
  const char* op = "gather_blocks";
  CacheSet c = cache_set(caches, op, "caches");
  const at::cuda::CUDAGuard guard(c.device);
  Tensor ids = ids_on(block_ids, c.device, op, "block_ids");
  TORCH_CHECK(out.is_contiguous(), op, ": out must be contiguous");
  TORCH_CHECK(out.is_cuda() ? out.device() == c.device : out.is_pinned(), op,
              ": out must live on the caches' device or in pinned host memory");
  TORCH_CHECK((int64_t)out.numel() * out.element_size() ==
                  (int64_t)c.ptrs.size() * ids.numel() * c.block_bytes,
              op, ": out must hold num_layers * len(block_ids) blocks");
  int32_t* bad = counter_ptr(bad_ids, c.device, op, "bad_ids");
  cudaStream_t st = at::cuda::getCurrentCUDAStream(c.device.index()).stream();
  check_status(pace_kv_gather_blocks(c.ptrs.data(), (int)c.ptrs.size(), ids.data_ptr<int32_t>(),
                                     ids.numel(), c.block_bytes, c.num_blocks, out.data_ptr(), bad,
                                     st),
               op);
}

// caches[l][block_ids[j]] = src[l, j]
void scatter_blocks(const Tensor& src, const std::vector<Tensor>& caches, const Tensor& block_ids,
                    const c10::optional<Tensor>& bad_ids) {
  const char* op = "scatter_blocks";
  CacheSet c = cache_set(caches, op, "caches");
  const at::cuda::CUDAGuard guard(c.device);
  Tensor ids = ids_on(block_ids, c.device, op, "block_ids");
  TORCH_CHECK(src.is_contiguous(), op, ": src must be contiguous");
  TORCH_CHECK(src.is_cuda() ? src.device() == c.device : src.is_pinned(), op,
              ": src must live on the caches' device or in pinned host memory");
  TORCH_CHECK((int64_t)src.numel() * src.element_size() ==
                  (int64_t)c.ptrs.size() * ids.numel() * c.block_bytes,
              op, ": src must hold num_layers * len(block_ids) blocks");
  int32_t* bad = counter_ptr(bad_ids, c.device, op, "bad_ids");
  cudaStream_t st = at::cuda::getCurrentCUDAStream(c.device.index()).stream();
  check_status(pace_kv_scatter_blocks(src.data_ptr(), c.ptrs.data(), (int)c.ptrs.size(),
                                      ids.data_ptr<int32_t>(), ids.numel(), c.block_bytes,
                                      c.num_blocks, bad, st),
               op);
}

// ------------------------------------------------------- paged-KV append --
// K or V rows of nnz tokens: [nnz, heads, hd] (heads contiguous) or [nnz, heads*hd].
int64_t kv_row_stride(const Tensor& t, int64_t heads, int64_t hd, const char* op, const char* name) {
  TORCH_CHECK(t.is_cuda(), op, ": ", name, " must be a CUDA tensor");
  if (t.dim() == 3) {
    TORCH_CHECK(t.size(1) == heads && t.size(2) == hd, op, ": ", name, " must be [nnz, ", heads,
                ", ", hd, "]");
    TORCH_CHECK((hd <= 1 || t.stride(2) == 1) && (heads <= 1 || t.stride(1) == hd), op, ": ", name,
                " heads must be contiguous");
    return t.size(0) <= 1 ? heads * hd : t.stride(0);
  }
  TORCH_CHECK(t.dim() == 2 && t.size(1) == heads * hd, op, ": ", name, " must be [nnz, ",
              heads * hd, "] or [nnz, ", heads, ", ", hd, "]");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, op, ": ", name, " rows must be contiguous");
  return t.size(0) <= 1 ? heads * hd : t.stride(0);
}

struct PagedCache {
  int64_t pages, page_size, heads, hd;
};

PagedCache paged_cache_of(const Tensor& c, const std::string& layout, const char* op) {
  TORCH_CHECK(layout == "NHD", op, ": only the NHD layout [pages, 2, page_size, kv_heads, head_dim] "
              "(PaceServe's, flashinfer_attention_wrapper.py:63-73) is supported");
  TORCH_CHECK(c.is_cuda() && c.dim() == 5 && c.size(1) == 2 && c.is_contiguous(), op,
              ": paged_kv_cache must be a contiguous CUDA tensor [pages, 2, page_size, kv_heads, "
              "head_dim]");
  return {c.size(0), c.size(2), c.size(3), c.size(4)};
}

Tensor int32_on(const Tensor& t, const Tensor& like, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device(), op, ": ", name, " must be on the cache's device");
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1, op, ": ", name,
              " must be a 1-D int32 tensor");
  return t.contiguous();
}

// flashinfer.page.append_paged_kv_cache's signature (FlashInfer 0.2.0).
void append_paged_kv_cache(const Tensor& append_key, const Tensor& append_value,
                           const Tensor& batch_indices, const Tensor& positions,
                           Tensor& paged_kv_cache, const Tensor& kv_indices,
                           const Tensor& kv_indptr, const Tensor& kv_last_page_len,
                           const std::string& kv_layout, const c10::optional<Tensor>& bad_tokens) {
  const char* op = "append_paged_kv_cache";
  const PagedCache pc = paged_cache_of(paged_kv_cache, kv_layout, op);
  TORCH_CHECK(append_key.scalar_type() == paged_kv_cache.scalar_type() &&
                  append_value.scalar_type() == paged_kv_cache.scalar_type(),
              op, ": key, value and cache must share a dtype");
  check_same_device(append_key, paged_kv_cache, op);
  check_same_device(append_value, paged_kv_cache, op);
  const int64_t ks = kv_row_stride(append_key, pc.heads, pc.hd, op, "append_key");
  const int64_t vs = kv_row_stride(append_value, pc.heads, pc.hd, op, "append_value");
  const int64_t nnz = append_key.size(0);
  TORCH_CHECK(append_value.size(0) == nnz, op, ": key and value token counts differ");
  Tensor bi = int32_on(batch_indices, paged_kv_cache, op, "batch_indices");
  Tensor po = int32_on(positions, paged_kv_cache, op, "positions");
  Tensor ki = int32_on(kv_indices, paged_kv_cache, op, "kv_indices");
  Tensor kp = int32_on(kv_indptr, paged_kv_cache, op, "kv_indptr");
  Tensor kl = int32_on(kv_last_page_len, paged_kv_cache, op, "kv_last_page_len");
  TORCH_CHECK(bi.numel() >= nnz && po.numel() >= nnz, op,
              ": batch_indices and positions need one entry per token");
  TORCH_CHECK(kp.numel() >= 1 && kl.numel() >= kp.numel() - 1, op,
              ": kv_indptr needs batch + 1 entries and kv_last_page_len batch entries");
  int32_t* bad = counter_ptr(bad_tokens, paged_kv_cache.device(), op, "bad_tokens");
  const at::cuda::CUDAGuard guard(paged_kv_cache.device());
  check_status(pace_append_paged_kv_cache(
                   append_key.data_ptr(), append_value.data_ptr(), nnz, (int)pc.heads, (int)pc.hd,
                   ks, vs, bi.data_ptr<int32_t>(), po.data_ptr<int32_t>(),
                   paged_kv_cache.data_ptr(), pc.pages, (int)pc.page_size, ki.data_ptr<int32_t>(),
                   ki.numel(), kp.data_ptr<int32_t>(), kl.data_ptr<int32_t>(), kp.numel() - 1, bad,
                   pace_dtype(paged_kv_cache), stream_of(paged_kv_cache)),
               op);
}

// One launch for get_seq_lens + get_batch_indices_positions + append.
void append_paged_kv_cache_by_indptr(const Tensor& append_key, const Tensor& append_value,
                                     const Tensor& append_indptr, Tensor& paged_kv_cache,
                                     const Tensor& kv_indices, const Tensor& kv_indptr,
                                     const Tensor& kv_last_page_len,
                                     const c10::optional<Tensor>& bad_tokens) {
  const char* op = "append_paged_kv_cache_by_indptr";
  const PagedCache pc = paged_cache_of(paged_kv_cache, "NHD", op);
  TORCH_CHECK(append_key.scalar_type() == paged_kv_cache.scalar_type() &&
                  append_value.scalar_type() == paged_kv_cache.scalar_type(),
              op, ": key, value and cache must share a dtype");
  check_same_device(append_key, paged_kv_cache, op);
  check_same_device(append_value, paged_kv_cache, op);
  const int64_t ks = kv_row_stride(append_key, pc.heads, pc.hd, op, "append_key");
  const int64_t vs = kv_row_stride(append_value, pc.heads, pc.hd, op, "append_value");
  const int64_t nnz = append_key.size(0);
  TORCH_CHECK(append_value.size(0) == nnz, op, ": key and value token counts differ");
  Tensor ai = int32_on(append_indptr, paged_kv_cache, op, "append_indptr");
  Tensor ki = int32_on(kv_indices, paged_kv_cache, op, "kv_indices");
  Tensor kp = int32_on(kv_indptr, paged_kv_cache, op, "kv_indptr");
  Tensor kl = int32_on(kv_last_page_len, paged_kv_cache, op, "kv_last_page_len");
  TORCH_CHECK(ai.numel() == kp.numel() && kl.numel() >= kp.numel() - 1 && kp.numel() >= 1, op,
              ": append_indptr and kv_indptr need batch + 1 entries, kv_last_page_len batch");
  int32_t* bad = counter_ptr(bad_tokens, paged_kv_cache.device(), op, "bad_tokens");
  const at::cuda::CUDAGuard guard(paged_kv_cache.device());
  check_status(pace_append_paged_kv_cache_by_indptr(
                   append_key.data_ptr(), append_value.data_ptr(), nnz, (int)pc.heads,
                   (int)pc.hd, ks, vs, ai.data_ptr<int32_t>(), paged_kv_cache.data_ptr(), pc.pages,
                   (int)pc.page_size, ki.data_ptr<int32_t>(), ki.numel(), kp.data_ptr<int32_t>(),
                   kl.data_ptr<int32_t>(), kp.numel() - 1, bad, pace_dtype(paged_kv_cache),
                   stream_of(paged_kv_cache)),
               op);
}

// -------------------------------------------------- quantised paged KV cache --
struct QuantisedCache {
  PagedCache pc;
  void* codes;
  void* exponents;
};

QuantisedCache quantised_cache_of(const Tensor& codes, const Tensor& exponents, const char* op) {
  const PagedCache pc = paged_cache_of(codes, "NHD", op);
  TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn, op, ": codes must be float8_e4m3fn");
  TORCH_CHECK(exponents.device() == codes.device() && exponents.scalar_type() == at::kByte &&
                  exponents.dim() == 4 && exponents.is_contiguous() &&
                  exponents.sizes() == codes.sizes().slice(0, 4),
              op, ": exponents must be a contiguous uint8 tensor [pages, 2, page_size, kv_heads] "
              "on the codes' device");
  return {pc, codes.data_ptr(), exponents.data_ptr()};
}

template <typename Fn>
void quantised_cache_op(Fn fn, const char* op, const Tensor& key, const Tensor& value,
                        const Tensor& indptr, const Tensor& codes, const Tensor& exponents,
                        const Tensor& kv_indices, const Tensor& kv_indptr,
                        const Tensor& kv_last_page_len, const c10::optional<Tensor>& bad_tokens) {
  const QuantisedCache q = quantised_cache_of(codes, exponents, op);
  check_same_device(key, codes, op);
  check_same_device(value, codes, op);
  TORCH_CHECK(is_float_type(key) && key.scalar_type() == value.scalar_type(), op,
              ": key and value must share one of float32, float16 and bfloat16");
  const int64_t ks = kv_row_stride(key, q.pc.heads, q.pc.hd, op, "key");
  const int64_t vs = kv_row_stride(value, q.pc.heads, q.pc.hd, op, "value");
  const int64_t rows = key.size(0);
  TORCH_CHECK(value.size(0) == rows, op, ": key and value token counts differ");
  Tensor ai = int32_on(indptr, codes, op, "indptr");
  Tensor ki = int32_on(kv_indices, codes, op, "kv_indices");
  Tensor kp = int32_on(kv_indptr, codes, op, "kv_indptr");
  Tensor kl = int32_on(kv_last_page_len, codes, op, "kv_last_page_len");
  TORCH_CHECK(ai.numel() == kp.numel() && kl.numel() >= kp.numel() - 1 && kp.numel() >= 1, op,
              ": the token indptr and kv_indptr need batch + 1 entries, kv_last_page_len batch");
  int32_t* bad = counter_ptr(bad_tokens, codes.device(), op, "bad_tokens");
  const at::cuda::CUDAGuard guard(codes.device());
  check_status(fn(key.data_ptr(), value.data_ptr(), rows, (int)q.pc.heads, (int)q.pc.hd, ks, vs,
                  ai.data_ptr<int32_t>(), q.codes, q.exponents, q.pc.pages, (int)q.pc.page_size,
                  ki.data_ptr<int32_t>(), ki.numel(), kp.data_ptr<int32_t>(),
                  kl.data_ptr<int32_t>(), kp.numel() - 1, bad, pace_dtype(key), stream_of(codes)),
               op);
}

void append_quantised_paged_kv_cache(const Tensor& append_key, const Tensor& append_value,
                                     const Tensor& append_indptr, Tensor& codes, Tensor& exponents,
                                     const Tensor& kv_indices, const Tensor& kv_indptr,
                                     const Tensor& kv_last_page_len,
                                     const c10::optional<Tensor>& bad_tokens) {
  quantised_cache_op(pace_append_quantised_paged_kv_cache, "append_quantised_paged_kv_cache",
                     append_key, append_value, append_indptr, codes, exponents, kv_indices,
                     kv_indptr, kv_last_page_len, bad_tokens);
}

void read_quantised_paged_kv_cache(Tensor& key, Tensor& value, const Tensor& out_indptr,
                                   const Tensor& codes, const Tensor& exponents,
                                   const Tensor& kv_indices, const Tensor& kv_indptr,
                                   const Tensor& kv_last_page_len,
                                   const c10::optional<Tensor>& bad_tokens) {
  quantised_cache_op(pace_read_quantised_paged_kv_cache, "read_quantised_paged_kv_cache", key,
                     value, out_indptr, codes, exponents, kv_indices, kv_indptr, kv_last_page_len,
                     bad_tokens);
}

// ------------------------------------------------------------ paged attention --
// A planned step: the C struct and its words in host memory (page-locked where
// a GPU is present, so that the copy to the device need not be waited for).
struct AttentionPlan {
  pace_attention_plan plan{};
  Tensor words;
};

const int32_t* host_ints(const c10::optional<Tensor>& t, int64_t n, const char* name, Tensor* keep) {
  const char* op = "plan_paged_attention";
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->is_cpu() && t->scalar_type() == at::kInt && t->dim() == 1 && t->numel() >= n, op,
              ": ", name, " must be a 1-D int32 CPU tensor of at least ", n, " entries");
  *keep = t->contiguous();
  return keep->data_ptr<int32_t>();
}

AttentionPlan plan_paged_attention(const Tensor& qo_indptr, const Tensor& kv_indptr,
                                   const Tensor& kv_indices, const Tensor& kv_last_page_len,
                                   int64_t num_heads, int64_t num_kv_heads, int64_t head_dim,
                                   int64_t page_size, int64_t window_left,
                                   const c10::optional<Tensor>& prefix_lens,
                                   const c10::optional<Tensor>& doc_starts, int64_t tree_words,
                                   int64_t num_sms) {
  const char* op = "plan_paged_attention";
  TORCH_CHECK(qo_indptr.dim() == 1 && qo_indptr.numel() >= 1 &&
                  qo_indptr.numel() == kv_indptr.numel(),
              op, ": qo_indptr and kv_indptr need batch + 1 entries");
  const int64_t batch = qo_indptr.numel() - 1;
  for (int64_t v : {num_heads, num_kv_heads, head_dim, page_size, window_left, tree_words, num_sms})
    TORCH_CHECK(v >= INT32_MIN && v <= INT32_MAX, op, ": argument out of range");
  Tensor keep[6];
  const int32_t* qo = host_ints(qo_indptr, batch + 1, "qo_indptr", &keep[0]);
  const int32_t* kp = host_ints(kv_indptr, batch + 1, "kv_indptr", &keep[1]);
  const int32_t* ki = host_ints(kv_indices, 0, "kv_indices", &keep[2]);
  const int32_t* kl = host_ints(kv_last_page_len, batch, "kv_last_page_len", &keep[3]);
  const int64_t total_q = qo[batch];
  TORCH_CHECK(total_q >= 0, op, ": qo_indptr must be ascending");
  const int32_t* pl = host_ints(prefix_lens, batch, "prefix_lens", &keep[4]);
  const int32_t* ds = host_ints(doc_starts, total_q, "doc_starts", &keep[5]);
  const int64_t words =
      pace_paged_attention_plan_words(batch, total_q, kv_indices.numel(), (int)num_sms);
  AttentionPlan p;
  p.words = torch::empty({words}, torch::TensorOptions().dtype(torch::kInt32).pinned_memory(
                                      at::cuda::is_available()));
  check_status(pace_paged_attention_plan(&p.plan, p.words.data_ptr<int32_t>(), words, qo, kp, ki,
                                         kv_indices.numel(), kl, batch, (int)num_heads,
                                         (int)num_kv_heads, (int)head_dim, (int)page_size,
                                         (int)window_left, pl, ds, (int)tree_words, (int)num_sms),
               op);
  p.words = p.words.narrow(0, 0, p.plan.num_words);
  return p;
}

int64_t heads_stride(const Tensor& t, int64_t heads, int64_t hd, const char* op, const char* name) {
  TORCH_CHECK(t.dim() == 3 && t.size(1) == heads && t.size(2) == hd, op, ": ", name, " must be [",
              "tokens, ", heads, ", ", hd, "]");
  TORCH_CHECK((hd <= 1 || t.stride(2) == 1) && (heads <= 1 || t.stride(1) == hd), op, ": ", name,
              " heads must be contiguous");
  return t.size(0) <= 1 ? heads * hd : t.stride(0);
}

void paged_attention(Tensor& out, const Tensor& query, const Tensor& paged_kv_cache,
                     const AttentionPlan& plan, const Tensor& plan_words, const Tensor& workspace,
                     double sm_scale, double logits_soft_cap,
                     const c10::optional<Tensor>& exponents,
                     const c10::optional<Tensor>& alibi_slopes,
                     const c10::optional<Tensor>& tree_mask, const c10::optional<Tensor>& lse,
                     const c10::optional<Tensor>& fault_flags) {
  const char* op = "paged_attention";
  const pace_attention_plan& pl = plan.plan;
  check_cuda(query, op, "query");
  check_same_device(out, query, op);
  check_same_device(paged_kv_cache, query, op);
  TORCH_CHECK(is_float_type(query) && out.scalar_type() == query.scalar_type(), op,
              ": query and out must share one of float32, float16 and bfloat16");
  const PagedCache pc = paged_cache_of(paged_kv_cache, "NHD", op);
  TORCH_CHECK(pc.heads == pl.num_kv_heads && pc.hd == pl.head_dim && pc.page_size == pl.page_size,
              op, ": the cache's pages [", pc.page_size, ", ", pc.heads, ", ", pc.hd,
              "] are not the plan's");
  if (exponents.has_value())
    quantised_cache_of(paged_kv_cache, *exponents, op);
  else
    TORCH_CHECK(paged_kv_cache.scalar_type() == query.scalar_type(), op,
                ": the cache must have the query's dtype, or be float8_e4m3fn codes with exponents");
  TORCH_CHECK(query.size(0) == pl.total_q && out.size(0) == pl.total_q, op, ": the plan is for ",
              pl.total_q, " tokens");
  const int64_t qs = heads_stride(query, pl.num_heads, pl.head_dim, op, "query");
  const int64_t os = heads_stride(out, pl.num_heads, pl.head_dim, op, "out");
  TORCH_CHECK(plan_words.device() == query.device() && plan_words.scalar_type() == at::kInt &&
                  plan_words.is_contiguous() && plan_words.numel() >= pl.num_words,
              op, ": plan_words must hold the plan's words on the query's device");
  TORCH_CHECK(workspace.device() == query.device() && workspace.scalar_type() == at::kByte &&
                  workspace.is_contiguous(),
              op, ": workspace must be a contiguous uint8 tensor on the query's device");
  const float* slopes = nullptr;
  if (alibi_slopes.has_value()) {
    TORCH_CHECK(alibi_slopes->device() == query.device() &&
                    alibi_slopes->scalar_type() == at::kFloat && alibi_slopes->is_contiguous() &&
                    alibi_slopes->numel() == pl.num_heads,
                op, ": alibi_slopes must be a float32 tensor [", pl.num_heads, "] on the query's "
                "device");
    slopes = alibi_slopes->data_ptr<float>();
  }
  const uint64_t* bits = nullptr;
  if (tree_mask.has_value()) {
    TORCH_CHECK(tree_mask->device() == query.device() && tree_mask->scalar_type() == at::kLong &&
                    tree_mask->is_contiguous() && tree_mask->dim() == 2 &&
                    tree_mask->size(0) == pl.total_q && tree_mask->size(1) == pl.tree_words,
                op, ": tree_mask must be a contiguous int64 tensor [", pl.total_q, ", ",
                pl.tree_words, "] on the query's device");
    bits = reinterpret_cast<const uint64_t*>(tree_mask->data_ptr<int64_t>());
  }
  float* lse_ptr = nullptr;
  if (lse.has_value()) {
    TORCH_CHECK(lse->device() == query.device() && lse->scalar_type() == at::kFloat &&
                    lse->is_contiguous() && lse->dim() == 2 && lse->size(0) == pl.total_q &&
                    lse->size(1) == pl.num_heads,
                op, ": lse must be a contiguous float32 tensor [", pl.total_q, ", ", pl.num_heads,
                "] on the query's device");
    lse_ptr = lse->data_ptr<float>();
  }
  int32_t* fault = counter_ptr(fault_flags, query.device(), op, "fault_flags");
  const at::cuda::CUDAGuard guard(query.device());
  check_status(pace_paged_attention(&pl, plan_words.data_ptr<int32_t>(), out.data_ptr(),
                                    query.data_ptr(), qs, os, paged_kv_cache.data_ptr(),
                                    exponents.has_value() ? exponents->data_ptr() : nullptr,
                                    pc.pages, (float)sm_scale, (float)logits_soft_cap, slopes, bits,
                                    lse_ptr, workspace.data_ptr(), (size_t)workspace.numel(), fault,
                                    pace_dtype(query), stream_of(query)),
               op);
}

// A plan with its words on the device, its workspace and (for a tree) its mask:
// what every layer of the step runs on.
struct AttentionStep {
  AttentionPlan plan;
  Tensor words, workspace;
  c10::optional<Tensor> tree_mask;
  cudaStream_t stream;
  at::cuda::CUDAEvent ready;
  bool captured = false;  // a CUDA graph holds the addresses of all three

  AttentionStep(const AttentionPlan& p, const Tensor& w, const Tensor& ws,
                const c10::optional<Tensor>& mask)
      : plan(p), words(w), workspace(ws), tree_mask(mask) {
    check_cuda(words, "AttentionStep", "words");
    const at::cuda::CUDAGuard guard(words.device());
    const auto cur = at::cuda::getCurrentCUDAStream(words.device().index());
    stream = cur.stream();
    ready.record(cur);
  }

  Tensor forward(const Tensor& query, const Tensor& paged_kv_cache,
                 const c10::optional<Tensor>& exponents, double sm_scale, double logits_soft_cap,
                 const c10::optional<Tensor>& alibi_slopes, const c10::optional<Tensor>& out,
                 const c10::optional<Tensor>& lse, const c10::optional<Tensor>& fault_flags) {
    check_cuda(query, "paged_attention", "query");
    const auto cur = at::cuda::getCurrentCUDAStream(query.device().index());
    if (at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) {
      captured = true;  // with the GPU idle; the step has to outlive the graph
    } else if (cur.stream() != stream && query.device() == words.device()) {
      // another stream than the plan's: its copy to the device comes first, and its memory is
      // kept from reuse until this stream is done with it
      ready.block(cur);
      words.record_stream(cur);
      workspace.record_stream(cur);
      if (tree_mask.has_value()) tree_mask->record_stream(cur);
    }
    Tensor o = out.has_value() ? *out : torch::empty(query.sizes(), query.options());
    paged_attention(o, query, paged_kv_cache, plan, words, workspace, sm_scale, logits_soft_cap,
                    exponents, alibi_slopes, tree_mask, lse, fault_flags);
    return o;
  }
};

// ------------------------------------------------------------- step tables --
// A tensor that the kernel writes (or reads) in place: int32 or int64, 1-D,
// contiguous, on the tables' device, with at least n entries.
template <typename I>
I* entries_of(const Tensor& t, const Tensor& like, int64_t n, const char* op, const char* name) {
  TORCH_CHECK(t.device() == like.device() && t.dim() == 1 && t.is_contiguous() &&
                  t.scalar_type() == c10::CppTypeToScalarType<I>::value && t.numel() >= n,
              op, ": ", name, " must be a contiguous 1-D ",
              c10::toString(c10::CppTypeToScalarType<I>::value), " tensor of at least ", n,
              " entries on ", like.device());
  return t.data_ptr<I>();
}

// Rows of block_tables.
int64_t table_rows(const Tensor& t, int64_t requests, const char* op) {
  check_cuda(t, op, "block_tables");
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 &&
                  (t.size(1) <= 1 || t.stride(1) == 1) && t.size(0) >= requests,
              op, ": block_tables must be int32 [at least ", requests,
              ", max_blocks], contiguous in its rows");
  TORCH_CHECK(requests <= 1 || t.stride(0) >= t.size(1), op, ": block_tables' rows overlap");
  return t.size(0) <= 1 ? t.size(1) : t.stride(0);
}

void build_step_tables(Tensor& block_tables, const Tensor& seq_lens, const Tensor& new_lens,
                       int64_t page_size, Tensor& free_pages, Tensor& free_count,
                       Tensor& append_indptr, Tensor& kv_indptr, Tensor& kv_indices,
                       Tensor& kv_last_page_len, Tensor& batch_indices, Tensor& positions,
                       Tensor& slot_mapping, Tensor& status, Tensor& arrivals) {
  const char* op = "build_step_tables";
  const int64_t r = seq_lens.numel(), tokens = slot_mapping.numel();
  const int64_t stride = table_rows(block_tables, r, op);
  const Tensor& like = block_tables;
  TORCH_CHECK(new_lens.numel() == r, op, ": seq_lens and new_lens differ in length");
  TORCH_CHECK(batch_indices.numel() == tokens && positions.numel() == tokens, op,
              ": batch_indices, positions and slot_mapping differ in length");
  const at::cuda::CUDAGuard guard(like.device());
  check_status(
      pace_build_step_tables(
          block_tables.data_ptr<int32_t>(), stride, block_tables.size(1),
          entries_of<int32_t>(seq_lens, like, r, op, "seq_lens"),
          entries_of<int32_t>(new_lens, like, r, op, "new_lens"), r, page_size,
          entries_of<int32_t>(free_pages, like, 0, op, "free_pages"), free_pages.numel(),
          entries_of<int32_t>(free_count, like, 1, op, "free_count"),
          entries_of<int32_t>(append_indptr, like, r + 1, op, "append_indptr"),
          entries_of<int32_t>(kv_indptr, like, r + 1, op, "kv_indptr"),
          entries_of<int32_t>(kv_indices, like, 0, op, "kv_indices"), kv_indices.numel(),
          entries_of<int32_t>(kv_last_page_len, like, r, op, "kv_last_page_len"),
          entries_of<int32_t>(batch_indices, like, 0, op, "batch_indices"),
          entries_of<int64_t>(positions, like, 0, op, "positions"),
          entries_of<int64_t>(slot_mapping, like, 0, op, "slot_mapping"), tokens,
          entries_of<int32_t>(status, like, 1, op, "status"),
          entries_of<int32_t>(arrivals, like, 1, op, "arrivals"), stream_of(like)),
      op);
}

void release_pages(const Tensor& block_tables, const Tensor& held_lens, const Tensor& kept_lens,
                   int64_t page_size, Tensor& free_pages, Tensor& free_count, Tensor& status,
                   Tensor& arrivals) {
  const char* op = "release_pages";
  const int64_t r = held_lens.numel();
  const int64_t stride = table_rows(block_tables, r, op);
  const Tensor& like = block_tables;
  TORCH_CHECK(kept_lens.numel() == r, op, ": held_lens and kept_lens differ in length");
  const at::cuda::CUDAGuard guard(like.device());
  check_status(pace_release_pages(block_tables.data_ptr<int32_t>(), stride, block_tables.size(1),
                                  entries_of<int32_t>(held_lens, like, r, op, "held_lens"),
                                  entries_of<int32_t>(kept_lens, like, r, op, "kept_lens"), r,
                                  page_size,
                                  entries_of<int32_t>(free_pages, like, 0, op, "free_pages"),
                                  free_pages.numel(),
                                  entries_of<int32_t>(free_count, like, 1, op, "free_count"),
                                  entries_of<int32_t>(status, like, 1, op, "status"),
                                  entries_of<int32_t>(arrivals, like, 1, op, "arrivals"),
                                  stream_of(like)),
               op);
}

// ----------------------------------------------- head norms with rotation --
struct HeadArgs {
  Rows q, k;
  int num_heads, num_kv_heads;
};

HeadArgs check_heads(const Tensor& positions, const Tensor& query, const Tensor& key,
                     const Tensor& q_weight, const Tensor& k_weight, int64_t head_size,
                     const Tensor& cos_sin_cache, const char* op) {
  check_cuda(query, op, "query");
  check_same_device(positions, query, op);
  check_same_device(key, query, op);
  check_same_device(q_weight, query, op);
  check_same_device(k_weight, query, op);
  check_same_device(cos_sin_cache, query, op);
  TORCH_CHECK(head_size > 0 && head_size <= INT32_MAX, op, ": head_size must be positive");
  TORCH_CHECK(is_float_type(query) && key.scalar_type() == query.scalar_type() &&
                  q_weight.scalar_type() == query.scalar_type() &&
                  k_weight.scalar_type() == query.scalar_type(),
              op, ": query, key and the weights must share a float dtype");
  TORCH_CHECK(q_weight.is_contiguous() && q_weight.numel() == head_size &&
                  k_weight.is_contiguous() && k_weight.numel() == head_size,
              op, ": q_weight and k_weight must be [", head_size, "] and contiguous");
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.is_contiguous(), op,
              ": positions must be a contiguous int64 tensor");
  TORCH_CHECK(cos_sin_cache.dim() == 2 && cos_sin_cache.is_contiguous(), op,
              ": cos_sin_cache must be a contiguous [max_position, rot_dim] tensor");
  TORCH_CHECK(cos_sin_cache.scalar_type() == at::kFloat ||
                  cos_sin_cache.scalar_type() == query.scalar_type(),
              op, ": cos_sin_cache must be float32 or the query dtype");
  HeadArgs a{qk_rows(query, head_size, op, "query"), qk_rows(key, head_size, op, "key"), 0, 0};
  TORCH_CHECK(a.k.rows == a.q.rows, op, ": query and key token counts differ");
  TORCH_CHECK(positions.numel() >= a.q.rows, op, ": positions has ", positions.numel(),
              " entries for ", a.q.rows, " tokens");
  a.num_heads = (int)(a.q.width / head_size);
  a.num_kv_heads = (int)(a.k.width / head_size);
  return a;
}

void qk_norm_rotary_embedding(Tensor& positions, Tensor& query, Tensor& key, Tensor& q_weight,
                              Tensor& k_weight, double epsilon, int64_t head_size,
                              Tensor& cos_sin_cache, bool is_neox,
                              const c10::optional<Tensor>& fault_flags) {
  const char* op = "qk_norm_rotary_embedding";
  const HeadArgs a =
      check_heads(positions, query, key, q_weight, k_weight, head_size, cos_sin_cache, op);
  int32_t* fault = counter_ptr(fault_flags, query.device(), op, "fault_flags");
  const at::cuda::CUDAGuard guard(query.device());
  check_status(pace_qk_norm_rotary_embedding(
                   positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(),
                   q_weight.data_ptr(), k_weight.data_ptr(), (float)epsilon, a.q.rows, a.num_heads,
                   a.num_kv_heads, (int)head_size, a.q.stride, a.k.stride,
                   cos_sin_cache.data_ptr(), pace_dtype(cos_sin_cache),
                   (int)cos_sin_cache.size(1), cos_sin_cache.size(0), is_neox ? 1 : 0,
                   pace_dtype(query), fault, stream_of(query)),
               op);
}

void qk_norm_rotary_append(Tensor& positions, Tensor& query, const Tensor& key,
                           const Tensor& value, Tensor& q_weight, Tensor& k_weight, double epsilon,
                           int64_t head_size, Tensor& cos_sin_cache, bool is_neox,
                           Tensor& paged_kv_cache, const Tensor& slot_mapping,
                           const c10::optional<Tensor>& bad_tokens,
                           const c10::optional<Tensor>& fault_flags) {
  const char* op = "qk_norm_rotary_append";
  const HeadArgs a =
      check_heads(positions, query, key, q_weight, k_weight, head_size, cos_sin_cache, op);
  check_same_device(value, query, op);
  check_same_device(paged_kv_cache, query, op);
  check_same_device(slot_mapping, query, op);
  const PagedCache pc = paged_cache_of(paged_kv_cache, "NHD", op);
  TORCH_CHECK(value.scalar_type() == query.scalar_type() &&
                  paged_kv_cache.scalar_type() == query.scalar_type(),
              op, ": query, key, value and cache must share a dtype");
  const Rows v = qk_rows(value, head_size, op, "value");
  TORCH_CHECK(v.rows == a.q.rows && v.width == a.k.width, op, ": key and value differ in shape");
  TORCH_CHECK(pc.heads == a.num_kv_heads && pc.hd == head_size, op, ": the cache holds ", pc.heads,
              " heads of ", pc.hd, ", the keys are ", a.num_kv_heads, " of ", head_size);
  TORCH_CHECK(slot_mapping.scalar_type() == at::kLong && slot_mapping.is_contiguous() &&
                  slot_mapping.numel() >= a.q.rows,
              op, ": slot_mapping must be a contiguous int64 tensor with an entry for each token");
  int32_t* bad = counter_ptr(bad_tokens, query.device(), op, "bad_tokens");
  int32_t* fault = counter_ptr(fault_flags, query.device(), op, "fault_flags");
  const at::cuda::CUDAGuard guard(query.device());
  check_status(pace_qk_norm_rotary_append(
                   positions.data_ptr<int64_t>(), query.data_ptr(), key.data_ptr(),
                   value.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(), (float)epsilon,
                   a.q.rows, a.num_heads, a.num_kv_heads, (int)head_size, a.q.stride, a.k.stride,
                   v.stride, cos_sin_cache.data_ptr(), pace_dtype(cos_sin_cache),
                   (int)cos_sin_cache.size(1), cos_sin_cache.size(0), is_neox ? 1 : 0,
                   paged_kv_cache.data_ptr(), pc.pages, (int)pc.page_size,
                   slot_mapping.data_ptr<int64_t>(), bad, pace_dtype(query), fault, stream_of(query)),
               op);
}

// ------------------------------------------------------- 8-bit projections --
// Codes [rows, width] int8 and their scales [rows], on the device of `like`.
Rows codes_of(const Tensor& codes, const Tensor& scales, const Tensor& like, const char* op,
              const char* name, const char* scales_name) {
  check_same_device(codes, like, op);
  check_same_device(scales, like, op);
  TORCH_CHECK(codes.scalar_type() == at::kChar && codes.dim() == 2, op, ": ", name,
              " must be int8 [rows, k]");
  const Rows r = rows_of(codes, op, name);
  TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.is_contiguous() &&
                  scales.numel() == r.rows,
              op, ": ", scales_name, " must be a contiguous float32 tensor with an entry for each of ",
              name, "'s ", r.rows, " rows");
  return r;
}

void quantise_rows(Tensor& codes, Tensor& scales, const Tensor& input) {
  const char* op = "quantise_rows";
  check_cuda(input, op, "input");
  TORCH_CHECK(is_float_type(input), op, ": input dtype must be float32, float16 or bfloat16");
  const Rows in = rows_of(input, op, "input");
  const Rows c = codes_of(codes, scales, input, op, "codes", "scales");
  TORCH_CHECK(c.rows == in.rows && c.width == in.width, op, ": codes ", codes.sizes(),
              " do not match input ", input.sizes());
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_quantise_rows(codes.data_ptr<int8_t>(), scales.data_ptr<float>(),
                                  input.data_ptr(), in.rows, in.width, in.stride, c.stride,
                                  pace_dtype(input), stream_of(input)),
               op);
}

void rms_norm_quantise(Tensor& codes, Tensor& scales, const Tensor& input, const Tensor& weight,
                       double epsilon, const c10::optional<Tensor>& residual) {
  const char* op = "rms_norm_quantise";
  check_cuda(input, op, "input");
  check_same_device(weight, input, op);
  TORCH_CHECK(is_float_type(input) && weight.scalar_type() == input.scalar_type(), op,
              ": input and weight must share one of float32, float16 and bfloat16");
  const Rows in = rows_of(input, op, "input");
  const Rows c = codes_of(codes, scales, input, op, "codes", "scales");
  TORCH_CHECK(c.rows == in.rows && c.width == in.width, op, ": codes ", codes.sizes(),
              " do not match input ", input.sizes());
  TORCH_CHECK(weight.is_contiguous() && weight.numel() == in.width, op, ": weight must be [",
              in.width, "] and contiguous");
  Rows r{0, 0, 0};
  if (residual.has_value()) {
    check_same_device(*residual, input, op);
    TORCH_CHECK(residual->scalar_type() == input.scalar_type(), op,
                ": residual must have the input's dtype");
    r = rows_of(*residual, op, "residual");
    TORCH_CHECK(r.rows == in.rows && r.width == in.width, op, ": residual shape ",
                residual->sizes(), " does not match input ", input.sizes());
  }
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_rms_norm_quantise(codes.data_ptr<int8_t>(), scales.data_ptr<float>(),
                                      input.data_ptr(),
                                      residual.has_value() ? residual->data_ptr() : nullptr,
                                      weight.data_ptr(), (float)epsilon, in.rows, in.width,
                                      in.stride, r.stride, c.stride, pace_dtype(input),
                                      stream_of(input)),
               op);
}

void silu_and_mul_quantise(Tensor& codes, Tensor& scales, const Tensor& input) {
  const char* op = "silu_and_mul_quantise";
  check_cuda(input, op, "input");
  TORCH_CHECK(is_float_type(input), op, ": input dtype must be float32, float16 or bfloat16");
  const Rows in = rows_of(input, op, "input");
  const Rows c = codes_of(codes, scales, input, op, "codes", "scales");
  TORCH_CHECK(c.rows == in.rows && 2 * c.width == in.width, op, ": codes ", codes.sizes(),
              " do not match input ", input.sizes());
  const at::cuda::CUDAGuard guard(input.device());
  check_status(pace_silu_and_mul_quantise(codes.data_ptr<int8_t>(), scales.data_ptr<float>(),
                                          input.data_ptr(), in.rows, c.width, in.stride, c.stride,
                                          pace_dtype(input), stream_of(input)),
               op);
}

struct Int8Args {
  Rows x, w, out;
  int32_t* fault;
};

Int8Args check_int8(const Tensor& out, const char* out_name, const Tensor& codes,
                    const Tensor& token_scales, const Tensor& weight, const Tensor& channel_scales,
                    bool gated, const c10::optional<Tensor>& fault_flags, const char* op) {
  check_cuda(out, op, out_name);
  TORCH_CHECK(is_float_type(out) && out.dim() == 2, op, ": ", out_name,
              " must be [tokens, features] of float32, float16 or bfloat16");
  const Int8Args a{codes_of(codes, token_scales, out, op, "codes", "token_scales"),
                   codes_of(weight, channel_scales, out, op, "weight", "channel_scales"),
                   rows_of(out, op, out_name),
                   counter_ptr(fault_flags, out.device(), op, "fault_flags")};
  TORCH_CHECK(!gated || a.w.rows % 2 == 0, op, ": weight needs as many gate as up rows");
  TORCH_CHECK(a.x.width == a.w.width && a.out.rows == a.x.rows &&
                  a.out.width == (gated ? a.w.rows / 2 : a.w.rows),
              op, ": shapes do not match: ", out_name, " ", out.sizes(), ", codes ", codes.sizes(),
              ", weight ", weight.sizes());
  return a;
}

void int8_linear_into(Tensor& out, const Tensor& codes, const Tensor& token_scales,
                      const Tensor& weight, const Tensor& channel_scales,
                      const c10::optional<Tensor>& bias, bool residual,
                      const c10::optional<Tensor>& fault_flags, const char* op) {
  const Int8Args a = check_int8(out, residual ? "residual" : "out", codes, token_scales, weight,
                                channel_scales, false, fault_flags, op);
  const void* b = nullptr;
  if (bias.has_value()) {
    check_same_device(*bias, out, op);
    TORCH_CHECK(bias->scalar_type() == out.scalar_type() && bias->is_contiguous() &&
                    bias->numel() == a.w.rows,
                op, ": bias must be a contiguous [", a.w.rows, "] tensor of the output's dtype");
    b = bias->data_ptr();
  }
  const at::cuda::CUDAGuard guard(out.device());
  check_status(pace_int8_linear(out.data_ptr(), codes.data_ptr<int8_t>(),
                                token_scales.data_ptr<float>(), weight.data_ptr<int8_t>(),
                                channel_scales.data_ptr<float>(), b,
                                residual ? out.data_ptr() : nullptr, a.x.rows, a.w.rows, a.x.width,
                                a.x.stride, a.w.stride, a.out.stride, a.out.stride,
                                pace_dtype(out), a.fault, stream_of(out)),
               op);
}

void int8_linear(Tensor& out, const Tensor& codes, const Tensor& token_scales,
                 const Tensor& weight, const Tensor& channel_scales,
                 const c10::optional<Tensor>& bias, const c10::optional<Tensor>& fault_flags) {
  int8_linear_into(out, codes, token_scales, weight, channel_scales, bias, false, fault_flags,
                   "int8_linear");
}

void int8_linear_residual(Tensor& residual, const Tensor& codes, const Tensor& token_scales,
                          const Tensor& weight, const Tensor& channel_scales,
                          const c10::optional<Tensor>& bias,
                          const c10::optional<Tensor>& fault_flags) {
  int8_linear_into(residual, codes, token_scales, weight, channel_scales, bias, true, fault_flags,
                   "int8_linear_residual");
}

void int8_gate_up_silu(Tensor& out, const Tensor& codes, const Tensor& token_scales,
                       const Tensor& weight, const Tensor& channel_scales,
                       const c10::optional<Tensor>& fault_flags) {
  const char* op = "int8_gate_up_silu";
  const Int8Args a =
      check_int8(out, "out", codes, token_scales, weight, channel_scales, true, fault_flags, op);
  const at::cuda::CUDAGuard guard(out.device());
  check_status(pace_int8_gate_up_silu(out.data_ptr(), codes.data_ptr<int8_t>(),
                                      token_scales.data_ptr<float>(), weight.data_ptr<int8_t>(),
                                      channel_scales.data_ptr<float>(), a.x.rows, a.out.width,
                                      a.x.width, a.x.stride, a.w.stride, a.out.stride,
                                      pace_dtype(out), a.fault, stream_of(out)),
               op);
}

py::tuple ipc_get_handle(const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "ipc_get_handle: tensor must be on a CUDA device");
  const at::cuda::CUDAGuard guard(t.device());
  char h[PACE_IPC_HANDLE_BYTES];
  int64_t off = 0;
  check_status(pace_ipc_get_handle(t.data_ptr(), h, &off), "ipc_get_handle");
  return py::make_tuple(py::bytes(h, PACE_IPC_HANDLE_BYTES), off);
}

int64_t ipc_open_handle(const py::bytes& handle, int64_t device) {
  std::string h = handle;
  TORCH_CHECK(h.size() == PACE_IPC_HANDLE_BYTES, "ipc_open_handle: handle must be ",
              PACE_IPC_HANDLE_BYTES, " bytes");
  void* base = nullptr;
  check_status(pace_ipc_open_handle(h.data(), (int)device, &base), "ipc_open_handle");
  return reinterpret_cast<int64_t>(base);
}

void ipc_close_handle(int64_t base) {
  check_status(pace_ipc_close_handle(reinterpret_cast<void*>(base)), "ipc_close_handle");
}

void enable_peer_access(int64_t device, int64_t peer) {
  check_status(pace_enable_peer_access((int)device, (int)peer), "enable_peer_access");
}

bool can_access_peer(int64_t device, int64_t peer) {
  int can = 0;
  check_status(pace_can_access_peer((int)device, (int)peer, &can), "can_access_peer");
  return can != 0;
}

}  // namespace

PYBIND11_MODULE(_C, m) {
  m.doc() = "PaceServe per-layer ops and KV transfer on B200 (sm_100a)";
  m.def("version", &pace_version);
  m.def("set_pdl", [](bool on) { pace_set_pdl(on ? 1 : 0); },
        "Enable/disable programmatic dependent launch for the per-layer ops.");
  m.def("get_pdl", []() { return pace_get_pdl() != 0; });

  auto ln = m.def_submodule("layernorm_ops");
  ln.def("rms_norm", &rms_norm, "Apply Root Mean Square (RMS) Normalization to the input tensor.",
         py::arg("out"), py::arg("input"), py::arg("weight"), py::arg("epsilon"));
  ln.def("linear_residual", &linear_residual,
         "residual += input @ weight^T on the tensor cores (o_proj / down_proj with the residual "
         "add in the epilogue); row_sumsq receives the new rows' sum-of-squares partials.",
         py::arg("residual"), py::arg("input"), py::arg("weight"),
         py::arg("row_sumsq") = py::none(), py::arg("workspace") = py::none(),
         py::arg("fault_flags") = py::none());
  ln.def("row_sumsq", &row_sumsq, "out[t, g] = sum of input[t, 32g:32g+32]^2 (float32).",
         py::arg("out"), py::arg("input"));
  ln.def("fused_add_rms_norm", &fused_add_rms_norm,
         "In place: residual += input; input = rms_norm(residual) * weight.", py::arg("input"),
         py::arg("residual"), py::arg("weight"), py::arg("epsilon"));

  auto pe = m.def_submodule("pos_encoding_ops");
  pe.def("rotary_embedding", &rotary_embedding,
         "Apply GPT-NeoX or GPT-J style rotary embedding to query and key", py::arg("positions"),
         py::arg("query"), py::arg("key"), py::arg("head_size"), py::arg("cos_sin_cache"),
         py::arg("is_neox"));
  pe.def("qk_norm_rotary_embedding", &qk_norm_rotary_embedding,
         "RMSNorm of every query and key head, then the rotary embedding, in place and in one "
         "pass.",
         py::arg("positions"), py::arg("query"), py::arg("key"), py::arg("q_weight"),
         py::arg("k_weight"), py::arg("epsilon"), py::arg("head_size"), py::arg("cos_sin_cache"),
         py::arg("is_neox"), py::arg("fault_flags") = py::none());
  pe.def("qk_norm_rotary_append", &qk_norm_rotary_append,
         "The same with the keys' result and the values written to their slots of a paged cache.",
         py::arg("positions"), py::arg("query"), py::arg("key"), py::arg("value"),
         py::arg("q_weight"), py::arg("k_weight"), py::arg("epsilon"), py::arg("head_size"),
         py::arg("cos_sin_cache"), py::arg("is_neox"), py::arg("paged_kv_cache"),
         py::arg("slot_mapping"), py::arg("bad_tokens") = py::none(),
         py::arg("fault_flags") = py::none());
  pe.def("qkv_proj_rotary_embedding", &qkv_proj_rotary_embedding,
         "qkv = hidden @ weight^T on the tensor cores with the rotary embedding applied to the "
         "q and k heads before rounding (fused qkv_proj + rotary_embedding).",
         py::arg("qkv"), py::arg("hidden"), py::arg("weight"), py::arg("positions"),
         py::arg("head_size"), py::arg("num_heads"), py::arg("num_kv_heads"),
         py::arg("cos_sin_cache"), py::arg("is_neox"), py::arg("fault_flags") = py::none(),
         py::arg("workspace") = py::none());
  pe.def("qkv_proj_rmsnorm_rotary_embedding", &qkv_proj_rmsnorm_rotary_embedding,
         "qkv = rope(inv * (hidden @ folded_weight^T)): input RMSNorm (weight folded into the "
         "projection, per-row factor from row_sumsq), qkv projection and rotary embedding in "
         "one tensor-core GEMM.",
         py::arg("qkv"), py::arg("hidden"), py::arg("folded_weight"), py::arg("row_sumsq"),
         py::arg("epsilon"), py::arg("positions"), py::arg("head_size"), py::arg("num_heads"),
         py::arg("num_kv_heads"), py::arg("cos_sin_cache"), py::arg("is_neox"),
         py::arg("fault_flags") = py::none(), py::arg("workspace") = py::none());
  pe.def("qkv_proj_rope_workspace_size",
         [](int64_t num_tokens, int64_t hidden_size, int64_t num_heads, int64_t num_kv_heads,
            int64_t device) {
           return pace_qkv_proj_rope_workspace_size(num_tokens, hidden_size, (int)num_heads,
                                                    (int)num_kv_heads, (int)device);
         },
         "Bytes of zero-filled workspace qkv_proj_rotary_embedding needs for this shape.",
         py::arg("num_tokens"), py::arg("hidden_size"), py::arg("num_heads"),
         py::arg("num_kv_heads"), py::arg("device"));

  auto act = m.def_submodule("activation_ops");
  act.def("silu_and_mul", &silu_and_mul, "Activation function used in SwiGLU.", py::arg("out"),
          py::arg("input"));
  act.def("gate_up_silu", &gate_up_silu,
          "out = silu(gate) * up, [gate | up] = hidden @ weight^T on the tensor cores "
          "(gate_up_proj + silu_and_mul in one GEMM); with row_sumsq the post-attention "
          "RMSNorm is a per-row factor and weight holds the norm weight folded in.",
          py::arg("out"), py::arg("hidden"), py::arg("weight"),
          py::arg("row_sumsq") = py::none(), py::arg("epsilon") = 1e-6,
          py::arg("workspace") = py::none(), py::arg("fault_flags") = py::none());
  act.def("gelu_and_mul", &gelu_and_mul, "GeGLU: gelu(x[:, :d]) * x[:, d:] (erf GELU).",
          py::arg("out"), py::arg("input"));
  act.def("gelu_tanh_and_mul", &gelu_tanh_and_mul,
          "GeGLU with the tanh-approximated GELU.", py::arg("out"), py::arg("input"));
  act.def("gelu_new", &gelu_new, "GELU implementation used in GPT-2.", py::arg("out"),
          py::arg("input"));
  act.def("gelu_fast", &gelu_fast, "Approximate GELU implementation.", py::arg("out"),
          py::arg("input"));

  auto moe = m.def_submodule("moe_ops");
  moe.def("topk_softmax", &topk_softmax, "Apply topk softmax to the gating outputs.",
          py::arg("topk_weights"), py::arg("topk_indices"), py::arg("token_expert_indices"),
          py::arg("gating_output"), py::arg("renormalize") = false);
  moe.def("moe_align_block_size", &moe_align_block_size,
          "Aligning the number of tokens to be processed by each expert such that it is "
          "divisible by the block size.",
          py::arg("topk_ids"), py::arg("num_experts"), py::arg("block_size"),
          py::arg("sorted_token_ids"), py::arg("experts_ids"), py::arg("num_tokens_post_pad"),
          py::arg("fill_padding") = false);
  moe.def("moe_gather_rows", &moe_gather_rows,
          "out[i] = input[sorted_token_ids[i] / top_k] (zero rows for padding ids).",
          py::arg("out"), py::arg("input"), py::arg("sorted_token_ids"),
          py::arg("num_tokens_post_pad"), py::arg("numel"), py::arg("top_k"));
  moe.def("moe_expert_gemm", &moe_expert_gemm,
          "Grouped expert GEMM on the tensor cores: mode 0 gate/up + SiLU-and-mul, mode 1 down "
          "projection times the routing weight (rows scattered to the token slots).",
          py::arg("out"), py::arg("a"), py::arg("w"), py::arg("sorted_token_ids"),
          py::arg("expert_ids"), py::arg("num_tokens_post_pad"), py::arg("numel"),
          py::arg("topk_weights") = py::none(), py::arg("mode") = 0,
          py::arg("fault_flags") = py::none());

  auto at_ = m.def_submodule("attention_ops");
  py::class_<AttentionPlan>(at_, "AttentionPlan")
      .def_property_readonly("words", [](const AttentionPlan& p) { return p.words; })
      .def_property_readonly("total_q", [](const AttentionPlan& p) { return p.plan.total_q; })
      .def_property_readonly("workspace_bytes",
                             [](const AttentionPlan& p) { return p.plan.workspace_bytes; })
      .def_property_readonly("num_few", [](const AttentionPlan& p) { return p.plan.num_few; })
      .def_property_readonly("num_many", [](const AttentionPlan& p) { return p.plan.num_many; })
      .def_property_readonly("few_slots", [](const AttentionPlan& p) { return p.plan.few_slots; })
      .def_property_readonly("many_slots",
                             [](const AttentionPlan& p) { return p.plan.many_slots; });
  at_.def("plan_paged_attention", &plan_paged_attention,
          "Plan one step's attention from its host metadata (int32 CPU tensors).",
          py::arg("qo_indptr"), py::arg("kv_indptr"), py::arg("kv_indices"),
          py::arg("kv_last_page_len"), py::arg("num_heads"), py::arg("num_kv_heads"),
          py::arg("head_dim"), py::arg("page_size"), py::arg("window_left") = -1,
          py::arg("prefix_lens") = py::none(), py::arg("doc_starts") = py::none(),
          py::arg("tree_words") = 0, py::arg("num_sms") = 148);
  at_.def("paged_attention", &paged_attention,
          "Attention of a planned step over a paged KV cache (16-bit, float32 or quantised).",
          py::arg("out"), py::arg("query"), py::arg("paged_kv_cache"), py::arg("plan"),
          py::arg("plan_words"), py::arg("workspace"), py::arg("sm_scale"),
          py::arg("logits_soft_cap") = 0.0, py::arg("exponents") = py::none(),
          py::arg("alibi_slopes") = py::none(), py::arg("tree_mask") = py::none(),
          py::arg("lse") = py::none(), py::arg("fault_flags") = py::none());

  py::class_<AttentionStep>(at_, "AttentionStep")
      .def(py::init<const AttentionPlan&, const Tensor&, const Tensor&,
                    const c10::optional<Tensor>&>(),
           py::arg("plan"), py::arg("words"), py::arg("workspace"),
           py::arg("tree_mask") = py::none())
      .def_readonly("captured", &AttentionStep::captured)
      .def("forward", &AttentionStep::forward, py::arg("query"), py::arg("paged_kv_cache"),
           py::arg("exponents"), py::arg("sm_scale"), py::arg("logits_soft_cap"),
           py::arg("alibi_slopes"), py::arg("out"), py::arg("lse"), py::arg("fault_flags"));

  auto i8 = m.def_submodule("int8_ops");
  i8.def("quantise_rows", &quantise_rows,
         "Rows as 8-bit integers with a scale each (the largest magnitude is 127).",
         py::arg("codes"), py::arg("scales"), py::arg("input"));
  i8.def("rms_norm_quantise", &rms_norm_quantise,
         "rms_norm(input) * weight quantised; with residual, residual += input and its norm.",
         py::arg("codes"), py::arg("scales"), py::arg("input"), py::arg("weight"),
         py::arg("epsilon"), py::arg("residual") = py::none());
  i8.def("silu_and_mul_quantise", &silu_and_mul_quantise,
         "silu(input[:, :d]) * input[:, d:] quantised.", py::arg("codes"), py::arg("scales"),
         py::arg("input"));
  i8.def("linear", &int8_linear,
         "out = (codes @ weight^T) * token_scales * channel_scales (+ bias) on the tensor cores, "
         "the sums exact in 32 bits.",
         py::arg("out"), py::arg("codes"), py::arg("token_scales"), py::arg("weight"),
         py::arg("channel_scales"), py::arg("bias") = py::none(),
         py::arg("fault_flags") = py::none());
  i8.def("linear_residual", &int8_linear_residual, "residual += the same product.",
         py::arg("residual"), py::arg("codes"), py::arg("token_scales"), py::arg("weight"),
         py::arg("channel_scales"), py::arg("bias") = py::none(),
         py::arg("fault_flags") = py::none());
  i8.def("gate_up_silu", &int8_gate_up_silu,
         "out = silu(gate) * up, [gate | up] the same product with a weight [2 I, k].",
         py::arg("out"), py::arg("codes"), py::arg("token_scales"), py::arg("weight"),
         py::arg("channel_scales"), py::arg("fault_flags") = py::none());

  auto kv = m.def_submodule("kv_transfer_ops");
  kv.def("copy_blocks_p2p", &copy_blocks_p2p,
         "Copy KV blocks src_block_ids of src_caches onto dst_block_ids of dst_caches "
         "(per-layer caches, possibly on different GPUs; pull on the destination GPU by default). "
         "method: 0 auto, 1 SIMT, 2 bulk (needs bad_pairs), 3 copy engines (host ids, no SM); "
         "max_ctas > 0 caps the kernel's CTAs; wait_limit_ns bounds the bulk method's waits.",
         py::arg("src_caches"), py::arg("dst_caches"), py::arg("src_block_ids"),
         py::arg("dst_block_ids"), py::arg("method") = 0, py::arg("push") = false,
         py::arg("bad_pairs") = py::none(), py::arg("max_ctas") = 0, py::arg("wait_limit_ns") = 0);
  kv.def("copy_blocks_from_ptrs", &copy_blocks_from_ptrs, py::arg("src_ptrs"),
         py::arg("src_num_blocks"), py::arg("dst_caches"), py::arg("src_block_ids"),
         py::arg("dst_block_ids"), py::arg("method") = 0, py::arg("bad_pairs") = py::none(),
         py::arg("max_ctas") = 0, py::arg("wait_limit_ns") = 0);
  kv.def("copy_blocks_to_ptrs", &copy_blocks_to_ptrs, py::arg("src_caches"), py::arg("dst_ptrs"),
         py::arg("dst_num_blocks"), py::arg("src_block_ids"), py::arg("dst_block_ids"),
         py::arg("method") = 0, py::arg("bad_pairs") = py::none(), py::arg("max_ctas") = 0,
         py::arg("wait_limit_ns") = 0);
  kv.def("gather_blocks", &gather_blocks, py::arg("caches"), py::arg("block_ids"), py::arg("out"),
         py::arg("bad_ids") = py::none());
  kv.def("scatter_blocks", &scatter_blocks, py::arg("src"), py::arg("caches"),
         py::arg("block_ids"), py::arg("bad_ids") = py::none());
  kv.def("append_paged_kv_cache", &append_paged_kv_cache,
         "Append K/V rows of new tokens to a paged cache (flashinfer.append_paged_kv_cache).",
         py::arg("append_key"), py::arg("append_value"), py::arg("batch_indices"),
         py::arg("positions"), py::arg("paged_kv_cache"), py::arg("kv_indices"),
         py::arg("kv_indptr"), py::arg("kv_last_page_len"), py::arg("kv_layout") = "NHD",
         py::arg("bad_tokens") = py::none());
  kv.def("append_paged_kv_cache_by_indptr", &append_paged_kv_cache_by_indptr,
         "Append, deriving each token's request and position from append_indptr in the kernel.",
         py::arg("append_key"), py::arg("append_value"), py::arg("append_indptr"),
         py::arg("paged_kv_cache"), py::arg("kv_indices"), py::arg("kv_indptr"),
         py::arg("kv_last_page_len"), py::arg("bad_tokens") = py::none());
  kv.def("append_quantised_paged_kv_cache", &append_quantised_paged_kv_cache,
         "Quantise K/V rows of new tokens (e4m3 codes, one power-of-two exponent per row and head) "
         "and append them to a paged cache of codes and exponents.",
         py::arg("append_key"), py::arg("append_value"), py::arg("append_indptr"),
         py::arg("codes"), py::arg("exponents"), py::arg("kv_indices"), py::arg("kv_indptr"),
         py::arg("kv_last_page_len"), py::arg("bad_tokens") = py::none());
  kv.def("read_quantised_paged_kv_cache", &read_quantised_paged_kv_cache,
         "Read requests' rows of a quantised paged cache back in sequence order.", py::arg("key"),
         py::arg("value"), py::arg("out_indptr"), py::arg("codes"), py::arg("exponents"),
         py::arg("kv_indices"), py::arg("kv_indptr"), py::arg("kv_last_page_len"),
         py::arg("bad_tokens") = py::none());
  kv.def("build_step_tables", &build_step_tables,
         "Block tables, index arrays and slots of a step from its requests' lengths; new pages "
         "come from a stack of free ones.",
         py::arg("block_tables"), py::arg("seq_lens"), py::arg("new_lens"), py::arg("page_size"),
         py::arg("free_pages"), py::arg("free_count"), py::arg("append_indptr"),
         py::arg("kv_indptr"), py::arg("kv_indices"), py::arg("kv_last_page_len"),
         py::arg("batch_indices"), py::arg("positions"), py::arg("slot_mapping"),
         py::arg("status"), py::arg("arrivals"));
  kv.def("release_pages", &release_pages,
         "The pages past the requests' kept tokens go back onto the stack of free ones.",
         py::arg("block_tables"), py::arg("held_lens"), py::arg("kept_lens"),
         py::arg("page_size"), py::arg("free_pages"), py::arg("free_count"), py::arg("status"),
         py::arg("arrivals"));
  kv.def("ipc_get_handle", &ipc_get_handle, py::arg("tensor"));
  kv.def("ipc_open_handle", &ipc_open_handle, py::arg("handle"), py::arg("device"));
  kv.def("ipc_close_handle", &ipc_close_handle, py::arg("base"));
  kv.def("enable_peer_access", &enable_peer_access, py::arg("device"), py::arg("peer"));
  kv.def("can_access_peer", &can_access_peer, py::arg("device"), py::arg("peer"));
}
