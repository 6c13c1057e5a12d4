// Thin PyTorch extension over the C ABI: registers `torch.ops.asymgemm_b200.m_grouped_gemm_nt`, the one launch every
// operator of the Python API funnels into. It plays the part of the reference's pybind layer (csrc/apis/gemm.hpp:1034-1115
// binds the operators, csrc/jit/kernel_runtime.hpp:99-119 launches on torch's current stream): take tensors, fill the
// plain descriptor, launch on the current CUDA stream of a's device, turn a failure into c10::Error (RuntimeError in
// Python). No arithmetic happens here and the GEMM operator allocates nothing; the library below it has no torch
// dependency.
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include "../../include/asymgemm_b200.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

void* ptr_of(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }

void check_index_tensor(const OptTensor& t, const char* name, const at::Tensor& a) {
  if (!t.has_value() || !t->defined()) return;
  TORCH_CHECK(t->is_cuda() && t->device() == a.device(), name, " must live on a's device");
  TORCH_CHECK(t->scalar_type() == at::kInt && t->is_contiguous(), name, " must be a contiguous int32 tensor");
}

// kind: 0 bf16, 1 fp8 (fp32 scales), 2 int8, 3 nvfp4, 4 fp8 with blocked UE8M0 scales. layout: 0 contiguous, 1 masked.
void m_grouped_gemm_nt(int64_t kind, int64_t layout, const at::Tensor& a, const OptTensor& sfa, const at::Tensor& b,
                       const OptTensor& sfb, at::Tensor& d, const OptTensor& offsets, const OptTensor& experts,
                       int64_t max_segments, const OptTensor& masked_m, int64_t m, int64_t n, int64_t k, int64_t num_groups,
                       const OptTensor& scratch, const at::Tensor& status, int64_t timeout_ms, const OptTensor& raw_dump,
                       double alpha, int64_t tile_config, int64_t no_split, const OptTensor& stage, int64_t stage_chunk_bytes,
                       int64_t num_sms, int64_t epilogue, const OptTensor& scatter_meta, const OptTensor& scatter_bases) {
  TORCH_CHECK(a.is_cuda(), "a must be a CUDA tensor");
  TORCH_CHECK(b.is_cuda() || b.is_pinned(), "b must be a CUDA tensor or pinned host memory (b.is_cuda() or b.is_pinned())");
  TORCH_CHECK(d.is_cuda() || d.is_pinned(), "d must be a CUDA tensor or pinned host memory");
  TORCH_CHECK(a.is_contiguous() && b.is_contiguous() && d.is_contiguous(), "a, b and d must be contiguous");
  TORCH_CHECK(d.scalar_type() == at::kBFloat16 || d.scalar_type() == at::kFloat, "d must be bfloat16 or float32");
  TORCH_CHECK(status.is_cuda() && status.device() == a.device() && status.scalar_type() == at::kInt && status.numel() >= 1,
              "status must be an int32 tensor on a's device");
  check_index_tensor(offsets, "offsets", a);
  check_index_tensor(experts, "experts", a);
  check_index_tensor(masked_m, "masked_m", a);
  if (raw_dump.has_value() && raw_dump->defined())
    TORCH_CHECK(raw_dump->is_cuda() && raw_dump->scalar_type() == at::kInt && raw_dump->is_contiguous(),
                "raw_dump must be a contiguous int32 CUDA tensor");

  ag_gemm_desc_t desc{};
  desc.layout = static_cast<int32_t>(layout);
  desc.d_dtype = d.scalar_type() == at::kFloat ? AG_D_FP32 : AG_D_BF16;
  desc.a = a.data_ptr();
  desc.sfa = ptr_of(sfa);
  desc.b = b.data_ptr();
  desc.sfb = ptr_of(sfb);
  desc.d = d.data_ptr();
  desc.offsets = static_cast<const int32_t*>(ptr_of(offsets));
  desc.experts = static_cast<const int32_t*>(ptr_of(experts));
  desc.max_segments = static_cast<int32_t>(max_segments);
  desc.masked_m = static_cast<const int32_t*>(ptr_of(masked_m));
  desc.m = m;
  desc.n = n;
  desc.k = k;
  desc.num_groups = static_cast<int32_t>(num_groups);
  if (scratch.has_value() && scratch->defined()) {
    desc.scratch = scratch->data_ptr();
    desc.scratch_bytes = static_cast<uint64_t>(scratch->numel()) * scratch->element_size();
  }
  desc.status = static_cast<int32_t*>(status.data_ptr());
  desc.epilogue = static_cast<int32_t>(epilogue);
  const bool has_meta = scatter_meta.has_value() && scatter_meta->defined();
  const bool has_bases = scatter_bases.has_value() && scatter_bases->defined();
  TORCH_CHECK(has_meta == has_bases, "scatter_meta and scatter_bases go together");
  if (has_meta) {
    TORCH_CHECK(scatter_meta->is_cuda() && scatter_meta->device() == a.device() && scatter_meta->scalar_type() == at::kLong &&
                    scatter_meta->is_contiguous() && scatter_meta->numel() >= m,
                "scatter_meta must be a contiguous int64 tensor on a's device with one entry per row of a");
    TORCH_CHECK(scatter_bases->is_cuda() && scatter_bases->device() == a.device() && scatter_bases->scalar_type() == at::kLong &&
                    scatter_bases->is_contiguous() && scatter_bases->numel() >= 1,
                "scatter_bases must be a contiguous int64 tensor of buffer addresses on a's device");
    desc.scatter_meta = static_cast<const int64_t*>(scatter_meta->data_ptr());
    desc.scatter_bases = static_cast<const int64_t*>(scatter_bases->data_ptr());
  }
  desc.num_sms = static_cast<int32_t>(num_sms > 0 ? num_sms : 0);   // 0: every SM, or the process-wide cap
  desc.timeout_ms = static_cast<uint32_t>(timeout_ms);
  desc.raw_dump = static_cast<int32_t*>(ptr_of(raw_dump));
  desc.alpha = static_cast<float>(alpha);
  desc.tile_config = static_cast<int32_t>(tile_config);
  desc.no_split = static_cast<int32_t>(no_split);
  if (stage.has_value() && stage->defined()) {
    TORCH_CHECK(stage->is_cuda() && stage->device() == a.device(), "stage must live on a's device");
    desc.stage = stage->data_ptr();
    desc.stage_bytes = static_cast<uint64_t>(stage->numel()) * stage->element_size();
    desc.stage_chunk_bytes = static_cast<uint64_t>(stage_chunk_bytes > 0 ? stage_chunk_bytes : 0);
  }

  int rc = AG_E_INVALID;
  {
    // device guard and launch in a scope of their own: a failure is raised after the guard has been released
    const c10::cuda::CUDAGuard guard(a.device());
    desc.stream = c10::cuda::getCurrentCUDAStream(a.device().index()).stream();
    switch (kind) {
      case 0: rc = ag_m_grouped_bf16_gemm_nt(&desc); break;
      case 1: rc = ag_m_grouped_fp8_gemm_nt(&desc); break;
      case 2: rc = ag_m_grouped_int8_gemm_nt(&desc); break;
      case 3: rc = ag_m_grouped_fp4_gemm_nt(&desc); break;
      case 4: rc = ag_m_grouped_fp8_ue8m0_gemm_nt(&desc); break;
      default: rc = AG_E_UNSUPPORTED; break;
    }
  }
  TORCH_CHECK(rc != AG_E_UNSUPPORTED || (kind >= 0 && kind <= 4), "asymgemm_b200: unknown kind ", kind);
  TORCH_CHECK(rc == AG_OK, "asymgemm_b200: ", ag_last_error(), " (code ", rc, ")");
}

// ---------------------------------------------------------------------------------------------- routing and combine gradient
// These allocate their outputs (and what workspace they need) through torch on the current stream, so that a captured
// graph owns them, and launch like the operator above.

// Uninitialised tensors from the caching allocator on the current stream, without the dispatcher's way there.
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}

// Several small outputs from one allocation, which takes the host less time than one each (five outputs: 3 us less). The tensors
// share its storage and are not views of one another.
class Pieces {
 public:
  explicit Pieces(const at::Tensor& like) : like_(like) {}
  // Room for another `numel` elements; pieces are numbered in the order of these calls.
  Pieces& add(int64_t numel, at::ScalarType type) {
    offset_[count_] = bytes_;
    numel_[count_] = numel;
    type_[count_++] = type;
    bytes_ += (numel * static_cast<int64_t>(c10::elementSize(type)) + 255) / 256 * 256;
    return *this;
  }
  void allocate() { base_ = empty({bytes_}, at::kByte, like_); }
  at::Tensor get(int i, at::IntArrayRef sizes) const {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base_.storage()), base_.key_set(), c10::scalarTypeToTypeMeta(type_[i]));
    t.unsafeGetTensorImpl()->set_storage_offset(offset_[i] / static_cast<int64_t>(c10::elementSize(type_[i])));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
    return t;
  }
  at::Tensor get(int i) const { return get(i, {numel_[i]}); }

 private:
  static constexpr int kMost = 6;
  const at::Tensor& like_;
  at::Tensor base_;
  int64_t offset_[kMost], numel_[kMost], bytes_ = 0;
  at::ScalarType type_[kMost];
  int count_ = 0;
};

void check_ok(int rc) { TORCH_CHECK(rc == AG_OK, "asymgemm_b200: ", ag_last_error(), " (code ", rc, ")"); }

// These operators have no forward-mode derivative (and are not recorded by autograd here): a tangent would be lost without a word.
void no_tangents(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* t : tensors)
    TORCH_CHECK(t == nullptr || !t->defined() || !t->_fw_grad(0).defined(), "asymgemm_b200: forward-mode derivatives are not supported here");
}
const at::Tensor* get(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }

int32_t type_code(at::ScalarType t, const char* name) {
  if (t == at::kBFloat16) return AG_T_BF16;
  if (t == at::kHalf) return AG_T_FP16;
  TORCH_CHECK(t == at::kFloat, name, " must be bfloat16, float16 or float32");
  return AG_T_FP32;
}

// 2-D, rows of consecutive elements, any distance between rows
void check_rows(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.dim() == 2, name, " must be a 2-D CUDA tensor");
  TORCH_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have consecutive elements in a row");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= t.size(1), name, " must not have overlapping rows");
}
// Rows that lie on one another (an expanded tensor) are copied out; everything else is taken as it is.
at::Tensor apart(const at::Tensor& t) {
  const bool expanded = t.dim() == 2 && t.size(0) > 1 && t.stride(0) < t.size(1) && (t.size(1) == 1 || t.stride(1) == 1);
  return expanded ? t.contiguous() : t;
}
OptTensor apart(const OptTensor& t) { return t.has_value() && t->defined() ? OptTensor(apart(*t)) : t; }
int64_t row_stride(const at::Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

void check_same_device(const OptTensor& t, const char* name, const at::Tensor& a, at::ScalarType type, int64_t numel) {
  if (!t.has_value() || !t->defined()) return;
  TORCH_CHECK(t->is_cuda() && t->device() == a.device(), name, " must live on the device of the call's first tensor");
  TORCH_CHECK(t->scalar_type() == type && t->is_contiguous() && t->numel() == numel, name, " must be a contiguous ", type, " tensor of ", numel,
              " elements");
}

std::tuple<at::Tensor, at::Tensor> route_topk(const at::Tensor& logits_in, int64_t top_k, int64_t scoring, const OptTensor& bias, int64_t groups,
                                              int64_t top_groups, bool group_max, bool renormalize, double scale, const OptTensor& rows_used) {
  no_tangents({&logits_in, get(bias)});
  const at::Tensor logits = apart(logits_in);
  check_rows(logits, "logits");
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  TORCH_CHECK(experts > 0 && experts <= 1024 && top_k > 0 && top_k <= 32, "route_topk wants 1 .. 1024 experts and top_k 1 .. 32");
  TORCH_CHECK(groups > 0 && groups <= 32 && top_groups > 0 && top_groups <= groups, "route_topk wants 1 .. 32 groups, of which 1 .. all take part");
  check_same_device(bias, "bias", logits, at::kFloat, experts);
  check_same_device(rows_used, "rows_used", logits, at::kInt, 1);
  ag_route_desc_t d{};
  d.dtype = type_code(logits.scalar_type(), "logits");
  const c10::cuda::CUDAGuard guard(logits.device());
  Pieces out(logits);
  out.add(tokens * top_k, at::kLong).add(tokens * top_k, at::kFloat).allocate();
  const at::Tensor ids = out.get(0, {tokens, top_k}), weights = out.get(1, {tokens, top_k});
  d.logits = logits.data_ptr();
  d.ld = row_stride(logits);
  d.bias = static_cast<const float*>(ptr_of(bias));
  d.rows_used = static_cast<const int32_t*>(ptr_of(rows_used));
  d.ids = static_cast<int64_t*>(ids.data_ptr());
  d.weights = static_cast<float*>(weights.data_ptr());
  d.tokens = tokens;
  d.experts = static_cast<int32_t>(experts);
  d.top_k = static_cast<int32_t>(top_k);
  d.groups = static_cast<int32_t>(groups);
  d.top_groups = static_cast<int32_t>(top_groups);
  d.scoring = static_cast<int32_t>(scoring);
  d.group_max = group_max;
  d.renormalize = renormalize;
  d.scale = static_cast<float>(scale);
  d.stream = c10::cuda::getCurrentCUDAStream(logits.device().index()).stream();
  check_ok(ag_route_topk(&d));
  return {ids, weights};
}

at::Tensor route_topk_backward(const at::Tensor& dweights, const at::Tensor& ids, const at::Tensor& logits_in, int64_t scoring, bool renormalize,
                               double scale) {
  no_tangents({&dweights, &logits_in});
  const at::Tensor logits = apart(logits_in);
  check_rows(logits, "logits");
  TORCH_CHECK(ids.dim() == 2 && ids.size(0) == logits.size(0) && ids.size(1) > 0 && ids.size(1) <= 32, "topk_ids must be [tokens, top_k], top_k 1 .. 32");
  TORCH_CHECK(dweights.sizes() == ids.sizes(), "dweights must have the shape of topk_ids");
  check_same_device(ids, "topk_ids", logits, at::kLong, ids.numel());
  check_same_device(dweights, "dweights", logits, at::kFloat, ids.numel());
  const int32_t type = type_code(logits.scalar_type(), "logits");
  const c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor dlogits = empty({logits.size(0), logits.size(1)}, logits.scalar_type(), logits);
  check_ok(ag_route_topk_backward(logits.data_ptr(), type, logits.size(0), row_stride(logits), static_cast<int32_t>(logits.size(1)),
                                  static_cast<const float*>(dweights.data_ptr()), static_cast<const int64_t*>(ids.data_ptr()),
                                  static_cast<int32_t>(ids.size(1)), static_cast<int32_t>(scoring), renormalize, static_cast<float>(scale),
                                  dlogits.data_ptr(), c10::cuda::getCurrentCUDAStream(logits.device().index()).stream()));
  return dlogits;
}

// Fills what both layouts share and launches.
void run_layout(ag_route_layout_desc_t& d, const at::Tensor& ids, int64_t experts, const at::Tensor& pair_row, const at::Tensor& row_token,
                const at::Tensor& status) {
  d.ids = ids.data_ptr();
  d.ids_64 = ids.scalar_type() == at::kLong;
  d.top_k = static_cast<int32_t>(ids.size(1));
  d.tokens = ids.size(0);
  d.experts = static_cast<int32_t>(experts);
  d.rows = row_token.numel();
  d.pair_row = static_cast<int64_t*>(pair_row.data_ptr());
  d.row_token = static_cast<int64_t*>(row_token.data_ptr());
  const uint64_t need = ag_route_layout_workspace_bytes(ids.numel(), static_cast<int32_t>(experts));
  at::Tensor workspace;
  if (need > 0) {
    workspace = empty({static_cast<int64_t>(need)}, at::kByte, ids);
    d.workspace = workspace.data_ptr();
    d.workspace_bytes = need;
  }
  d.status = static_cast<int32_t*>(status.data_ptr());
  d.stream = c10::cuda::getCurrentCUDAStream(ids.device().index()).stream();
  check_ok(ag_route_layout(&d));
}

void check_layout_args(const at::Tensor& ids, int64_t experts, const at::Tensor& status) {
  TORCH_CHECK(ids.is_cuda() && ids.dim() == 2 && ids.is_contiguous() && ids.size(1) > 0, "topk_ids must be a contiguous CUDA tensor [tokens, top_k]");
  TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "topk_ids must be int64 or int32");
  TORCH_CHECK(experts > 0 && experts <= 1024, "the layout tables are built for 1 .. 1024 experts");
  TORCH_CHECK(ids.numel() < (int64_t{1} << 30), "too many (token, slot) pairs");
  TORCH_CHECK(status.is_cuda() && status.device() == ids.device() && status.scalar_type() == at::kInt && status.numel() >= 1,
              "status must be an int32 tensor on the device of topk_ids");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> route_layout(const at::Tensor& ids, int64_t experts, int64_t alignment,
                                                                                    const at::Tensor& status) {
  check_layout_args(ids, experts, status);
  TORCH_CHECK(alignment > 0 && alignment <= 65536, "alignment must be 1 .. 65536");
  const int64_t pairs = ids.numel();
  const int64_t rows = pairs > 0 ? (pairs + alignment - 1) / alignment * alignment + experts * alignment : 0;
  const c10::cuda::CUDAGuard guard(ids.device());
  Pieces out(ids);
  out.add(pairs, at::kLong).add(rows, at::kLong).add(experts, at::kLong).add(2 * experts, at::kInt).add(experts + 1, at::kInt).allocate();
  const at::Tensor pair_row = out.get(0), row_token = out.get(1), rows_per_expert = out.get(2), offsets = out.get(3), expert_list = out.get(4);
  ag_route_layout_desc_t d{};
  d.alignment = static_cast<int32_t>(alignment);
  d.rows_per_expert = static_cast<int64_t*>(rows_per_expert.data_ptr());
  d.offsets = static_cast<int32_t*>(offsets.data_ptr());
  d.expert_list = static_cast<int32_t*>(expert_list.data_ptr());
  run_layout(d, ids, experts, pair_row, row_token, status);
  return {pair_row, row_token, rows_per_expert, offsets, expert_list};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> route_layout_masked(const at::Tensor& ids, int64_t experts, int64_t max_rows, const at::Tensor& status) {
  check_layout_args(ids, experts, status);
  TORCH_CHECK(max_rows > 0 && max_rows < (int64_t{1} << 31) / experts, "max_rows must be positive, and experts * max_rows below 2^31");
  const c10::cuda::CUDAGuard guard(ids.device());
  Pieces out(ids);
  out.add(ids.numel(), at::kLong).add(experts * max_rows, at::kLong).add(experts, at::kInt).allocate();
  const at::Tensor pair_row = out.get(0), row_token = out.get(1), masked_m = out.get(2);
  ag_route_layout_desc_t d{};
  d.max_rows = static_cast<int32_t>(max_rows);
  d.masked_m = static_cast<int32_t*>(masked_m.data_ptr());
  run_layout(d, ids, experts, pair_row, row_token, status);
  return {pair_row, row_token, masked_m};
}

std::tuple<at::Tensor, at::Tensor> combine_topk_backward(const at::Tensor& dy, const at::Tensor& rows, const OptTensor& pos, const at::Tensor& weights,
                                                         bool need_rows, bool need_weights, const at::Tensor& status) {
  no_tangents({&dy, &rows, &weights});
  TORCH_CHECK(dy.is_cuda() && dy.dim() == 2 && dy.is_contiguous() && dy.scalar_type() == at::kBFloat16, "dy must be a contiguous bf16 CUDA tensor [tokens, cols]");
  TORCH_CHECK(rows.is_cuda() && rows.device() == dy.device() && rows.dim() == 2 && rows.is_contiguous() && rows.size(1) == dy.size(1),
              "rows must be a contiguous tensor [num_rows, cols] on dy's device");
  TORCH_CHECK(rows.scalar_type() == at::kBFloat16 || rows.scalar_type() == at::kFloat, "rows must be bfloat16 or float32");
  TORCH_CHECK(weights.dim() == 2 && weights.size(0) == dy.size(0) && weights.size(1) > 0, "weights must be [tokens, top_k]");
  check_same_device(weights, "weights", dy, at::kFloat, weights.numel());
  check_same_device(pos, "pos", dy, at::kLong, weights.numel());
  TORCH_CHECK(status.is_cuda() && status.device() == dy.device() && status.scalar_type() == at::kInt && status.numel() >= 1,
              "status must be an int32 tensor on dy's device");
  const c10::cuda::CUDAGuard guard(dy.device());
  at::Tensor drows, dweights, seen;
  if (need_rows) {
    drows = empty(rows.sizes(), rows.scalar_type(), rows);
    seen = empty({(rows.size(0) + 3) / 4 * 4}, at::kByte, rows);
  }
  if (need_weights) dweights = empty(weights.sizes(), at::kFloat, weights);
  check_ok(ag_combine_topk_backward(dy.data_ptr(), rows.data_ptr(), rows.scalar_type() == at::kFloat, rows.size(0),
                                    static_cast<const int64_t*>(ptr_of(pos)), static_cast<const float*>(weights.data_ptr()), dy.size(0),
                                    static_cast<int32_t>(weights.size(1)), dy.size(1), need_rows ? drows.data_ptr() : nullptr,
                                    need_weights ? static_cast<float*>(dweights.data_ptr()) : nullptr, need_rows ? seen.data_ptr() : nullptr,
                                    static_cast<int32_t*>(status.data_ptr()), c10::cuda::getCurrentCUDAStream(dy.device().index()).stream()));
  return {drows, dweights};
}

// ---------------------------------------------------------------------------------------------- dense product
// Shapes, types and strides of x and weight; returns the descriptor with them filled in.
ag_linear_desc_t linear_desc(const at::Tensor& x, const at::Tensor& weight, int64_t activation, const at::Tensor& status, int64_t timeout_ms) {
  check_rows(x, "x");
  check_rows(weight, "weight");
  TORCH_CHECK(weight.device() == x.device(), "weight must live on x's device");
  TORCH_CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf, "x must be bfloat16 or float16");
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), "weight must be of x's type");
  TORCH_CHECK(weight.size(1) == x.size(1) && weight.size(0) > 0 && x.size(1) > 0, "x is [m, k] and weight [n, k], n and k positive");
  TORCH_CHECK(status.is_cuda() && status.device() == x.device() && status.scalar_type() == at::kInt && status.numel() >= 1,
              "status must be an int32 tensor on x's device");
  ag_linear_desc_t d{};
  d.dtype = type_code(x.scalar_type(), "x");
  d.activation = static_cast<int32_t>(activation);
  d.m = x.size(0);
  d.n = weight.size(0);
  d.k = x.size(1);
  d.x = x.data_ptr();
  d.weight = weight.data_ptr();
  d.ldx = row_stride(x);
  d.ldw = row_stride(weight);
  d.bias_dtype = d.dtype;
  d.status = static_cast<int32_t*>(status.data_ptr());
  d.timeout_ms = static_cast<uint32_t>(timeout_ms);
  return d;
}

at::Tensor linear_workspace(ag_linear_desc_t& d, const at::Tensor& x, bool backward) {
  at::Tensor workspace;
  const uint64_t need = ag_linear_workspace_bytes(&d, backward);
  if (need > 0) {
    workspace = empty({static_cast<int64_t>(need)}, at::kByte, x);
    d.workspace = workspace.data_ptr();
    d.workspace_bytes = need;
  }
  return workspace;
}

std::tuple<at::Tensor, at::Tensor> linear(const at::Tensor& x_in, const at::Tensor& weight_in, const OptTensor& bias, int64_t activation,
                                          const OptTensor& residual_in, bool out_fp32, bool keep_pre, const at::Tensor& status, int64_t timeout_ms) {
  no_tangents({&x_in, &weight_in, get(bias), get(residual_in)});
  const at::Tensor x = apart(x_in), weight = apart(weight_in);
  const OptTensor residual = apart(residual_in);
  ag_linear_desc_t d = linear_desc(x, weight, activation, status, timeout_ms);
  const at::ScalarType out_type = out_fp32 ? at::kFloat : x.scalar_type();
  d.out_dtype = type_code(out_type, "out");
  if (bias.has_value() && bias->defined()) {
    TORCH_CHECK(bias->is_cuda() && bias->device() == x.device() && bias->dim() == 1 && bias->size(0) == d.n && bias->is_contiguous() &&
                    (bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat),
                "bias must be a contiguous tensor [n] on x's device, of x's type or float32");
    d.bias = bias->data_ptr();
    d.bias_dtype = type_code(bias->scalar_type(), "bias");
  }
  if (residual.has_value() && residual->defined()) {
    check_rows(*residual, "residual");
    TORCH_CHECK(residual->device() == x.device() && residual->scalar_type() == out_type && residual->size(0) == d.m && residual->size(1) == d.n,
                "residual must be [m, n] on x's device, of the output's type");
    d.residual = residual->data_ptr();
    d.ldr = row_stride(*residual);
  }
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = empty({d.m, d.n}, out_type, x), pre;
  d.y = y.data_ptr();
  d.ldy = d.n;
  if (keep_pre) {
    pre = empty({d.m, d.n}, x.scalar_type(), x);
    d.pre = pre.data_ptr();
    d.ldp = d.n;
  }
  const at::Tensor workspace = linear_workspace(d, x, false);
  d.stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  check_ok(ag_linear(&d));
  return {y, pre};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_backward(const at::Tensor& dy_in, const at::Tensor& x_in, const at::Tensor& weight_in,
                                                               int64_t activation, const OptTensor& pre_in, bool need_x, bool need_weight, bool need_bias, bool bias_fp32,
                                                               const at::Tensor& status, int64_t timeout_ms) {
  no_tangents({&dy_in, &x_in, &weight_in, get(pre_in)});
  const at::Tensor dy = apart(dy_in), x = apart(x_in), weight = apart(weight_in);
  const OptTensor pre = apart(pre_in);
  ag_linear_desc_t d = linear_desc(x, weight, activation, status, timeout_ms);
  check_rows(dy, "dy");
  TORCH_CHECK(dy.device() == x.device() && dy.size(0) == d.m && dy.size(1) == d.n && (dy.scalar_type() == x.scalar_type() || dy.scalar_type() == at::kFloat),
              "dy must be [m, n] on x's device, of x's type or float32");
  d.out_dtype = type_code(dy.scalar_type(), "dy");
  d.dy = dy.data_ptr();
  d.lddy = row_stride(dy);
  if (pre.has_value() && pre->defined()) {
    check_rows(*pre, "pre");
    TORCH_CHECK(pre->device() == x.device() && pre->scalar_type() == x.scalar_type() && pre->size(0) == d.m && pre->size(1) == d.n,
                "pre must be [m, n] on x's device, of x's type");
    d.pre = pre->data_ptr();
    d.ldp = row_stride(*pre);
  }
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor dx, dweight, dbias, workspace;
  if (need_x) {
    dx = empty({d.m, d.k}, x.scalar_type(), x);
    d.dx = dx.data_ptr();
  }
  if (need_weight) {
    dweight = empty({d.n, d.k}, x.scalar_type(), x);
    d.dweight = dweight.data_ptr();
  }
  if (need_bias) {
    dbias = empty({d.n}, bias_fp32 ? at::kFloat : x.scalar_type(), x);
    d.bias_dtype = bias_fp32 ? AG_T_FP32 : d.dtype;
    d.dbias = dbias.data_ptr();
  }
  workspace = linear_workspace(d, x, true);
  d.stream = c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
  check_ok(ag_linear_backward(&d));
  return {dx, dweight, dbias};
}

}  // namespace

TORCH_LIBRARY(asymgemm_b200, m) {
  m.def(
      "linear(Tensor x, Tensor weight, Tensor? bias, int activation, Tensor? residual, bool out_fp32, bool keep_pre, Tensor status, int timeout_ms) "
      "-> (Tensor, Tensor)");
  m.def(
      "linear_backward(Tensor dy, Tensor x, Tensor weight, int activation, Tensor? pre, bool need_x, bool need_weight, bool need_bias, bool bias_fp32, "
      "Tensor status, int timeout_ms) -> (Tensor, Tensor, Tensor)");
  m.def(
      "route_topk(Tensor logits, int top_k, int scoring, Tensor? bias, int groups, int top_groups, bool group_max, bool renormalize, float scale, "
      "Tensor? rows_used) -> (Tensor, Tensor)");
  m.def("route_topk_backward(Tensor dweights, Tensor topk_ids, Tensor logits, int scoring, bool renormalize, float scale) -> Tensor");
  m.def("route_layout(Tensor topk_ids, int num_experts, int alignment, Tensor status) -> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def("route_layout_masked(Tensor topk_ids, int num_experts, int max_rows, Tensor status) -> (Tensor, Tensor, Tensor)");
  m.def(
      "combine_topk_backward(Tensor dy, Tensor rows, Tensor? pos, Tensor weights, bool need_rows, bool need_weights, Tensor status) -> (Tensor, Tensor)");
  m.def(
      "m_grouped_gemm_nt(int kind, int layout, Tensor a, Tensor? sfa, Tensor b, Tensor? sfb, Tensor(a!) d, Tensor? offsets, "
      "Tensor? experts, int max_segments, Tensor? masked_m, int m, int n, int k, int num_groups, Tensor? scratch, "
      "Tensor status, int timeout_ms, Tensor? raw_dump, float alpha, int tile_config, int no_split, Tensor? stage, int stage_chunk_bytes, "
      "int num_sms, int epilogue, Tensor? scatter_meta, Tensor? scatter_bases) -> ()");
}

TORCH_LIBRARY_IMPL(asymgemm_b200, CUDA, m) {
  m.impl("m_grouped_gemm_nt", &m_grouped_gemm_nt);
  m.impl("linear", &linear);
  m.impl("linear_backward", &linear_backward);
  m.impl("route_topk", &route_topk);
  m.impl("route_topk_backward", &route_topk_backward);
  m.impl("route_layout", &route_layout);
  m.impl("route_layout_masked", &route_layout_masked);
  m.impl("combine_topk_backward", &combine_topk_backward);
}
