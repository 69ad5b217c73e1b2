// PyTorch extension module over the C ABI of libops3d_fda.so: the tensor-level entry points of
// the reference's `_C` (csrc/vision.cpp:23-24 -> csrc/flash_deform_attn.h:7-52), plus the two
// calls FlashDeformAttnFunction makes (forward keeping the head-major copy of value, backward
// reusing it) and the offset-mode pair.  Host code only: argument checks, output allocation through torch's caching
// allocator, torch's current HIP stream, then one C ABI call.  It exists for host overhead --
// the same checks and calls through ctypes cost several times as much per call.
//
// Errors: a failed check or an OPS3D_FDA_EINVAL from the library raises ValueError
// (std::invalid_argument, as the reference's), OPS3D_FDA_ERUNTIME raises RuntimeError.
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

// torch's current HIP stream of a device (c10's native HIP API); the device is made current
// with HIP's own calls (DeviceGuard below)
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>

#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/ops3d_fda.h"
#include "../../include/ops3d_dcnv4.h"
#include "../../include/ops3d_linear.h"
#include "../../include/ops3d_nms3d.h"
#include "../../include/ops3d_roi_align3d.h"

namespace {

int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return OPS3D_FDA_F32;
    case at::kHalf: return OPS3D_FDA_F16;
    case at::kBFloat16: return OPS3D_FDA_BF16;
    default: throw std::invalid_argument(std::string("unsupported value dtype ") + c10::toString(t.scalar_type()));
  }
}

void check_tensor(const at::Tensor &t, const char *name, const at::Tensor &value) {
  // reference csrc/flash_deform_attn.h:24,51 (CPU tensors are not implemented)
  if (!t.is_cuda()) throw std::runtime_error(std::string("Not implemented on the CPU (") + name + " is on the CPU)");
  if (!t.is_contiguous()) throw std::runtime_error(std::string(name) + " tensor has to be contiguous");
  if (t.device() != value.device()) throw std::runtime_error(std::string(name) + " is on another device than value");
}

struct Sizes {
  int code, B, S, G, D, L, Q, K;
};

// Shared checks of every entry point; returns the problem sizes.
Sizes common(const at::Tensor &value, const at::Tensor &shapes, const at::Tensor &lsi, const at::Tensor &sla,
             int64_t K) {
  check_tensor(value, "value", value);
  check_tensor(shapes, "spatial_shapes", value);
  check_tensor(lsi, "level_start_index", value);
  check_tensor(sla, "sampling_loc_attn", value);
  Sizes z{};
  z.code = dtype_code(value);
  if (sla.scalar_type() != value.scalar_type())
    throw std::invalid_argument("sampling_loc_attn dtype differs from value dtype");
  if (shapes.scalar_type() != at::kLong || lsi.scalar_type() != at::kLong)
    throw std::invalid_argument("spatial_shapes and level_start_index must be int64");
  if (value.dim() != 4) throw std::invalid_argument("value must be [B, S, G, D]");
  if (shapes.dim() != 2 || shapes.size(1) != 3) throw std::invalid_argument("spatial_shapes must be [L, 3]");
  const int64_t L = shapes.size(0);
  if (lsi.dim() != 1 || lsi.size(0) != L) throw std::invalid_argument("level_start_index must be [L]");
  if (sla.dim() != 4 || sla.size(0) != value.size(0) || sla.size(2) != value.size(2))
    throw std::invalid_argument("sampling_loc_attn must be [B, Q, G, P]");
  if (sla.size(3) != L * K * 4)
    throw std::invalid_argument("sampling_loc_attn last dimension (" + std::to_string(sla.size(3)) +
                                ") does not match L=" + std::to_string(L) + ", K=" + std::to_string(K) +
                                " (expected " + std::to_string(L * K * 4) + ")");
  z.B = (int)value.size(0);
  z.S = (int)value.size(1);
  z.G = (int)value.size(2);
  z.D = (int)value.size(3);
  z.L = (int)L;
  z.Q = (int)sla.size(1);
  z.K = (int)K;
  return z;
}

void raise(int rc, const char *what) {
  const char *msg = ops3d_fda_last_error();
  const std::string m = (msg && *msg) ? msg : what;
  if (rc == OPS3D_FDA_EINVAL) throw std::invalid_argument(m);
  throw std::runtime_error(m);
}

hipStream_t stream_of(const at::Tensor &value) {
  return c10::hip::getCurrentHIPStream(value.device().index()).stream();
}

// Makes value's device current for the call and restores the previous one (the reference's
// entry points rely on the current device; torch's own guard types for ROCm label HIP devices
// as cuda, so plain HIP calls are used here).
class DeviceGuard {
 public:
  explicit DeviceGuard(const c10::Device &d) {
    if (hipGetDevice(&prev_) != hipSuccess) prev_ = -1;
    if (d.has_index() && d.index() != prev_ && hipSetDevice(d.index()) == hipSuccess) set_ = true;
  }
  ~DeviceGuard() {
    if (set_ && prev_ >= 0) (void)hipSetDevice(prev_);
  }
  DeviceGuard(const DeviceGuard &) = delete;
  DeviceGuard &operator=(const DeviceGuard &) = delete;

 private:
  int prev_ = -1;
  bool set_ = false;
};

void *ptr(const at::Tensor &t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

void check_grad_output(const at::Tensor &grad_output, const at::Tensor &value, const Sizes &z) {
  check_tensor(grad_output, "grad_output", value);
  if (grad_output.scalar_type() != value.scalar_type())
    throw std::invalid_argument("grad_output dtype differs from value dtype");
  if (grad_output.numel() != (int64_t)z.B * z.Q * z.G * z.D)
    throw std::invalid_argument("grad_output must have B*Q*G*D elements");
}

// Forward; returns the output and the forward workspace (the head-major copy of value), which
// is undefined (None) when the library makes no copy.
std::tuple<at::Tensor, c10::optional<at::Tensor>> forward_keep_head_major(
    const at::Tensor &value, const at::Tensor &shapes, const at::Tensor &lsi, const at::Tensor &sla,
    int64_t im2col_step, int64_t K) {
  const Sizes z = common(value, shapes, lsi, sla, K);
  const DeviceGuard guard(value.device());
  at::Tensor out = at::empty({z.B, z.Q, (int64_t)z.G * z.D}, value.options());
  const size_t n = ops3d_fda_forward_workspace_bytes(z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K);
  c10::optional<at::Tensor> ws;
  if (n) ws = at::empty({(int64_t)n}, value.options().dtype(at::kByte));
  const int rc = ops3d_fda_forward(ptr(value), shapes.data_ptr<int64_t>(), lsi.data_ptr<int64_t>(), ptr(sla),
                                   ptr(out), ws ? ws->data_ptr() : nullptr, n, z.code, z.B, z.S, z.G, z.D, z.L, z.Q,
                                   z.K, (int)im2col_step, stream_of(value));
  if (rc != OPS3D_FDA_OK) raise(rc, "flash_deform_attn_forward failed");
  return {out, ws};
}

// Backward; value_head_major: the forward workspace for this value, or None.
std::vector<at::Tensor> backward_with_head_major(const at::Tensor &value,
                                                 const c10::optional<at::Tensor> &value_head_major,
                                                 const at::Tensor &shapes, const at::Tensor &lsi,
                                                 const at::Tensor &sla, const at::Tensor &grad_output,
                                                 int64_t im2col_step, int64_t K) {
  const Sizes z = common(value, shapes, lsi, sla, K);
  check_grad_output(grad_output, value, z);
  const void *vhm = nullptr;
  if (value_head_major && value_head_major->defined()) {
    const at::Tensor &h = *value_head_major;
    const size_t need = ops3d_fda_forward_workspace_bytes(z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K);
    if (h.device() != value.device() || h.scalar_type() != at::kByte || (size_t)h.numel() != need)
      throw std::invalid_argument("value_head_major is not a forward workspace of this value");
    vhm = h.data_ptr();
  }
  const DeviceGuard guard(value.device());
  at::Tensor grad_value = at::empty_like(value);
  at::Tensor grad_sla = at::empty_like(sla);
  const size_t n = ops3d_fda_backward_workspace_bytes(z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K);
  at::Tensor ws;
  if (n) ws = at::empty({(int64_t)n}, value.options().dtype(at::kByte));
  const int rc = ops3d_fda_backward_ex(ptr(value), vhm, shapes.data_ptr<int64_t>(), lsi.data_ptr<int64_t>(),
                                       ptr(sla), ptr(grad_output), ptr(grad_value), ptr(grad_sla), ptr(ws), n,
                                       z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K, (int)im2col_step,
                                       stream_of(value));
  if (rc != OPS3D_FDA_OK) raise(rc, "flash_deform_attn_backward failed");
  return {grad_value, grad_sla};
}

// Offset mode: reference_points [B,Q,1 or L,3] fp32; returns ref_levels.
int ref_levels_of(const at::Tensor &ref, const at::Tensor &value, const Sizes &z) {
  check_tensor(ref, "reference_points", value);
  if (ref.scalar_type() != at::kFloat) throw std::invalid_argument("reference_points must be float32");
  if (ref.dim() != 4 || ref.size(0) != z.B || ref.size(1) != z.Q || ref.size(3) != 3 ||
      (ref.size(2) != 1 && ref.size(2) != z.L))
    throw std::invalid_argument("reference_points must be [B, Q, 1 or L, 3]");
  return (int)ref.size(2);
}

// Forward with offsets in voxels of their level in place of locations (ops3d_fda_forward_offsets).
std::tuple<at::Tensor, c10::optional<at::Tensor>> forward_offsets(
    const at::Tensor &value, const at::Tensor &shapes, const at::Tensor &lsi, const at::Tensor &offset_attn,
    const at::Tensor &reference_points, int64_t im2col_step, int64_t K) {
  const Sizes z = common(value, shapes, lsi, offset_attn, K);
  const int R = ref_levels_of(reference_points, value, z);
  const DeviceGuard guard(value.device());
  at::Tensor out = at::empty({z.B, z.Q, (int64_t)z.G * z.D}, value.options());
  const size_t n = ops3d_fda_forward_workspace_bytes(z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K);
  c10::optional<at::Tensor> ws;
  if (n) ws = at::empty({(int64_t)n}, value.options().dtype(at::kByte));
  const int rc = ops3d_fda_forward_offsets(ptr(value), shapes.data_ptr<int64_t>(), lsi.data_ptr<int64_t>(),
                                           ptr(offset_attn), reference_points.data_ptr<float>(), R, ptr(out),
                                           ws ? ws->data_ptr() : nullptr, n, z.code, z.B, z.S, z.G, z.D, z.L, z.Q,
                                           z.K, (int)im2col_step, stream_of(value));
  if (rc != OPS3D_FDA_OK) raise(rc, "flash_deform_attn_forward_offsets failed");
  return {out, ws};
}

// Backward of forward_offsets (ops3d_fda_backward_offsets): [grad_value, grad_offset_attn,
// grad_reference_points] (the last undefined -- None -- unless want_ref_grad).
std::vector<at::Tensor> backward_offsets(const at::Tensor &value, const c10::optional<at::Tensor> &value_head_major,
                                         const at::Tensor &shapes, const at::Tensor &lsi,
                                         const at::Tensor &offset_attn, const at::Tensor &reference_points,
                                         const at::Tensor &grad_output, int64_t im2col_step, int64_t K,
                                         bool want_ref_grad) {
  const Sizes z = common(value, shapes, lsi, offset_attn, K);
  check_grad_output(grad_output, value, z);
  const int R = ref_levels_of(reference_points, value, z);
  const void *vhm = nullptr;
  if (value_head_major && value_head_major->defined()) {
    const at::Tensor &h = *value_head_major;
    const size_t need = ops3d_fda_forward_workspace_bytes(z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K);
    if (h.device() != value.device() || h.scalar_type() != at::kByte || (size_t)h.numel() != need)
      throw std::invalid_argument("value_head_major is not a forward workspace of this value");
    vhm = h.data_ptr();
  }
  const DeviceGuard guard(value.device());
  at::Tensor grad_value = at::empty_like(value);
  at::Tensor grad_oa = at::empty_like(offset_attn);
  at::Tensor grad_ref;
  if (want_ref_grad) grad_ref = at::zeros_like(reference_points);
  const size_t n = ops3d_fda_backward_workspace_bytes(z.code, z.B, z.S, z.G, z.D, z.L, z.Q, z.K);
  at::Tensor ws;
  if (n) ws = at::empty({(int64_t)n}, value.options().dtype(at::kByte));
  const int rc = ops3d_fda_backward_offsets(ptr(value), vhm, shapes.data_ptr<int64_t>(), lsi.data_ptr<int64_t>(),
                                            ptr(offset_attn), reference_points.data_ptr<float>(), R, ptr(grad_output),
                                            ptr(grad_value), ptr(grad_oa),
                                            want_ref_grad ? grad_ref.data_ptr<float>() : nullptr, ptr(ws), n, z.code, z.B, z.S, z.G, z.D,
                                            z.L, z.Q, z.K, (int)im2col_step, stream_of(value));
  if (rc != OPS3D_FDA_OK) raise(rc, "flash_deform_attn_backward_offsets failed");
  return {grad_value, grad_oa, grad_ref};
}

// reference csrc/flash_deform_attn.h:7-25 (d_stride, block_thread and use_reg are launch hints
// of the CUDA build; the gfx950 library chooses its own geometry)
at::Tensor flash_deform_attn_forward(const at::Tensor &value, const at::Tensor &shapes, const at::Tensor &lsi,
                                     const at::Tensor &sla, int64_t im2col_step, int64_t K, int64_t /*d_stride*/,
                                     int64_t /*block_thread*/, bool /*use_reg*/) {
  return std::get<0>(forward_keep_head_major(value, shapes, lsi, sla, im2col_step, K));
}

// reference csrc/flash_deform_attn.h:27-52
std::vector<at::Tensor> flash_deform_attn_backward(const at::Tensor &value, const at::Tensor &shapes,
                                                   const at::Tensor &lsi, const at::Tensor &sla,
                                                   const at::Tensor &grad_output, int64_t im2col_step, int64_t K,
                                                   int64_t /*d_stride*/, int64_t /*block_thread*/) {
  return backward_with_head_major(value, c10::nullopt, shapes, lsi, sla, grad_output, im2col_step, K);
}

// reference csrc/nms_3d.h:27-44 -> nms_3d_cuda (csrc/cuda/nms_3d_cuda.cu:105-162): boxes [N,6]
// (x1,y1,z1,x2,y2,z2) and scores [N] on the GPU -> int64 indices of the kept boxes in
// decreasing score order.  Ties in score keep index order (a stable sort).  The kept count is
// read back to size the result (the reference synchronises too).
at::Tensor nms_3d(const at::Tensor &dets, const at::Tensor &scores, double threshold) {
  if (!dets.is_cuda()) throw std::runtime_error("Not compiled with CPU support");
  if (dets.numel() == 0) return at::empty({0}, dets.options().dtype(at::kLong));
  if (dets.dim() != 2 || dets.size(1) != 6) throw std::invalid_argument("dets must be [N, 6] (x1,y1,z1,x2,y2,z2)");
  if (scores.dim() != 1 || scores.size(0) != dets.size(0) || scores.device() != dets.device())
    throw std::invalid_argument("scores must be [N] on the boxes' device");
  const DeviceGuard guard(dets.device());
  const int64_t n64 = dets.size(0);
  if (n64 > INT32_MAX) throw std::invalid_argument("nms_3d: too many boxes (at most 2^19)");
  const int n = (int)n64;
  const float thr = (float)threshold;
  at::Tensor keep = at::empty({n}, dets.options().dtype(at::kLong));
  at::Tensor num = at::empty({1}, dets.options().dtype(at::kInt));
  at::Tensor order;
  const size_t wsb = ops3d_nms3d_workspace_bytes(n), pairs = thr >= 0.f ? ops3d_nms3d_pairs_workspace_bytes(n) : 0;
  const bool ranked = ops3d_nms3d_pairs_ranks(n) != 0;
  const auto sk = scores.scalar_type();
  int rc;
  if (pairs && (!ranked || sk == at::kFloat || sk == at::kHalf || sk == at::kBFloat16)) {
    // from the list of overlapping pairs; -1 when they are too many
    // (resolve_neg: the imaginary part of a conjugate is a view whose memory holds the negatives)
    const at::Tensor b = dets.to(at::kFloat).resolve_neg(), s = ranked ? scores.to(at::kFloat).resolve_neg() : scores;
    if (!ranked) order = std::get<1>(scores.sort(/*stable=*/true, /*dim=*/0, /*descending=*/true));
    const int64_t *ord = ranked ? nullptr : order.data_ptr<int64_t>();
    at::Tensor pws = at::empty({(int64_t)pairs}, dets.options().dtype(at::kByte));
    rc = ops3d_nms3d_pairs(b.data_ptr<float>(), b.stride(0), b.stride(1), ranked ? s.data_ptr<float>() : nullptr,
                           ranked ? s.stride(0) : 0, ord, n, thr, pws.data_ptr(), pairs, keep.data_ptr<int64_t>(),
                           num.data_ptr<int32_t>(), stream_of(dets));
    if (rc != OPS3D_FDA_OK) throw std::runtime_error("nms_3d: kernel launch failed");
    const int kept = num.item<int32_t>();
    if (kept >= 0) return keep.narrow(0, 0, kept);
    at::Tensor ws = at::empty({(int64_t)wsb}, dets.options().dtype(at::kByte));
    rc = ops3d_nms3d_after_pairs(pws.data_ptr(), pairs, ord, n, thr, ws.data_ptr(), wsb, keep.data_ptr<int64_t>(),
                                 num.data_ptr<int32_t>(), stream_of(dets));
  } else {
    order = std::get<1>(scores.sort(/*stable=*/true, /*dim=*/0, /*descending=*/true));
    const at::Tensor boxes = dets.index_select(0, order).to(at::kFloat).contiguous();
    at::Tensor ws = at::empty({(int64_t)wsb}, dets.options().dtype(at::kByte));
    rc = ops3d_nms3d(boxes.data_ptr<float>(), order.data_ptr<int64_t>(), n, thr, ws.data_ptr(), wsb,
                     keep.data_ptr<int64_t>(), num.data_ptr<int32_t>(), stream_of(dets));
  }
  if (rc == OPS3D_FDA_EINVAL) throw std::invalid_argument("nms_3d: too many boxes (at most 2^19)");
  if (rc != OPS3D_FDA_OK) throw std::runtime_error("nms_3d: kernel launch failed");
  return keep.narrow(0, 0, num.item<int32_t>());
}

// RoI Align 3-D (reference csrc/roi_align_3d.h:35-136): shared checks; returns the dtype code.
int roi_checks(const at::Tensor &data, const at::Tensor &rois, const at::Tensor &other) {
  if (!data.is_cuda()) throw std::runtime_error("RoIAlign is not implemented on CPU");
  if (rois.dim() != 2 || rois.size(1) != 7) throw std::runtime_error("wrong roi size! size_rois should be 7");
  for (const at::Tensor *t : {&rois, &other}) {
    if (t->device() != data.device()) throw std::runtime_error("RoIAlign tensors must be on one device");
    if (t->scalar_type() != data.scalar_type()) throw std::invalid_argument("RoIAlign tensors must share a dtype");
  }
  if (!other.is_contiguous()) throw std::runtime_error("RoIAlign output tensor has to be contiguous");
  return dtype_code(data);
}

// Features already in channels_last_3d memory ([N,D,H,W,C] order, 16-byte aligned).
bool is_channels_last_input(const at::Tensor &input) {
  return !input.is_contiguous() && input.is_contiguous(at::MemoryFormat::ChannelsLast3d) &&
         (reinterpret_cast<uintptr_t>(input.data_ptr()) & 15u) == 0;
}

// Whether the forward runs the channels-last kernel: always on channels-last input it supports;
// on [N,C,D,H,W] input when the output has at least kRoiClMinOutputs elements, so that the
// transposed copy of the features is repaid (below that the NCDHW kernel is as fast).
constexpr int64_t kRoiClMinOutputs = (int64_t)1 << 19;
bool roi_channels_last(const at::Tensor &input, int code, int R, int pd, int ph, int pw) {
  const int C = (int)input.size(1);
  if (!ops3d_roi_align3d_channels_last_supported(code, C, (int)input.size(2), (int)input.size(3),
                                                 (int)input.size(4), pw) ||
      input.size(0) > 65535)
    return false;
  return is_channels_last_input(input) || (int64_t)R * C * pd * ph * pw >= kRoiClMinOutputs;
}

void roi_align_3d_forward(const at::Tensor &input, const at::Tensor &rois, at::Tensor output, int64_t pd, int64_t ph,
                          int64_t pw, double spatial_scale, int64_t sampling_ratio, int64_t order) {
  const int code = roi_checks(input, rois, output);
  if (input.dim() != 5) throw std::invalid_argument("features must be [N, C, D, H, W]");
  const at::Tensor r = rois.contiguous();
  if (output.dim() != 5 || output.size(0) != r.size(0) || output.size(1) != input.size(1) || output.size(2) != pd ||
      output.size(3) != ph || output.size(4) != pw)
    throw std::invalid_argument("output must be [R, C, out_d, out_h, out_w]");
  const DeviceGuard guard(input.device());
  const int N = (int)input.size(0), C = (int)input.size(1), D = (int)input.size(2), H = (int)input.size(3),
            W = (int)input.size(4), R = (int)r.size(0);
  int rc;
  if (roi_channels_last(input, code, R, (int)pd, (int)ph, (int)pw)) {
    // channels-last kernel: on the caller's channels_last_3d memory, or on a transposed copy
    at::Tensor fc = input;
    if (!is_channels_last_input(input)) {
      const at::Tensor f = input.contiguous();
      fc = at::empty({N, D, H, W, C}, input.options());
      rc = ops3d_roi_align3d_to_channels_last(ptr(f), ptr(fc), code, N, C, D, H, W, stream_of(input));
      if (rc != OPS3D_FDA_OK) throw std::runtime_error("roi_align_3d_forward: channels-last copy failed");
    }
    rc = ops3d_roi_align3d_forward_channels_last(ptr(fc), ptr(r), ptr(output), code, N, C, D, H, W, R, (int)pd,
                                                 (int)ph, (int)pw, (float)spatial_scale, (int)sampling_ratio,
                                                 (int)order, stream_of(input));
  } else {
    const at::Tensor f = input.contiguous();
    rc = ops3d_roi_align3d_forward(ptr(f), ptr(r), ptr(output), code, N, C, D, H, W, R, (int)pd, (int)ph, (int)pw,
                                   (float)spatial_scale, (int)sampling_ratio, (int)order, stream_of(input));
  }
  if (rc == OPS3D_FDA_EINVAL) throw std::invalid_argument("roi_align_3d_forward: invalid sizes or order");
  if (rc != OPS3D_FDA_OK) throw std::runtime_error("roi_align_3d_forward: kernel launch failed");
}

void roi_align_3d_backward(const at::Tensor &top_grad, const at::Tensor &rois, at::Tensor bottom_grad, int64_t pd,
                           int64_t ph, int64_t pw, double spatial_scale, int64_t sampling_ratio, int64_t order) {
  const int code = roi_checks(top_grad, rois, bottom_grad);
  if (bottom_grad.dim() != 5) throw std::invalid_argument("bottom_grad must be [N, C, D, H, W]");
  const at::Tensor g = top_grad.contiguous(), r = rois.contiguous();
  const int N = (int)bottom_grad.size(0), C = (int)bottom_grad.size(1), D = (int)bottom_grad.size(2),
            H = (int)bottom_grad.size(3), W = (int)bottom_grad.size(4);
  if (g.dim() != 5 || g.size(0) != r.size(0) || g.size(1) != C || g.size(2) != pd || g.size(3) != ph ||
      g.size(4) != pw)
    throw std::invalid_argument("top_grad must be [R, C, out_d, out_h, out_w]");
  const DeviceGuard guard(top_grad.device());
  const size_t wsb =
      ops3d_roi_align3d_backward_workspace_bytes(code, N, C, D, H, W, (int)r.size(0), (int)pd, (int)ph, (int)pw);
  at::Tensor ws;
  if (wsb) ws = at::empty({(int64_t)((wsb + 3) / 4)}, top_grad.options().dtype(at::kFloat));
  const int rc = ops3d_roi_align3d_backward(ptr(g), ptr(r), ptr(bottom_grad), ptr(ws), wsb, code, N, C, D, H, W,
                                            (int)r.size(0), (int)pd, (int)ph, (int)pw, (float)spatial_scale,
                                            (int)sampling_ratio, (int)order, stream_of(top_grad));
  if (rc == OPS3D_FDA_EINVAL) throw std::invalid_argument("roi_align_3d_backward: invalid sizes or order");
  if (rc != OPS3D_FDA_OK) throw std::runtime_error("roi_align_3d_backward: kernel launch failed");
}

// DCNv4-3D (reference csrc/dcnv4.h:7-60): value [B,Din,Hin,Win,G*D], p_offset
// [B,Dout,Hout,Wout,padded]; d_stride and block_thread are launch hints of the CUDA build
// (accepted, not used).
struct DcnArgs {
  int B, Din, Hin, Win, code;
};

DcnArgs dcn_check(const at::Tensor &value, const at::Tensor &p_offset, int64_t group, int64_t group_channels) {
  if (!value.is_cuda()) throw std::runtime_error("Not implemented on the CPU");
  if (!p_offset.is_cuda()) throw std::runtime_error("offset must be a CUDA tensor");
  if (!value.is_contiguous()) throw std::runtime_error("input tensor has to be contiguous");
  if (!p_offset.is_contiguous()) throw std::runtime_error("offset tensor has to be contiguous");
  if (value.dim() != 5 || p_offset.dim() != 5) throw std::invalid_argument("value and p_offset must be 5-D");
  if (p_offset.scalar_type() != value.scalar_type()) throw std::invalid_argument("p_offset dtype differs from value");
  if (value.size(4) != group * group_channels)
    throw std::runtime_error("Input channels and group times group channels dont match");
  return {(int)value.size(0), (int)value.size(1), (int)value.size(2), (int)value.size(3), dtype_code(value)};
}

at::Tensor dcnv4_forward(const at::Tensor &value, const at::Tensor &p_offset, int64_t kd, int64_t kh, int64_t kw,
                         int64_t sd, int64_t sh, int64_t sw, int64_t pd, int64_t ph, int64_t pw, int64_t dd,
                         int64_t dh, int64_t dw, int64_t group, int64_t group_channels, double offset_scale,
                         int64_t im2col_step, int64_t remove_center, int64_t /*d_stride*/, int64_t /*block_thread*/,
                         bool softmax) {
  const DcnArgs z = dcn_check(value, p_offset, group, group_channels);
  const int Dout = (z.Din + 2 * (int)pd - ((int)dd * ((int)kd - 1) + 1)) / (int)sd + 1;
  const int Hout = (z.Hin + 2 * (int)ph - ((int)dh * ((int)kh - 1) + 1)) / (int)sh + 1;
  const int Wout = (z.Win + 2 * (int)pw - ((int)dw * ((int)kw - 1) + 1)) / (int)sw + 1;
  if (p_offset.size(0) != z.B || p_offset.size(1) != Dout || p_offset.size(2) != Hout || p_offset.size(3) != Wout)
    throw std::invalid_argument("p_offset must be [B, Dout, Hout, Wout, padded_offset_dim]");
  const DeviceGuard guard(value.device());
  at::Tensor out = at::empty({z.B, Dout, Hout, Wout, group * group_channels}, value.options());
  const size_t wsb = ops3d_dcnv4_workspace_bytes(z.code, z.B, z.Din, z.Hin, z.Win, (int)group, (int)group_channels,
                                                 (int)kd, (int)kh, (int)kw, (int)sd, (int)sh, (int)sw, (int)pd,
                                                 (int)ph, (int)pw, (int)dd, (int)dh, (int)dw, (int)remove_center, 0);
  at::Tensor ws = at::empty({(int64_t)(wsb ? wsb : 256)}, value.options().dtype(at::kByte));
  const int rc = ops3d_dcnv4_forward(ptr(value), ptr(p_offset), ptr(out), ws.data_ptr(), wsb, z.code, z.B, z.Din,
                                     z.Hin, z.Win, (int)group, (int)group_channels, (int)kd, (int)kh, (int)kw,
                                     (int)sd, (int)sh, (int)sw, (int)pd, (int)ph, (int)pw, (int)dd, (int)dh, (int)dw,
                                     (float)offset_scale, (int)remove_center, softmax ? 1 : 0,
                                     (int)p_offset.size(4), (int)im2col_step, stream_of(value));
  if (rc != OPS3D_FDA_OK) raise(rc, "dcnv4_forward failed");
  return out;
}

std::vector<at::Tensor> dcnv4_backward(const at::Tensor &value, const at::Tensor &p_offset, int64_t kd, int64_t kh,
                                       int64_t kw, int64_t sd, int64_t sh, int64_t sw, int64_t pd, int64_t ph,
                                       int64_t pw, int64_t dd, int64_t dh, int64_t dw, int64_t group,
                                       int64_t group_channels, double offset_scale, int64_t im2col_step,
                                       const at::Tensor &grad_output, int64_t remove_center,
                                       int64_t /*d_stride*/, int64_t /*block_thread*/, bool softmax) {
  const DcnArgs z = dcn_check(value, p_offset, group, group_channels);
  if (!grad_output.is_cuda() || !grad_output.is_contiguous() || grad_output.scalar_type() != value.scalar_type())
    throw std::runtime_error("grad_output tensor has to be a contiguous CUDA tensor of the value dtype");
  const DeviceGuard guard(value.device());
  at::Tensor grad_value = at::empty_like(value);
  // every unit's record is written; only a row padding has to be cleared
  const int64_t used = group * 4 * (kd * kh * kw - (remove_center ? 1 : 0));
  at::Tensor grad_offset = p_offset.size(4) == used ? at::empty_like(p_offset) : at::zeros_like(p_offset);
  const size_t wsb = ops3d_dcnv4_workspace_bytes(z.code, z.B, z.Din, z.Hin, z.Win, (int)group, (int)group_channels,
                                                 (int)kd, (int)kh, (int)kw, (int)sd, (int)sh, (int)sw, (int)pd,
                                                 (int)ph, (int)pw, (int)dd, (int)dh, (int)dw, (int)remove_center, 1);
  at::Tensor ws = at::empty({(int64_t)(wsb ? wsb : 256)}, value.options().dtype(at::kByte));
  const int rc = ops3d_dcnv4_backward(ptr(value), ptr(p_offset), ptr(grad_output), ptr(grad_value), ptr(grad_offset),
                                      ws.data_ptr(), wsb, z.code, z.B, z.Din, z.Hin, z.Win, (int)group,
                                      (int)group_channels, (int)kd, (int)kh, (int)kw, (int)sd, (int)sh, (int)sw,
                                      (int)pd, (int)ph, (int)pw, (int)dd, (int)dh, (int)dw, (float)offset_scale,
                                      (int)remove_center, softmax ? 1 : 0, (int)p_offset.size(4), (int)im2col_step,
                                      stream_of(value));
  if (rc != OPS3D_FDA_OK) raise(rc, "dcnv4_backward failed");
  return {grad_value, grad_offset};
}

// Linear operators (include/ops3d_linear.h).  Tensors may have any row distance; what cannot be seen
// as rows of consecutive elements is copied.
const at::Tensor &linear_check(const at::Tensor &t, const char *name, const at::Tensor &x) {
  if (!t.is_cuda()) throw std::runtime_error(std::string("Not implemented on the CPU (") + name + " is on the CPU)");
  if (t.layout() != at::kStrided) throw std::invalid_argument(std::string(name) + " must be a dense tensor");
  if (t.device() != x.device()) throw std::runtime_error(std::string(name) + " is on another device than x");
  if (t.scalar_type() != x.scalar_type())
    throw std::invalid_argument(std::string(name) + " dtype differs from x dtype");
  return t;
}

// t as rows of its last axis, `ld` elements apart; a copy where it is not.
at::Tensor as_rows(const at::Tensor &t_, int64_t &ld) {
  at::Tensor t = t_.is_neg() ? t_.resolve_neg() : t_;
  const int64_t d = t.dim(), n = t.size(d - 1);
  bool rows = t.stride(d - 1) == 1 || n == 1;
  int64_t step = -1, count = 1;   // of the axes seen so far, from the last but one outwards
  for (int64_t i = d - 2; i >= 0 && rows; --i) {
    if (t.size(i) == 1) continue;
    if (step < 0) step = t.stride(i);
    else rows = t.stride(i) == step * count;
    count *= t.size(i);
  }
  if (!rows) {
    ld = n;
    return t.contiguous();
  }
  ld = step < 0 ? n : step;
  return t;
}

at::Tensor dense(const at::Tensor &t) { return (t.is_neg() ? t.resolve_neg() : t).contiguous(); }

struct LinearSizes {
  int code, batch, groups, N, K;
  int64_t rows;
  const int64_t *start;
  int count;
};

int linear_int(int64_t v, const char *what) {
  if (v < 0 || v > 0x7fffffff) throw std::invalid_argument(std::string(what) + " is too large");
  return (int)v;
}

// rows: x or grad_y, whose last axis is not looked at; groups 0: one weight.
LinearSizes linear_sizes(const at::Tensor &rows, const c10::optional<at::Tensor> &group_start, int64_t groups, int64_t N,
                         int64_t K) {
  LinearSizes z{};
  z.code = dtype_code(rows);
  z.N = linear_int(N, "out_features");
  z.K = linear_int(K, "in_features");
  if (!group_start) {
    int64_t n = 1;
    for (int64_t i = 0; i + 1 < rows.dim(); ++i) n *= rows.size(i);
    z.batch = z.groups = 1;
    z.rows = n;
    return z;
  }
  const at::Tensor &g = *group_start;
  if (!g.is_cuda()) throw std::runtime_error("Not implemented on the CPU (group_start is on the CPU)");
  if (g.device() != rows.device()) throw std::runtime_error("group_start is on another device than x");
  if (g.scalar_type() != at::kLong || g.dim() != 1 || !g.is_contiguous())
    throw std::invalid_argument("group_start must be a contiguous int64 tensor of one axis");
  z.groups = linear_int(groups, "the number of groups");
  if (g.size(0) != groups && g.size(0) != groups + 1)
    throw std::invalid_argument("group_start must have " + std::to_string(groups) + " or " + std::to_string(groups + 1) +
                                " entries, got " + std::to_string(g.size(0)));
  z.count = (int)g.size(0);
  z.start = g.data_ptr<int64_t>();
  z.batch = rows.dim() == 3 ? linear_int(rows.size(0), "the batch") : 1;
  z.rows = rows.size(rows.dim() - 2);
  return z;
}

// [y, act_grad]; act_grad (None without an activation) when keep.
std::tuple<at::Tensor, c10::optional<at::Tensor>> linear_forward(
    const at::Tensor &x, const at::Tensor &weight, const c10::optional<at::Tensor> &bias,
    const c10::optional<at::Tensor> &residual, const c10::optional<at::Tensor> &group_start, int64_t act, bool keep) {
  linear_check(x, "x", x);
  linear_check(weight, "weight", x);
  const bool grouped = group_start.has_value();
  if (grouped ? weight.dim() != 3 : weight.dim() != 2)
    throw std::invalid_argument(grouped ? "weight must be [groups, out_features, in_features]"
                                        : "weight must be [out_features, in_features]");
  const int64_t N = weight.size(-2), K = weight.size(-1);
  if (grouped ? x.dim() != 2 && x.dim() != 3 : x.dim() < 1)
    throw std::invalid_argument("x must be [rows, in_features] or [batch, rows, in_features]");
  if (x.size(-1) != K)
    throw std::invalid_argument("x has " + std::to_string(x.size(-1)) + " features, weight " + std::to_string(K));
  if (bias) {
    linear_check(*bias, "bias", x);
    if (grouped ? bias->dim() != 2 || bias->size(0) != weight.size(0) || bias->size(1) != N
                : bias->dim() != 1 || bias->size(0) != N)
      throw std::invalid_argument(grouped ? "bias must be [groups, out_features]" : "bias must be [out_features]");
  }
  auto shape = x.sizes().vec();
  shape.back() = N;
  if (residual) {
    linear_check(*residual, "residual", x);
    if (residual->sizes().vec() != shape) throw std::invalid_argument("residual must have the output's shape");
  }
  const LinearSizes z = linear_sizes(x, group_start, grouped ? weight.size(0) : 0, N, K);
  const DeviceGuard guard(x.device());
  int64_t ldx = 0, ldr = 0;
  const at::Tensor xr = as_rows(x, ldx), w = dense(weight);
  const at::Tensor b = bias ? dense(*bias) : at::Tensor(), r = residual ? as_rows(*residual, ldr) : at::Tensor();
  at::Tensor y = at::empty(shape, x.options());
  c10::optional<at::Tensor> act_grad;
  if (keep && act != OPS3D_LINEAR_ACT_NONE)
    act_grad = at::empty(shape, x.scalar_type() == at::kFloat ? x.options() : x.options().dtype(at::kShort));
  const size_t n = ops3d_linear_forward_workspace_bytes(z.code, z.batch, z.rows, z.groups, z.N, z.K, grouped);
  at::Tensor ws;
  if (n) ws = at::empty({(int64_t)n}, x.options().dtype(at::kByte));
  const int rc = ops3d_linear_forward(ptr(xr), ldx, ptr(w), ptr(b), ptr(r), ldr, z.start, z.count, ptr(y),
                                      act_grad ? ptr(*act_grad) : nullptr, ptr(ws), n, z.code, (int)act, z.batch, z.rows,
                                      z.groups, z.N, z.K, stream_of(x));
  if (rc != OPS3D_FDA_OK) raise(rc, "linear_forward failed");
  return {y, act_grad};
}

// [grad_x (with weight), grad_weight, grad_bias], None where not wanted.  groups 0: one weight.
std::tuple<c10::optional<at::Tensor>, c10::optional<at::Tensor>, c10::optional<at::Tensor>> linear_backward(
    const c10::optional<at::Tensor> &x, const c10::optional<at::Tensor> &weight,
    const c10::optional<at::Tensor> &group_start, const c10::optional<at::Tensor> &act_grad, const at::Tensor &grad_y,
    int64_t in_features, int64_t groups, bool need_w, bool need_b) {
  linear_check(grad_y, "grad_output", grad_y);
  const bool grouped = group_start.has_value();
  if (grouped ? grad_y.dim() != 2 && grad_y.dim() != 3 : grad_y.dim() < 1)
    throw std::invalid_argument("grad_output must be [rows, out_features] or [batch, rows, out_features]");
  const int64_t N = grad_y.size(-1), K = in_features;
  auto shape = grad_y.sizes().vec();
  shape.back() = K;
  if ((need_w || need_b) && !x) throw std::invalid_argument("x is needed for the gradients of weight and bias");
  if (x) {
    linear_check(*x, "x", grad_y);
    if (x->sizes().vec() != shape) throw std::invalid_argument("x and grad_output differ in their rows");
  }
  const std::vector<int64_t> wshape = grouped ? std::vector<int64_t>{groups, N, K} : std::vector<int64_t>{N, K};
  if (weight) {
    linear_check(*weight, "weight", grad_y);
    if (weight->sizes().vec() != wshape) throw std::invalid_argument("weight does not fit grad_output");
  }
  if (act_grad && (!act_grad->is_cuda() || act_grad->device() != grad_y.device() || !act_grad->is_contiguous() ||
                   act_grad->sizes() != grad_y.sizes() ||
                   act_grad->scalar_type() != (grad_y.scalar_type() == at::kFloat ? at::kFloat : at::kShort)))
    throw std::invalid_argument("act_grad is not a forward's of this shape");
  const LinearSizes z = linear_sizes(grad_y, group_start, groups, N, K);
  const DeviceGuard guard(grad_y.device());
  int64_t ldx = 0, ldg = 0;
  const at::Tensor g = as_rows(grad_y, ldg), xr = x ? as_rows(*x, ldx) : at::Tensor();
  const at::Tensor w = weight ? dense(*weight) : at::Tensor();
  c10::optional<at::Tensor> gx, gw, gb;
  if (weight) gx = at::empty(shape, grad_y.options());
  if (need_w) gw = at::empty(wshape, grad_y.options());
  if (need_b) gb = at::empty(grouped ? std::vector<int64_t>{groups, N} : std::vector<int64_t>{N}, grad_y.options());
  const int want = (gx ? OPS3D_LINEAR_WANT_X : 0) | (gw ? OPS3D_LINEAR_WANT_WEIGHT : 0) | (gb ? OPS3D_LINEAR_WANT_BIAS : 0);
  const size_t n = ops3d_linear_backward_workspace_bytes_for(z.code, z.batch, z.rows, z.groups, z.N, z.K, grouped,
                                                             act_grad.has_value(), want);
  at::Tensor ws;
  if (n) ws = at::empty({(int64_t)n}, grad_y.options().dtype(at::kByte));
  const int rc = ops3d_linear_backward(ptr(xr), ldx, ptr(w), z.start, z.count, act_grad ? ptr(*act_grad) : nullptr, ptr(g),
                                       ldg, gx ? ptr(*gx) : nullptr, gw ? ptr(*gw) : nullptr, gb ? ptr(*gb) : nullptr,
                                       ptr(ws), n, z.code, z.batch, z.rows, z.groups, z.N, z.K, stream_of(grad_y));
  if (rc != OPS3D_FDA_OK) raise(rc, "linear_backward failed");
  return {gx, gw, gb};
}

// t with zeros in rows of no group.
at::Tensor keep_rows(const at::Tensor &t, const at::Tensor &group_start, int64_t groups) {
  linear_check(t, "the rows", t);
  if (t.dim() != 2 && t.dim() != 3)
    throw std::invalid_argument("the rows must be [rows, features] or [batch, rows, features]");
  const LinearSizes z = linear_sizes(t, group_start, groups, t.size(-1), 1);
  const DeviceGuard guard(t.device());
  int64_t ld = 0;
  const at::Tensor rows = as_rows(t, ld);
  at::Tensor out = at::empty(t.sizes(), t.options());
  const int rc = ops3d_linear_keep_rows(ptr(rows), ld, z.start, z.count, ptr(out), z.code, z.batch, z.rows, z.groups, z.N,
                                        stream_of(t));
  if (rc != OPS3D_FDA_OK) raise(rc, "linear_keep_rows failed");
  return out;
}

// The same through autograd; it is its own gradient.
class KeepRowsNode : public torch::autograd::Function<KeepRowsNode> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &t, const at::Tensor &group_start,
                            int64_t groups) {
    ctx->save_for_backward({group_start});
    ctx->saved_data["groups"] = groups;
    return keep_rows(t, group_start, groups);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    return {KeepRowsNode::apply(grads[0], ctx->get_saved_variables()[0], ctx->saved_data["groups"].toInt()), at::Tensor(),
            at::Tensor()};
  }
};

at::Tensor linear_keep_rows(const at::Tensor &t, const at::Tensor &group_start, int64_t groups) {
  return KeepRowsNode::apply(t, group_start, groups);
}

// The operator with its autograd node here: a training step on a small crop is bound by host time, of
// which a node in Python costs several times as much.  Once differentiable: with create_graph the
// gradients that are no constants raise when they are differentiated (a residual's may be).
class LinearNode : public torch::autograd::Function<LinearNode> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, const at::Tensor &weight,
                            const c10::optional<at::Tensor> &bias, const c10::optional<at::Tensor> &residual,
                            const c10::optional<at::Tensor> &group_start, int64_t act) {
    const bool need_x = x.requires_grad(), need_w = weight.requires_grad(), need_b = bias && bias->requires_grad();
    auto [y, act_grad] = linear_forward(x, weight, bias, residual, group_start, act, need_x || need_w || need_b);
    ctx->save_for_backward({need_w || need_b ? x : at::Tensor(), need_x ? weight : at::Tensor(),
                            group_start ? *group_start : at::Tensor(), act_grad ? *act_grad : at::Tensor()});
    ctx->saved_data["sizes"] = std::vector<int64_t>{weight.size(-1), weight.dim() == 3 ? weight.size(0) : 0, need_x,
                                                    need_w, need_b, residual && residual->requires_grad(), bias.has_value()};
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto sizes = ctx->saved_data["sizes"].toIntVector();
    const at::Tensor &grad = grads[0];
    torch::autograd::variable_list out(6);
    const auto some = [](const at::Tensor &t) { return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt; };
    {
      const at::NoGradGuard no_grad;
      // of the gradients that could be, those that this pass asks for
      const bool x = sizes[2] && ctx->needs_input_grad(0), w = sizes[3] && ctx->needs_input_grad(1),
                 b = sizes[4] && ctx->needs_input_grad(2);
      if (x || w || b) {
        auto [gx, gw, gb] = linear_backward(some(saved[0]), x ? some(saved[1]) : c10::nullopt, some(saved[2]), some(saved[3]),
                                            grad, sizes[0], sizes[1], w, b);
        if (gx) out[0] = *gx;
        if (gw) out[1] = *gw;
        if (gb) out[2] = *gb;
      }
    }
    if (sizes[5] && ctx->needs_input_grad(sizes[6] ? 3 : 2))   // y is 0 in rows of no group
      out[3] = saved[2].defined() ? linear_keep_rows(grad, saved[2], sizes[1]) : grad;
    if (at::GradMode::is_enabled()) {   // each that depends on something with a gradient
      const bool act = saved[3].defined(), depends[3] = {sizes[3] || act, sizes[2] || act, act};
      for (int i = 0; i < 3; ++i) {
        if (!out[i].defined() || !(depends[i] || grad.requires_grad())) continue;
        const auto error = std::make_shared<torch::autograd::DelayedError>(
            "trying to differentiate twice a linear operator that is differentiable once", 1);
        out[i] = (*error)({out[i].detach().set_requires_grad(true)})[0];
      }
    }
    return out;
  }
};

// A tangent would be lost without a word: y comes from a kernel that knows of none.
void refuse_tangent(const at::Tensor &t) {
  if (t.defined() && t._fw_grad(0).defined())
    throw std::runtime_error("the linear operators have no forward-mode derivatives");
}

at::Tensor linear(const at::Tensor &x, const at::Tensor &weight, const c10::optional<at::Tensor> &bias,
                  const c10::optional<at::Tensor> &residual, const c10::optional<at::Tensor> &group_start, int64_t act) {
  if (torch::jit::tracer::isTracing())   // a trace would record y's allocation without the kernel that fills it
    throw std::runtime_error("the linear operators cannot be traced");
  refuse_tangent(x);
  refuse_tangent(weight);
  if (bias) refuse_tangent(*bias);
  if (residual) refuse_tangent(*residual);
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()) ||
                                     (residual && residual->requires_grad())))
    return LinearNode::apply(x, weight, bias, residual, group_start, act);
  return std::get<0>(linear_forward(x, weight, bias, residual, group_start, act, false));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("flash_deform_attn_forward", &flash_deform_attn_forward, "flash_deform_attn_forward",
        py::arg("value"), py::arg("spatial_shapes"), py::arg("level_start_index"), py::arg("sampling_loc_attn"),
        py::arg("im2col_step"), py::arg("K"), py::arg("d_stride") = 8, py::arg("block_thread") = 0,
        py::arg("use_reg") = true);
  m.def("flash_deform_attn_backward", &flash_deform_attn_backward, "flash_deform_attn_backward",
        py::arg("value"), py::arg("spatial_shapes"), py::arg("level_start_index"), py::arg("sampling_loc_attn"),
        py::arg("grad_output"), py::arg("im2col_step"), py::arg("K"), py::arg("d_stride") = 1,
        py::arg("block_thread") = 0);
  m.def("forward_keep_head_major", &forward_keep_head_major, "forward that also returns its workspace");
  m.def("backward_with_head_major", &backward_with_head_major, "backward reusing the forward workspace");
  m.def("forward_offsets", &forward_offsets, "forward from offsets and reference points");
  m.def("backward_offsets", &backward_offsets, "backward of forward_offsets");
  m.def("nms_3d", &nms_3d, "non-maximum suppression for 3d");
  m.def("dcnv4_forward", &dcnv4_forward, "dcnv4_forward");
  m.def("dcnv4_backward", &dcnv4_backward, "dcnv4_backward");
  m.def("linear_forward", &linear_forward, "act(x W^T + b) + residual, one weight or one per group of rows");
  m.def("linear", &linear, "linear_forward with its gradients through autograd");
  m.def("linear_backward", &linear_backward, "gradients of linear_forward");
  m.def("linear_keep_rows", &linear_keep_rows, "zeros in rows of no group");
  m.def("roi_align_3d_forward", &roi_align_3d_forward, "roi_align_3d_forward");
  m.def("roi_align_3d_backward", &roi_align_3d_backward, "roi_align_3d_backward");
}
