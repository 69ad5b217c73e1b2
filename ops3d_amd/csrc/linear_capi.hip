// C entry points of the linear operators (include/ops3d_linear.h).
#include "linear_kernels.h"

#include <stdarg.h>
#include <stdio.h>

#include "../../include/ops3d_linear.h"

namespace ops3d_fda {
int set_last_error(int code, const char *text);   // fda_capi.hip
}

namespace {

using namespace ops3d_linear;

int fail(int code, const char *fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return ops3d_fda::set_last_error(code, buf);
}

int elem_size(int dtype) {
  return dtype == OPS3D_FDA_F32 ? 4 : dtype == OPS3D_FDA_F16 || dtype == OPS3D_FDA_BF16 ? 2 : 0;
}

constexpr int64_t kMaxRows = 0x7fffffff - 4096;   // rows of all items and tile counts stay 32-bit
constexpr int kMaxFeatures = 1 << 24;
constexpr int kWantAll = OPS3D_LINEAR_WANT_X | OPS3D_LINEAR_WANT_WEIGHT | OPS3D_LINEAR_WANT_BIAS;

int check_sizes(int dtype, int batch, int64_t rows, int groups, int out_features, int in_features) {
  if (elem_size(dtype) == 0) return fail(OPS3D_FDA_EINVAL, "unsupported dtype code %d", dtype);
  if (batch < 0 || rows < 0 || (batch > 0 && rows > kMaxRows / batch))
    return fail(OPS3D_FDA_EINVAL, "invalid or too many rows: %d items of %lld", batch, (long long)rows);
  if (out_features < 1 || in_features < 1 || out_features > kMaxFeatures || in_features > kMaxFeatures)
    return fail(OPS3D_FDA_EINVAL, "out_features and in_features must be in 1..%d, got %d and %d", kMaxFeatures, out_features,
                in_features);
  if (groups < 1 || groups > OPS3D_LINEAR_MAX_GROUPS)
    return fail(OPS3D_FDA_EINVAL, "groups must be in 1..%d, got %d", OPS3D_LINEAR_MAX_GROUPS, groups);
  // every segment may end inside a tile of 16 rows or a chunk
  if ((int64_t)batch * (groups + 2) + (int64_t)batch * rows / 16 > kMaxRows)
    return fail(OPS3D_FDA_EINVAL, "too many groups for %d items", batch);
  return OPS3D_FDA_OK;
}

int make_groups(const int64_t *start, int count, int batch, int64_t rows, int groups, Groups &g) {
  if (!start) {
    if (groups != 1) return fail(OPS3D_FDA_EINVAL, "group_start is NULL but there are %d groups", groups);
    g = Groups{nullptr, 0, 1, 1, (int)(batch * rows)};
    return OPS3D_FDA_OK;
  }
  if (count != groups && count != groups + 1)
    return fail(OPS3D_FDA_EINVAL, "group_start must have groups or groups + 1 entries (%d), got %d", groups, count);
  if (reinterpret_cast<uintptr_t>(start) & 7u) return fail(OPS3D_FDA_EINVAL, "group_start must be 8-byte aligned");
  g = Groups{start, count, groups, batch, (int)rows};
  return OPS3D_FDA_OK;
}

// The plan of the weights' gradients; batch and rows as the caller gave them.
ChunkPlan plan_of(int dtype, bool grouped, int batch, int64_t rows, int groups, int N, int K) {
  return grouped ? ChunkPlan(elem_size(dtype), true, batch, rows, groups, N, K)
                 : ChunkPlan(elem_size(dtype), false, 1, batch * rows, 1, N, K);
}

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

bool sizes_ok(int dtype, int batch, int64_t rows, int groups, int N, int K, bool grouped) {
  return elem_size(dtype) != 0 && batch >= 1 && rows >= 1 && rows <= kMaxRows / batch && groups >= 1 &&
         groups <= OPS3D_LINEAR_MAX_GROUPS && N >= 1 && K >= 1 && N <= kMaxFeatures && K <= kMaxFeatures &&
         (grouped || groups == 1);
}

// Bytes of the parts of a rows kernel's split sums.
size_t split_bytes(int dtype, int64_t rows, int groups, int N, int K) {
  const int n = split_count(elem_size(dtype), rows, groups, N, K);
  return n > 1 ? align256((size_t)n * rows * N * 4) : 0;
}
void set_split(RowsArgs &p, bool on, void *part, int dtype, int64_t rows, int groups) {
  p.rows = rows;
  p.splits = 1;
  if (!on) return;
  const int kc = 128 / elem_size(dtype);
  p.splits = split_count(elem_size(dtype), rows, groups, p.N, p.K);
  p.per_split = ceil_div(ceil_div(p.K, kc), p.splits) * kc;
  p.part = static_cast<float *>(part);
}

int check_workspace(const void *workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need))
    return fail(OPS3D_FDA_EINVAL, "workspace too small: %zu bytes given, %zu needed", bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(OPS3D_FDA_EINVAL, "workspace must be 256-byte aligned");
  return OPS3D_FDA_OK;
}

// Workspace of the backward, of what is wanted: dz (behind an activation), then the parts of the input gradient's split
// sums and, after it and in the same place, the chunks' partial sums.
struct Layout {
  ChunkPlan plan;
  size_t dz, part, part_b, split, bytes;
  Layout(int dtype, bool grouped, int batch, int64_t rows, int groups, int N, int K, bool act_grad, int want)
      : plan(plan_of(dtype, grouped, batch, rows, groups, N, K)) {
    const bool x = want & OPS3D_LINEAR_WANT_X, w = want & OPS3D_LINEAR_WANT_WEIGHT, b = want & OPS3D_LINEAR_WANT_BIAS;
    dz = 0;
    part = act_grad && (w || b) ? align256((size_t)batch * rows * N * elem_size(dtype)) : 0;
    part_b = part + (plan.joined && w ? align256((size_t)plan.slots * N * K * 4) : 0);
    bytes = part_b + (plan.joined && b ? align256((size_t)plan.slots * N * 4) : 0);
    split = x && rows > 0 && batch > 0 ? split_bytes(dtype, batch * rows, groups, K, N) : 0;
    if (bytes < part + split) bytes = part + split;
  }
};

template <typename F> int run(int dtype, const char *what, F f) {
  hipError_t e = dtype == OPS3D_FDA_F32 ? f(float()) : dtype == OPS3D_FDA_F16 ? f(_Float16()) : f(__bf16());
  if (e == hipSuccess) return OPS3D_FDA_OK;
  if (e == hipErrorInvalidConfiguration) return fail(OPS3D_FDA_EINVAL, "%s: 2^31 tiles or more", what);
  return fail(OPS3D_FDA_ERUNTIME, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
}

bool misaligned(const void *p, int esize) { return reinterpret_cast<uintptr_t>(p) & (uintptr_t)(esize - 1); }

}  // namespace

extern "C" {

size_t ops3d_linear_forward_workspace_bytes(int dtype, int batch, int64_t rows, int groups, int out_features,
                                            int in_features, int grouped) {
  if (!sizes_ok(dtype, batch, rows, groups, out_features, in_features, grouped != 0) || batch * rows / groups <= kFewRows)
    return 0;
  return split_bytes(dtype, batch * rows, groups, out_features, in_features);
}

int ops3d_linear_forward(const void *x, int64_t ld_x, const void *weight, const void *bias, const void *residual,
                         int64_t ld_residual, const int64_t *group_start, int group_start_count, void *y, void *act_grad,
                         void *workspace, size_t workspace_bytes, int dtype, int act, int batch, int64_t rows, int groups, int out_features,
                         int in_features, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  int rc = check_sizes(dtype, batch, rows, groups, out_features, in_features);
  if (rc) return rc;
  if (act < OPS3D_LINEAR_ACT_NONE || act > OPS3D_LINEAR_ACT_SILU) return fail(OPS3D_FDA_EINVAL, "unknown activation %d", act);
  if (act_grad && act == OPS3D_LINEAR_ACT_NONE)
    return fail(OPS3D_FDA_EINVAL, "act_grad must be NULL without an activation");
  if (ld_x < 0 || (residual && ld_residual < 0)) return fail(OPS3D_FDA_EINVAL, "row distances must not be negative");
  if (batch * rows == 0) return OPS3D_FDA_OK;
  RowsArgs p{};
  if ((rc = make_groups(group_start, group_start_count, batch, rows, groups, p.g))) return rc;
  if (!x || !weight || !y) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  const int es = elem_size(dtype);
  if (misaligned(x, es) || misaligned(weight, es) || misaligned(y, es) || misaligned(bias, es) || misaligned(residual, es) ||
      misaligned(act_grad, es))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  p.a = x;
  p.lda = ld_x;
  p.w = weight;
  p.w_group = (int64_t)out_features * in_features;
  p.bias = bias;
  p.res = residual;
  p.ld_res = ld_residual;
  p.c = y;
  p.act_grad = act_grad;
  p.act = act;
  p.N = out_features;
  p.K = in_features;
  const size_t need = ops3d_linear_forward_workspace_bytes(dtype, batch, rows, groups, out_features, in_features,
                                                           group_start != nullptr);
  if ((rc = check_workspace(workspace, workspace_bytes, need))) return rc;
  set_split(p, need != 0, workspace, dtype, batch * rows, groups);
  return run(dtype, "linear forward", [&](auto t) { return ops3d_linear::forward<decltype(t)>(p, static_cast<hipStream_t>(stream)); });
}

size_t ops3d_linear_backward_workspace_bytes_for(int dtype, int batch, int64_t rows, int groups, int out_features,
                                                 int in_features, int grouped, int with_act_grad, int want) {
  if (!sizes_ok(dtype, batch, rows, groups, out_features, in_features, grouped != 0) || !(want & kWantAll)) return 0;
  return Layout(dtype, grouped != 0, batch, rows, groups, out_features, in_features, with_act_grad != 0, want).bytes;
}

size_t ops3d_linear_backward_workspace_bytes(int dtype, int batch, int64_t rows, int groups, int out_features,
                                             int in_features, int grouped, int with_act_grad) {
  return ops3d_linear_backward_workspace_bytes_for(dtype, batch, rows, groups, out_features, in_features, grouped,
                                                   with_act_grad, kWantAll);
}

int ops3d_linear_backward(const void *x, int64_t ld_x, const void *weight, const int64_t *group_start,
                          int group_start_count, const void *act_grad, const void *grad_y, int64_t ld_grad_y,
                          void *grad_x, void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes,
                          int dtype, int batch, int64_t rows, int groups, int out_features, int in_features,
                          void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  int rc = check_sizes(dtype, batch, rows, groups, out_features, in_features);
  if (rc) return rc;
  if (ld_x < 0 || ld_grad_y < 0) return fail(OPS3D_FDA_EINVAL, "row distances must not be negative");
  const bool wants_w = grad_weight || grad_bias, empty = batch * rows == 0;
  Groups g{};
  if ((rc = make_groups(group_start, group_start_count, batch, rows, groups, g))) return rc;
  if (!empty && (!grad_y || (grad_x && !weight) || (wants_w && !x))) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  const int es = elem_size(dtype);
  if (misaligned(x, es) || misaligned(weight, es) || misaligned(act_grad, es) || misaligned(grad_y, es) ||
      misaligned(grad_x, es) || misaligned(grad_weight, es) || misaligned(grad_bias, es))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  const hipStream_t st = static_cast<hipStream_t>(stream);
  const int want = (grad_x ? OPS3D_LINEAR_WANT_X : 0) | (grad_weight ? OPS3D_LINEAR_WANT_WEIGHT : 0) |
                   (grad_bias ? OPS3D_LINEAR_WANT_BIAS : 0);
  const Layout lay(dtype, group_start != nullptr, empty ? 1 : batch, empty ? 0 : rows, groups, out_features, in_features,
                   act_grad != nullptr, want);
  if ((rc = check_workspace(workspace, workspace_bytes, empty ? 0 : lay.bytes))) return rc;
  char *const ws = static_cast<char *>(workspace);
  void *const dz = wants_w && act_grad && !empty ? ws + lay.dz : nullptr;
  if (grad_x && !empty) {
    RowsArgs p{};
    p.a = grad_y;
    p.lda = ld_grad_y;
    p.scale = act_grad;
    p.dz = dz;
    p.w = weight;
    p.w_group = (int64_t)out_features * in_features;
    p.c = grad_x;
    p.N = in_features;
    p.K = out_features;
    p.g = g;
    set_split(p, lay.split != 0, ws + lay.part, dtype, batch * rows, groups);
    rc = run(dtype, "linear input gradient", [&](auto t) { return ops3d_linear::grad_x<decltype(t)>(p, st); });
  } else if (dz) {
    rc = run(dtype, "linear gradient", [&](auto t) {
      return ops3d_linear::scale<decltype(t)>(grad_y, ld_grad_y, act_grad, dz, batch * rows, out_features, st);
    });
  }
  if (rc || !wants_w) return rc;
  WeightArgs p{};
  p.u = dz ? dz : grad_y;
  p.ldu = dz ? out_features : ld_grad_y;
  p.x = x;
  p.ldx = ld_x;
  p.gw = grad_weight;
  p.gb = grad_bias;
  p.N = out_features;
  p.K = in_features;
  p.chunk = lay.plan.chunk;
  p.items = lay.plan.items;
  p.slots = (int)lay.plan.slots;
  if (!empty && lay.plan.joined) {
    p.part = reinterpret_cast<float *>(ws + lay.part);
    p.part_b = reinterpret_cast<float *>(ws + lay.part_b);
  }
  p.g = g;
  if (empty) p.g.B = 1, p.g.S = 0;   // one chunk of no rows a group
  return run(dtype, "linear weight gradient", [&](auto t) {
    return ops3d_linear::grad_weight<decltype(t)>(p, lay.plan.tile, !empty && lay.plan.joined, st);
  });
}

int ops3d_linear_keep_rows(const void *src, int64_t ld_src, const int64_t *group_start, int group_start_count, void *dst,
                           int dtype, int batch, int64_t rows, int groups, int features, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  int rc = check_sizes(dtype, batch, rows, groups, features, 1);
  if (rc) return rc;
  if (ld_src < 0) return fail(OPS3D_FDA_EINVAL, "row distances must not be negative");
  if (!group_start) return fail(OPS3D_FDA_EINVAL, "group_start is NULL");
  if (batch * rows == 0) return OPS3D_FDA_OK;
  Groups g{};
  if ((rc = make_groups(group_start, group_start_count, batch, rows, groups, g))) return rc;
  if (!src || !dst) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  if (misaligned(src, elem_size(dtype)) || misaligned(dst, elem_size(dtype)))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  return run(dtype, "rows of groups", [&](auto t) {
    return ops3d_linear::keep_rows<decltype(t)>(src, ld_src, dst, batch * rows, features, g, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
