// C entry points of attention over all tokens (include/ops3d_attention.h).
#include <stdarg.h>
#include <stdio.h>

#include "../../include/ops3d_attention.h"
#include "attention_kernels.h"

namespace ops3d_fda {
int set_last_error(int code, const char *text);   // fda_capi.hip
}

namespace {

using namespace ops3d_attention;

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
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kMaxRows = 0x7fffffff - 65536;   // rows and columns of an item, and tiles, stay 32-bit

// Sizes that any call may have; 0 or the error that is set.
int check(const ops3d_attention_problem *p) {
  if (!p) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  if (!elem_size(p->dtype)) return fail(OPS3D_FDA_EINVAL, "unsupported dtype code %d", p->dtype);
  if (p->kv_heads < 1 || p->heads < 1 || p->heads % p->kv_heads)
    return fail(OPS3D_FDA_EINVAL, "heads (%d) must be a multiple of kv_heads (%d)", p->heads, p->kv_heads);
  if (p->dim < 1 || p->dim > OPS3D_ATTENTION_MAX_DIM)
    return fail(OPS3D_FDA_EINVAL, "heads must have 1..%d channels, got %d", OPS3D_ATTENTION_MAX_DIM, p->dim);
  if (!(p->scale > 0.f) || p->scale > 1e30f) return fail(OPS3D_FDA_EINVAL, "scale must be positive and finite");
  const int64_t G = p->heads / p->kv_heads;
  if (p->q_rows < 0 || p->k_rows < 0 || p->items < 0 || p->q_rows > kMaxRows / G || p->k_rows > kMaxRows ||
      p->items > (1 << 24))
    return fail(OPS3D_FDA_EINVAL, "invalid or too many rows: %d items of %lld queries (times %lld heads) and %lld keys", p->items,
                (long long)p->q_rows, (long long)G, (long long)p->k_rows);
  if (!p->q_start != !p->k_start) return fail(OPS3D_FDA_EINVAL, "q_start and k_start go together");
  if (p->q_start) {
    if (p->items != 1 || p->q_len || p->k_len) return fail(OPS3D_FDA_EINVAL, "packed sequences are one item, without lengths");
    if (p->sequences < 1 || p->sequences > OPS3D_ATTENTION_MAX_SEQUENCES)
      return fail(OPS3D_FDA_EINVAL, "there must be 1..%d sequences, got %d", OPS3D_ATTENTION_MAX_SEQUENCES, p->sequences);
    for (const int n : {p->q_start_count, p->k_start_count})
      if (n != p->sequences && n != p->sequences + 1)
        return fail(OPS3D_FDA_EINVAL, "starts must have sequences or sequences + 1 entries (%d), got %d", p->sequences, n);
  }
  for (const int64_t *t : {p->q_start, p->k_start, p->q_len, p->k_len})
    if (reinterpret_cast<uintptr_t>(t) & 7u) return fail(OPS3D_FDA_EINVAL, "starts and lengths must be 8-byte aligned");
  return OPS3D_FDA_OK;
}

int padded_dim(int dim) { return dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

// How a side's columns are tiled, and into how many parts the other side's rows are cut.
struct Plan {
  int shape, tiles, tiles_item, splits;
};

// columns and others: of an item, or of all packed sequences.  Measured in bf16 (us):
//   wide tiles read the rows that come by least often, if there are two blocks a CU: 8192 x 8192, 8 heads of 32
//     channels, forward: 141 in tiles of 128, 151 of 64, 298 of 16; 4096 x 4096: 51, 47, 81
//   narrow tiles, where there are few columns and few rows: 1024 x 1024: 15, 12, 10; and where sequences are short
//   parts, where few columns see many rows: 200 x 37376, 2 items: 360 in one, 49 in 8, 42 in 16; one query of 32/8
//     heads of 128 over 8 caches of 8192: 42 in 8, 39 in 16, 50 in narrow tiles
//   twice the blocks, where sequences or a causal mask give them different amounts to do: grad k v of 8192 causal
//     tokens, 16/4 heads of 128: 273 in one part, 189 + 16 for the join in 2
Plan plan_of(const ops3d_attention_problem *p, int64_t columns, int64_t others, int widest) {
  const int64_t runs = p->q_start ? p->sequences : p->items;   // what has tiles of its own
  const int64_t per = p->q_start ? ceil_div(columns, runs) : columns;
  // of packed sequences the largest count, of which the sizes here say little
  const int64_t mean = p->q_start ? ceil_div(others, runs) : others, far = p->q_start && 4 * mean < others ? 4 * mean : others;
  const int64_t stages = far / (elem_size(p->dtype) == 4 ? 32 : 64);
  const bool uneven = p->causal || p->q_start;
  const auto blocks = [&](int width) { return ceil_div(per, width) * runs * p->kv_heads; };
  const auto parts = [&](int64_t target, int64_t blocks) {
    const int64_t n = blocks ? (target + blocks / 2) / blocks : 1, most = stages / 2;
    return (int)(n < 2 || most < 2 ? 1 : n < most ? n : most);
  };
  Plan plan{};
  plan.splits = 1;
  if (widest == kMany && per > 64 && blocks(128) >= 512) {
    plan.shape = kMany;
    plan.splits = uneven ? parts(1024, blocks(128)) : 1;
  } else if (per > 16 && blocks(64) >= 256) {
    plan.shape = kSome;
    plan.splits = uneven ? parts(1024, blocks(64)) : 1;
  } else if (stages >= 32) {
    plan.shape = kSome;
    plan.splits = parts(1024, blocks(64));
  } else {
    plan.shape = kFew;
  }
  const int width = plan.shape == kMany ? 128 : plan.shape == kSome ? 64 : 16;
  plan.tiles_item = (int)ceil_div(columns, width);
  plan.tiles = p->q_start ? (int)(columns / width + p->sequences + 2) : 0;   // packed: each segment may end inside a tile
  return plan;
}
Plan plan_queries(const ops3d_attention_problem *p) { return plan_of(p, p->q_rows * (p->heads / p->kv_heads), p->k_rows, kMany); }
// Keys of 128 channels: two results, K and V for each column are too many registers for tiles of 128 columns
// (grad k v of 8192 causal tokens, 16/4 heads: 374 us, in tiles of 64 273 us).
Plan plan_keys(const ops3d_attention_problem *p) {
  return plan_of(p, p->k_rows, p->q_rows * (p->heads / p->kv_heads), p->dim > 64 ? kSome : kMany);
}

// false: 2^31 blocks or more, which are counted in 32 bits
bool set_plan(Args &a, const ops3d_attention_problem *p, const Plan &plan) {
  const int64_t tiles = p->q_start ? plan.tiles : (int64_t)plan.tiles_item * p->items;
  if (tiles * p->kv_heads > 0x7fffffff / plan.splits) return false;
  a.tiles = (int)tiles;
  a.tiles_item = plan.tiles_item;
  a.splits = plan.splits;
  return true;
}

// Bytes of the table of a plan's tiles, where sequences are many.
size_t table_bytes(const ops3d_attention_problem *p, const Plan &plan) {
  return p->q_start && p->sequences > kWalk ? align256((size_t)plan.tiles * 32) : 0;
}

int64_t cells_of(const ops3d_attention_problem *p) { return (int64_t)p->items * p->heads * p->q_rows; }
int64_t keys_of(const ops3d_attention_problem *p) { return (int64_t)p->items * p->kv_heads * p->k_rows; }

size_t forward_bytes(const ops3d_attention_problem *p) {
  const Plan plan = plan_queries(p);
  return table_bytes(p, plan) + (plan.splits > 1 ? align256((size_t)plan.splits * cells_of(p) * (padded_dim(p->dim) + 4) * 4) : 0);
}
// The larger of the two kernels' tables, then delta, then the larger of their parts.
size_t backward_table(const ops3d_attention_problem *p) {
  const size_t q = table_bytes(p, plan_queries(p)), k = table_bytes(p, plan_keys(p));
  return q > k ? q : k;
}
size_t backward_bytes(const ops3d_attention_problem *p) {
  const size_t row = (size_t)padded_dim(p->dim) * 4;
  const int q = plan_queries(p).splits, k = plan_keys(p).splits;
  const size_t a = q > 1 ? q * cells_of(p) * row : 0, b = k > 1 ? 2 * k * keys_of(p) * row : 0;
  return backward_table(p) + align256((size_t)cells_of(p) * 4) + align256(a > b ? a : b);
}

int take(Tensor &t, const ops3d_attention_tensor *x, int es) {
  if (!x || !x->data) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  if (reinterpret_cast<uintptr_t>(x->data) & (uintptr_t)(es - 1))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  if (x->item < 0 || x->token < 0 || x->head < 0) return fail(OPS3D_FDA_EINVAL, "strides must not be negative");
  t = Tensor{x->data, x->item, x->token, x->head};
  return OPS3D_FDA_OK;
}

Args args_of(const ops3d_attention_problem *p) {
  Args a{};
  a.q_start = p->q_start;
  a.k_start = p->k_start;
  a.q_len = p->q_len;
  a.k_len = p->k_len;
  a.q_count = p->q_start_count;
  a.k_count = p->k_start_count;
  a.E = p->sequences;
  a.Sq = (int)p->q_rows;
  a.Sk = (int)p->k_rows;
  a.Hk = p->kv_heads;
  a.G = p->heads / p->kv_heads;
  a.D = p->dim;
  // c < 2^31: with 2^(shift - 1) < G <= 2^shift, magic = ceil(2^(31 + shift) / G) fits 32 bits and c magic is less
  // than 2^(31 + shift) / G too large
  while ((1 << a.shift) < a.G) ++a.shift;
  a.magic = (uint32_t)((((uint64_t)1 << (31 + a.shift)) + a.G - 1) / a.G);
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.c = (float)(p->scale * 1.4426950408889634);
  a.heads = p->items * p->kv_heads;
  a.cells = cells_of(p);
  return a;
}

// Whether a stage's rows may go straight to LDS: whole chunks at 16-byte boundaries, whose places in a stage of
// 128 and in a group of heads fit 32 bits.
bool direct(const ops3d_attention_problem *p, const Tensor &t) {
  const int64_t es = elem_size(p->dtype);
  return p->dim * es % 16 == 0 && !((reinterpret_cast<uintptr_t>(t.p) | (uint64_t)(t.item * es) | (uint64_t)(t.token * es) | (uint64_t)(t.head * es)) & 15u) &&
         t.token < (1 << 20) && t.head < (1 << 20) && p->heads / p->kv_heads <= 256;   // 2^31 bytes, of 4 an element
}

template <typename F> int run(int dtype, const char *what, F f) {
  const hipError_t e = dtype == OPS3D_FDA_F32 ? f(float()) : dtype == OPS3D_FDA_F16 ? f(_Float16()) : f(__bf16());
  if (e == hipSuccess) return OPS3D_FDA_OK;
  return fail(OPS3D_FDA_ERUNTIME, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
}

int check_workspace(const void *workspace, size_t bytes, size_t need) {
  if (need && (!workspace || bytes < need))
    return fail(OPS3D_FDA_EINVAL, "workspace too small: %zu bytes given, %zu needed", bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 255u)) return fail(OPS3D_FDA_EINVAL, "workspace must be 256-byte aligned");
  return OPS3D_FDA_OK;
}

// Quietly: whether check() would pass.
bool valid(const ops3d_attention_problem *p) {
  const int rc = check(p);
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  return rc == OPS3D_FDA_OK;
}

}  // namespace

extern "C" {

size_t ops3d_attention_forward_workspace_bytes(const ops3d_attention_problem *problem) {
  return valid(problem) && cells_of(problem) ? forward_bytes(problem) : 0;
}

int ops3d_attention_forward(const ops3d_attention_problem *problem, const ops3d_attention_tensor *q,
                            const ops3d_attention_tensor *k, const ops3d_attention_tensor *v,
                            const ops3d_attention_tensor *out, void *out_rest, float *lse, void *workspace,
                            size_t workspace_bytes, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  int rc = check(problem);
  if (rc) return rc;
  if (cells_of(problem) == 0) return OPS3D_FDA_OK;
  Args a = args_of(problem);
  const int es = elem_size(problem->dtype);
  if ((rc = take(a.q, q, es)) || (rc = take(a.o, out, es))) return rc;
  if (problem->k_rows && ((rc = take(a.k, k, es)) || (rc = take(a.v, v, es)))) return rc;
  if (reinterpret_cast<uintptr_t>(lse) & 3u) return fail(OPS3D_FDA_EINVAL, "lse must be 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(out_rest) & (uintptr_t)(es - 1))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  a.rest = out_rest;
  a.lse = lse;
  const size_t need = forward_bytes(problem);
  if ((rc = check_workspace(workspace, workspace_bytes, need))) return rc;
  const Plan plan = plan_queries(problem);
  if (!set_plan(a, problem, plan)) return fail(OPS3D_FDA_EINVAL, "attention: 2^31 tiles or more");
  const int dp = padded_dim(problem->dim);
  a.dma = direct(problem, a.k) && direct(problem, a.v) ? 1 : 0;
  const size_t table = table_bytes(problem, plan);
  a.table = table ? static_cast<const int4 *>(workspace) : nullptr;
  a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) + table);
  a.part_ml = reinterpret_cast<f32x4 *>(a.part + (size_t)a.splits * a.cells * dp);
  return run(problem->dtype, "attention forward",
             [&](auto t) { return ops3d_attention::forward<decltype(t)>(a, dp, plan.shape, static_cast<hipStream_t>(stream)); });
}

size_t ops3d_attention_backward_workspace_bytes(const ops3d_attention_problem *problem) {
  return valid(problem) && problem->items ? backward_bytes(problem) : 0;
}

int ops3d_attention_backward(const ops3d_attention_problem *problem, const ops3d_attention_tensor *q,
                             const ops3d_attention_tensor *k, const ops3d_attention_tensor *v,
                             const ops3d_attention_tensor *out, const void *out_rest, const float *lse,
                             const ops3d_attention_tensor *grad_out,
                             const ops3d_attention_tensor *grad_q, const ops3d_attention_tensor *grad_k,
                             const ops3d_attention_tensor *grad_v, void *workspace, size_t workspace_bytes, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  int rc = check(problem);
  if (rc) return rc;
  if (!grad_k != !grad_v) return fail(OPS3D_FDA_EINVAL, "grad_k and grad_v go together");
  const int64_t cells = cells_of(problem), keys = keys_of(problem);
  const bool wants_q = grad_q && cells, wants_k = grad_k && keys;
  if (!wants_q && !wants_k) return OPS3D_FDA_OK;
  Args a = args_of(problem);
  const int es = elem_size(problem->dtype);
  if (cells) {
    if ((rc = take(a.q, q, es)) || (rc = take(a.o, out, es)) || (rc = take(a.g, grad_out, es))) return rc;
    if (reinterpret_cast<uintptr_t>(out_rest) & (uintptr_t)(es - 1))
      return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
    a.rest = const_cast<void *>(out_rest);
    if (!lse) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
    if (reinterpret_cast<uintptr_t>(lse) & 3u) return fail(OPS3D_FDA_EINVAL, "lse must be 4-byte aligned");
  }
  if (keys && ((rc = take(a.k, k, es)) || (rc = take(a.v, v, es)))) return rc;
  if (wants_q && (rc = take(a.gq, grad_q, es))) return rc;
  if (wants_k && ((rc = take(a.gk, grad_k, es)) || (rc = take(a.gv, grad_v, es)))) return rc;
  a.lse = const_cast<float *>(lse);
  if ((rc = check_workspace(workspace, workspace_bytes, backward_bytes(problem)))) return rc;
  const size_t table = backward_table(problem);
  a.table = table ? static_cast<const int4 *>(workspace) : nullptr;
  a.delta = reinterpret_cast<float *>(static_cast<char *>(workspace) + table);
  a.part = a.delta + align256((size_t)cells * 4) / 4;
  const int dp = padded_dim(problem->dim);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  a.dma = (keys && direct(problem, a.k) && direct(problem, a.v) ? 1 : 0) | (cells && direct(problem, a.q) && direct(problem, a.g) ? 2 : 0);
  if (cells) {
    const Plan plan = plan_queries(problem);
    if (!set_plan(a, problem, plan)) return fail(OPS3D_FDA_EINVAL, "attention: 2^31 tiles or more");
    if (!wants_q) a.splits = 1;   // delta alone
    rc = run(problem->dtype, "attention query gradient", [&](auto t) { return ops3d_attention::grad_q<decltype(t)>(a, dp, plan.shape, st); });
    if (rc) return rc;
  }
  if (!wants_k) return OPS3D_FDA_OK;
  const Plan plan = plan_keys(problem);
  if (!set_plan(a, problem, plan)) return fail(OPS3D_FDA_EINVAL, "attention: 2^31 tiles or more");
  return run(problem->dtype, "attention key gradient", [&](auto t) { return ops3d_attention::grad_kv<decltype(t)>(a, dp, plan.shape, st); });
}

}  // extern "C"
