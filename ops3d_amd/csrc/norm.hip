// Layer norm over the last axis (gfx950), forward and backward (include/ops3d_norm.h).
//
// The bytes bound it: x in and y out, or x and grad_y in and grad_x out.  A row stays in registers from its
// first sum to its result, so it is read once:
//   up to 1024 values   a wave, or 8, 16 or 32 of its lanes, has the row
//   up to 8192          a block of 256 or 512 threads has it
//   longer              a block of 256 reads it again for each step (from its L2)
// Rows follow one another in a wave, the next one's loads under way while one is summed; the weight and
// the bias stay in registers.
//
// The mean is formed twice: m from the row, then d = mean(x - m), whose rounding is one of the deviations
// and not of the values; the variance is mean((x - m)^2) - d^2.  Rows far from 0 lose nothing by it.
//
// Backward: the gradients of weight and bias are sums over rows.  A lane keeps them for its columns over
// all rows it sees, the block adds its waves' in LDS and stores one row of partial sums, and a second
// kernel adds those in order.
//
// 73728 x 256 bf16: forward 16.8 us (75.5 MB at 4.5 TB/s), backward 22.2 + 4.0 for the join (113 MB at 5.1); 2053 x 4101
// fp32, rows that start anywhere: 17.7 (67 MB, 3.8) and 28.0 + 6.0 (101 MB, 3.6); 400 x 256: 3.2, a launch.  (A copy of
// 256 MB reaches 5.4 TB/s.)
#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include <type_traits>

#include "../../include/ops3d_norm.h"
#include "elements.h"
#include "reduce.h"

namespace ops3d_fda {
int set_last_error(int code, const char *text);   // fda_capi.hip
}

namespace {

using namespace ops3d_elements;
using ops3d_reduce::sum;

struct Args {
  const void *x, *g;     // rows; grad_y
  int64_t ldx, ldg;
  const void *w, *b;     // [C] or nullptr
  void *out;             // y, or grad_x (nullptr: not wanted)
  float *stats;          // [rows, 3]
  float *part_w, *part_b;   // partial sums [blocks, C] (nullptr: not wanted)
  int64_t rows;
  int C;
  float eps;
};

// CH consecutive values of a vector of the weight's type, or `none` where there is no vector; zeros
// behind its end.
template <typename T, typename W>
__device__ __forceinline__ void load_vector(float (&v)[16 / sizeof(T)], const void *base, int col, int C, float none) {
  constexpr int CH = 16 / (int)sizeof(T), N = sizeof(W) / sizeof(T);
#pragma unroll
  for (int i = 0; i < CH; ++i) v[i] = none;
  if (!base) return;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    Chunk<W> c;
    c.raw = fetch(static_cast<const W *>(base), 0, 0, col + n * (16 / (int)sizeof(W)), 1, C);
#pragma unroll
    for (int i = 0; i < 16 / (int)sizeof(W); ++i) v[n * (16 / (int)sizeof(W)) + i] = (float)c.e[i];
  }
}

template <typename T> __device__ __forceinline__ uint4 pack(const float (&v)[16 / sizeof(T)]) {
  Chunk<T> c;
#pragma unroll
  for (int i = 0; i < 16 / (int)sizeof(T); ++i) c.e[i] = (T)v[i];
  return c.raw;
}

// Over the L lanes that have a row: within a wave, or over a block's waves through LDS.
template <int L> __device__ __forceinline__ float row_sum(float v, float *lds) {
  if constexpr (L <= 64) {
    return sum<L>(v);
  } else {
    v = sum<64>(v);
    __syncthreads();   // the values of the sum before are read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = lds[0];
#pragma unroll
    for (int i = 1; i < L / 64; ++i) s += lds[i];
    return s;
  }
}

// Two sums at once.
template <int L> __device__ __forceinline__ float2 row_sums(float u, float v, float *lds) {
  if constexpr (L <= 64) {
    return make_float2(sum<L>(u), sum<L>(v));
  } else {
    u = sum<64>(u);
    v = sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      lds[(threadIdx.x >> 6) * 2] = u;
      lds[(threadIdx.x >> 6) * 2 + 1] = v;
    }
    __syncthreads();
    float2 s = make_float2(lds[0], lds[1]);
#pragma unroll
    for (int i = 1; i < L / 64; ++i) {
      s.x += lds[2 * i];
      s.y += lds[2 * i + 1];
    }
    return s;
  }
}

// The product, rounded: not one with a difference that it goes into, which would then be another mean than
// the one that is stored.
__device__ __forceinline__ float rounded(float a, float b) {
  float m = a * b;
  asm volatile("" : "+v"(m));
  return m;
}

// L lanes a row, NCH chunks a lane: chunk j of lane i is chunk j L + i of the row.
template <typename T, typename W, int NCH, int L, int NT> __global__ __launch_bounds__(NT) void forward_kernel(Args p) {
  constexpr int CH = 16 / (int)sizeof(T), G = NT / L;
  __shared__ float lds[L > 64 ? L / 32 : 1];
  const int lane = threadIdx.x % L;
  const T *x = static_cast<const T *>(p.x);
  float w[NCH][CH], b[NCH][CH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    load_vector<T, W>(w[j], p.w, (j * L + lane) * CH, p.C, 1.f);
    load_vector<T, W>(b[j], p.b, (j * L + lane) * CH, p.C, 0.f);
  }
  const float inv = 1.f / (float)p.C;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L;
  uint4 next[NCH];
  const auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) next[j] = fetch(x + r * p.ldx, 0, 0, (j * L + lane) * CH, 1, p.C);
  };
  if (row < p.rows) load(row);
  for (; row < p.rows; row += step) {
    float v[NCH][CH], s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      Chunk<T> c;
      c.raw = next[j];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        v[j][i] = (float)c.e[i];
        s += v[j][i];
      }
    }
    if (row + step < p.rows) load(row + step);
    const float mean = rounded(row_sum<L>(s, lds), inv);
    float d = 0.f, dd = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        v[j][i] -= mean;
        const float u = (j * L + lane) * CH + i < p.C ? v[j][i] : 0.f;
        d += u;
        dd = fmaf(u, u, dd);
      }
    }
    const float2 sums = row_sums<L>(d, dd, lds);
    const float rest = rounded(sums.x, inv);
    const float var = fmaf(-rest, rest, sums.y * inv);
    const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + p.eps);
    if (p.stats && lane == 0) {
      p.stats[3 * row] = mean;
      p.stats[3 * row + 1] = rest;
      p.stats[3 * row + 2] = rstd;
    }
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * L + lane) * CH;
      if (col >= p.C) continue;
      float y[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) y[i] = fmaf((v[j][i] - rest) * rstd, w[j][i], b[j][i]);
      store_chunk<T>(static_cast<T *>(p.out) + row * p.C + col, pack<T>(y), p.C - col);
    }
  }
}

// The same for rows that no block's registers hold.
template <typename T, typename W> __global__ __launch_bounds__(256) void forward_long_kernel(Args p) {
  constexpr int CH = 16 / (int)sizeof(T), L = 256;
  __shared__ float lds[L / 32];
  const float inv = 1.f / (float)p.C;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(p.x) + row * p.ldx;
    float s = 0.f, d = 0.f, dd = 0.f;
    for (int col = threadIdx.x * CH; col < p.C; col += L * CH) {
      Chunk<T> c;
      c.raw = fetch(x, 0, 0, col, 1, p.C);
#pragma unroll
      for (int i = 0; i < CH; ++i) s += (float)c.e[i];
    }
    const float mean = rounded(row_sum<L>(s, lds), inv);
    for (int col = threadIdx.x * CH; col < p.C; col += L * CH) {
      Chunk<T> c;
      c.raw = fetch(x, 0, 0, col, 1, p.C);
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float u = col + i < p.C ? (float)c.e[i] - mean : 0.f;
        d += u;
        dd = fmaf(u, u, dd);
      }
    }
    const float2 sums = row_sums<L>(d, dd, lds);
    const float rest = rounded(sums.x, inv);
    const float var = fmaf(-rest, rest, sums.y * inv);
    const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + p.eps);
    if (p.stats && threadIdx.x == 0) {
      p.stats[3 * row] = mean;
      p.stats[3 * row + 1] = rest;
      p.stats[3 * row + 2] = rstd;
    }
    for (int col = threadIdx.x * CH; col < p.C; col += L * CH) {
      Chunk<T> c;
      c.raw = fetch(x, 0, 0, col, 1, p.C);
      float w[CH], b[CH], y[CH];
      load_vector<T, W>(w, p.w, col, p.C, 1.f);
      load_vector<T, W>(b, p.b, col, p.C, 0.f);
#pragma unroll
      for (int i = 0; i < CH; ++i) y[i] = fmaf((((float)c.e[i] - mean) - rest) * rstd, w[i], b[i]);
      store_chunk<T>(static_cast<T *>(p.out) + row * p.C + col, pack<T>(y), p.C - col);
    }
  }
}

// The sums of a block's waves for their columns: each wave's values in turn, the groups of a wave added
// before.  Called by all threads.
template <int CH, int NCH, int L, int NT>
__device__ __forceinline__ void store_partial(float *part, float (&v)[NCH][CH], float *lds, int C) {
  if (!part) return;
  part += (int64_t)blockIdx.x * C;
  const int lane = threadIdx.x % L;
  if constexpr (L >= NT) {
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < CH; ++i)
        if ((j * L + lane) * CH + i < C) part[(j * L + lane) * CH + i] = v[j][i];
  } else {
    constexpr int kWaves = NT / 64, kLanes = L < 64 ? L : 64;
    const int wave = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NCH; ++j)
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        float s = v[j][i];
        for (int o = kLanes; o < 64; o <<= 1) s += __shfl_xor(s, o);
        if ((int)(threadIdx.x & 63) < kLanes) lds[(wave * NCH * CH + j * CH + i) * kLanes + lane] = s;
      }
    __syncthreads();
    for (int c = threadIdx.x; c < NCH * CH * kLanes; c += NT) {
      const int col = (c / (CH * kLanes) * kLanes + c % kLanes) * CH + c / kLanes % CH;
      float s = lds[c];
      for (int k = 1; k < kWaves; ++k) s += lds[k * NCH * CH * kLanes + c];
      if (col < C) part[col] = s;
    }
  }
}

template <typename T, typename W, int NCH, int L, int NT> __global__ __launch_bounds__(NT) void backward_kernel(Args p) {
  constexpr int CH = 16 / (int)sizeof(T), G = NT / L;
  __shared__ float lds[L >= NT ? L / 32 : NT / 64 * NCH * CH * (L < 64 ? L : 64)];
  const int lane = threadIdx.x % L;
  const T *x = static_cast<const T *>(p.x), *g = static_cast<const T *>(p.g);
  float w[NCH][CH], aw[NCH][CH], ab[NCH][CH];
#pragma unroll
  for (int j = 0; j < NCH; ++j) {
    load_vector<T, W>(w[j], p.w, (j * L + lane) * CH, p.C, 1.f);
#pragma unroll
    for (int i = 0; i < CH; ++i) aw[j][i] = ab[j][i] = 0.f;
  }
  const float inv = 1.f / (float)p.C;
  const int64_t step = (int64_t)gridDim.x * G;
  int64_t row = (int64_t)blockIdx.x * G + threadIdx.x / L;
  uint4 nx[NCH], ng[NCH];
  float mean, rest, rstd;
  const auto load = [&](int64_t r) {
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      nx[j] = fetch(x + r * p.ldx, 0, 0, (j * L + lane) * CH, 1, p.C);
      ng[j] = fetch(g + r * p.ldg, 0, 0, (j * L + lane) * CH, 1, p.C);
    }
    mean = p.stats[3 * r];
    rest = p.stats[3 * r + 1];
    rstd = p.stats[3 * r + 2];
  };
  if (row < p.rows) load(row);
  for (; row < p.rows; row += step) {
    float n[NCH][CH], gw[NCH][CH], s = 0.f, sn = 0.f;
    const float r = rstd;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      Chunk<T> cx, cg;
      cx.raw = nx[j];
      cg.raw = ng[j];   // zeros behind the row's end
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const float gi = (float)cg.e[i];
        n[j][i] = (((float)cx.e[i] - mean) - rest) * r;
        ab[j][i] += gi;
        aw[j][i] = fmaf(gi, n[j][i], aw[j][i]);
        gw[j][i] = gi * w[j][i];
        s += gw[j][i];
        sn = fmaf(gw[j][i], n[j][i], sn);
      }
    }
    if (row + step < p.rows) load(row + step);
    if (!p.out) continue;
    const float2 sums = row_sums<L>(s, sn, lds);
    s = sums.x * inv;
    sn = sums.y * inv;
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int col = (j * L + lane) * CH;
      if (col >= p.C) continue;
      float dx[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) dx[i] = r * (fmaf(-n[j][i], sn, gw[j][i] - s));
      store_chunk<T>(static_cast<T *>(p.out) + row * p.C + col, pack<T>(dx), p.C - col);
    }
  }
  store_partial<CH, NCH, L, NT>(p.part_w, aw, lds, p.C);
  store_partial<CH, NCH, L, NT>(p.part_b, ab, lds, p.C);
}

// Rows that no block's registers hold: grad_x, a block a row ...
template <typename T, typename W> __global__ __launch_bounds__(256) void backward_long_kernel(Args p) {
  constexpr int CH = 16 / (int)sizeof(T), L = 256;
  __shared__ float lds[L / 32];
  const float inv = 1.f / (float)p.C;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T *x = static_cast<const T *>(p.x) + row * p.ldx, *g = static_cast<const T *>(p.g) + row * p.ldg;
    const float mean = p.stats[3 * row], rest = p.stats[3 * row + 1], r = p.stats[3 * row + 2];
    float s = 0.f, sn = 0.f;
    for (int step = 0; step < 2; ++step) {
      for (int col = threadIdx.x * CH; col < p.C; col += L * CH) {
        Chunk<T> cx, cg;
        cx.raw = fetch(x, 0, 0, col, 1, p.C);
        cg.raw = fetch(g, 0, 0, col, 1, p.C);
        float w[CH], dx[CH];
        load_vector<T, W>(w, p.w, col, p.C, 1.f);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const float gw = (float)cg.e[i] * w[i], n = (((float)cx.e[i] - mean) - rest) * r;
          if (step == 0) {
            s += gw;
            sn = fmaf(gw, n, sn);
          } else {
            dx[i] = r * fmaf(-n, sn, gw - s);
          }
        }
        if (step) store_chunk<T>(static_cast<T *>(p.out) + row * p.C + col, pack<T>(dx), p.C - col);
      }
      if (step == 0) {
        const float2 sums = row_sums<L>(s, sn, lds);
        s = sums.x * inv;
        sn = sums.y * inv;
      }
    }
  }
}
// ... and the partial sums of the other two, a block for 256 chunks of columns of every gridDim.y-th row.
template <typename T> __global__ __launch_bounds__(256) void columns_kernel(Args p) {
  constexpr int CH = 16 / (int)sizeof(T);
  const int col = (blockIdx.x * 256 + threadIdx.x) * CH;
  float aw[CH], ab[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) aw[i] = ab[i] = 0.f;
  if (col >= p.C) return;
  for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
    const float mean = p.stats[3 * row], rest = p.stats[3 * row + 1], r = p.stats[3 * row + 2];
    Chunk<T> cx, cg;
    cx.raw = fetch(static_cast<const T *>(p.x) + row * p.ldx, 0, 0, col, 1, p.C);
    cg.raw = fetch(static_cast<const T *>(p.g) + row * p.ldg, 0, 0, col, 1, p.C);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      ab[i] += (float)cg.e[i];
      aw[i] = fmaf((float)cg.e[i], (((float)cx.e[i] - mean) - rest) * r, aw[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (col + i < p.C) {
      if (p.part_w) p.part_w[(int64_t)blockIdx.y * p.C + col + i] = aw[i];
      if (p.part_b) p.part_b[(int64_t)blockIdx.y * p.C + col + i] = ab[i];
    }
}

// The sums of n rows of partial sums: 16 columns a block, 64 threads a column, each adding every 64th
// row; then those in order.  blockIdx.y: weight or bias.
template <typename W>
__global__ __launch_bounds__(1024) void join_kernel(const float *part_w, const float *part_b, void *gw, void *gb, int n, int C) {
  __shared__ float lds[64][17];
  const float *part = blockIdx.y ? part_b : part_w;
  W *out = static_cast<W *>(blockIdx.y ? gb : gw);
  if (!out) return;
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, col = blockIdx.x * 16 + c;
  float s = 0.f;
  if (col < C)
    for (int i = r; i < n; i += 64) s += part[(int64_t)i * C + col];
  lds[r][c] = s;
  __syncthreads();
  for (int o = 32; o; o >>= 1) {
    if (r < o) lds[r][c] += lds[r + o][c];
    __syncthreads();
  }
  if (r == 0 && col < C) out[col] = (W)lds[0][c];
}

// ---------------------------------------------------------------------------------------------

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
bool misaligned(const void *p, int esize) { return reinterpret_cast<uintptr_t>(p) & (uintptr_t)(esize - 1); }

constexpr int kMaxWidth = 1 << 24;
constexpr int64_t kMaxRows = (int64_t)1 << 40;   // bytes of rows and statistics stay 64-bit

// What has a row: `lanes` lanes with `chunks` chunks each, 16 values a lane at most; 0 lanes: a block,
// again and again.
struct Plan {
  int lanes, chunks;
  Plan(int dtype, int C) {
    const int per = 16 / elem_size(dtype), n = (C + per - 1) / per, most = 16 / per;
    lanes = n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 * most ? 64 : n <= 256 * most ? 256 : n <= 512 * most ? 512
            : 0;
    chunks = lanes ? (n + lanes - 1) / lanes : 1;
  }
  // Rows of partial sums: one a block; few enough that adding them costs little.
  int blocks(int64_t rows) const {
    const bool wave = lanes && lanes <= 64;
    const int64_t per = wave ? 512 / lanes : 1, most = wave ? 512 : 256;
    const int64_t n = (rows + per - 1) / per;
    return (int)(n < most ? n : most);
  }
};

template <typename T, typename F> hipError_t with_plan(const Plan &p, F f) {
#define OPS3D_PLAN(l, c)                          \
  if constexpr (c * (16 / (int)sizeof(T)) <= 16)  \
    if (p.lanes == l && p.chunks == c) return f(std::integral_constant<int, l>(), std::integral_constant<int, c>());
#define OPS3D_PLANS(l) OPS3D_PLAN(l, 1) OPS3D_PLAN(l, 2) OPS3D_PLAN(l, 3) OPS3D_PLAN(l, 4)
  OPS3D_PLAN(8, 1) OPS3D_PLAN(16, 1) OPS3D_PLAN(32, 1) OPS3D_PLANS(64) OPS3D_PLANS(256) OPS3D_PLANS(512)
#undef OPS3D_PLANS
#undef OPS3D_PLAN
  return hipErrorInvalidValue;
}

unsigned grid_for(int64_t blocks, int64_t most) { return (unsigned)(blocks < most ? blocks : most); }

template <typename T, typename W> hipError_t forward(const Args &a, int dtype, hipStream_t st) {
  const Plan plan(dtype, a.C);
  if (!plan.lanes) {
    forward_long_kernel<T, W><<<grid_for(a.rows, 2048), 256, 0, st>>>(a);
    return hipGetLastError();
  }
  return with_plan<T>(plan, [&](auto l, auto c) {
    constexpr int L = decltype(l)::value, NT = L < 256 ? 256 : L;
    // as many blocks as the CUs hold: each loads its next row while it sums one (2053 x 4101 fp32: 17.6 us, with twice as
    // many 21.2)
    constexpr int kMost = L > 64 ? 512 * 512 / NT : 2048;
    forward_kernel<T, W, decltype(c)::value, L, NT><<<grid_for((a.rows + NT / L - 1) / (NT / L), kMost), NT, 0, st>>>(a);
    return hipGetLastError();
  });
}

template <typename T, typename W> hipError_t backward(const Args &a, int dtype, void *gw, void *gb, hipStream_t st) {
  const Plan plan(dtype, a.C);
  const int n = plan.blocks(a.rows);
  if (n) {
    hipError_t e = hipSuccess;
    if (!plan.lanes) {
      constexpr int CH = 16 / (int)sizeof(T);
      if (a.out) backward_long_kernel<T, W><<<grid_for(a.rows, 2048), 256, 0, st>>>(a);
      if (gw || gb) columns_kernel<T><<<dim3((a.C + 256 * CH - 1) / (256 * CH), n), 256, 0, st>>>(a);
      e = hipGetLastError();
    } else {
      e = with_plan<T>(plan, [&](auto l, auto c) {
        constexpr int L = decltype(l)::value, NT = L <= 64 ? 512 : L;
        backward_kernel<T, W, decltype(c)::value, L, NT><<<n, NT, 0, st>>>(a);
        return hipGetLastError();
      });
    }
    if (e != hipSuccess) return e;
  }
  if (gw || gb) join_kernel<W><<<dim3((a.C + 15) / 16, 2), 1024, 0, st>>>(a.part_w, a.part_b, gw, gb, n, a.C);
  return hipGetLastError();
}

template <typename F> int run(int dtype, int weight_dtype, const char *what, F f) {
  hipError_t e;
  if (dtype == OPS3D_FDA_F32) e = f(float(), float());
  else if (dtype == OPS3D_FDA_F16) e = weight_dtype == dtype ? f(_Float16(), _Float16()) : f(_Float16(), float());
  else e = weight_dtype == dtype ? f(__bf16(), __bf16()) : f(__bf16(), float());
  if (e == hipSuccess) return OPS3D_FDA_OK;
  return fail(OPS3D_FDA_ERUNTIME, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
}

int check(int dtype, int weight_dtype, int64_t rows, int width) {
  if (elem_size(dtype) == 0) return fail(OPS3D_FDA_EINVAL, "unsupported dtype code %d", dtype);
  if (weight_dtype != dtype && weight_dtype != OPS3D_FDA_F32)
    return fail(OPS3D_FDA_EINVAL, "weight_dtype must be dtype or F32, got %d", weight_dtype);
  if (rows < 0 || rows > kMaxRows) return fail(OPS3D_FDA_EINVAL, "invalid or too many rows: %lld", (long long)rows);
  if (width < 1 || width > kMaxWidth)
    return fail(OPS3D_FDA_EINVAL, "the normalised axis must have 1..%d elements, got %d", kMaxWidth, width);
  return OPS3D_FDA_OK;
}

}  // namespace

extern "C" {

int ops3d_layer_norm_forward(const void *x, int64_t ld_x, const void *weight, const void *bias, void *y, float *stats,
                             int dtype, int weight_dtype, int64_t rows, int width, float eps, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  if (const int rc = check(dtype, weight_dtype, rows, width)) return rc;
  if (ld_x < 0) return fail(OPS3D_FDA_EINVAL, "row distances must not be negative");
  if (!(eps >= 0.f) || eps > 3e38f) return fail(OPS3D_FDA_EINVAL, "eps must be finite and not negative");
  if (rows == 0) return OPS3D_FDA_OK;
  if (!x || !y) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  const int es = elem_size(dtype), ws = elem_size(weight_dtype);
  if (misaligned(x, es) || misaligned(y, es) || misaligned(weight, ws) || misaligned(bias, ws) || misaligned(stats, 4))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  Args a{};
  a.x = x;
  a.ldx = ld_x;
  a.w = weight;
  a.b = bias;
  a.out = y;
  a.stats = stats;
  a.rows = rows;
  a.C = width;
  a.eps = eps;
  return run(dtype, weight_dtype, "layer norm forward",
             [&](auto t, auto w) { return forward<decltype(t), decltype(w)>(a, dtype, static_cast<hipStream_t>(stream)); });
}

size_t ops3d_layer_norm_backward_workspace_bytes(int dtype, int64_t rows, int width, int want_weight, int want_bias) {
  if (elem_size(dtype) == 0 || rows < 1 || rows > kMaxRows || width < 1 || width > kMaxWidth) return 0;
  return ((want_weight != 0) + (want_bias != 0)) * align256((size_t)Plan(dtype, width).blocks(rows) * width * 4);
}

int ops3d_layer_norm_backward(const void *x, int64_t ld_x, const void *weight, const float *stats, const void *grad_y,
                              int64_t ld_grad_y, void *grad_x, void *grad_weight, void *grad_bias, void *workspace,
                              size_t workspace_bytes, int dtype, int weight_dtype, int64_t rows, int width, void *stream) {
  ops3d_fda::set_last_error(OPS3D_FDA_OK, "");
  if (const int rc = check(dtype, weight_dtype, rows, width)) return rc;
  if (ld_x < 0 || ld_grad_y < 0) return fail(OPS3D_FDA_EINVAL, "row distances must not be negative");
  if (!grad_x && !grad_weight && !grad_bias) return OPS3D_FDA_OK;
  if (rows && (!x || !stats || !grad_y)) return fail(OPS3D_FDA_EINVAL, "NULL pointer argument");
  const int es = elem_size(dtype), ws = elem_size(weight_dtype);
  if (misaligned(x, es) || misaligned(grad_y, es) || misaligned(grad_x, es) || misaligned(weight, ws) ||
      misaligned(grad_weight, ws) || misaligned(grad_bias, ws) || misaligned(stats, 4))
    return fail(OPS3D_FDA_EINVAL, "data pointers must be aligned to their element size");
  const size_t need = ops3d_layer_norm_backward_workspace_bytes(dtype, rows, width, grad_weight != nullptr, grad_bias != nullptr);
  if (need && (!workspace || workspace_bytes < need))
    return fail(OPS3D_FDA_EINVAL, "workspace too small: %zu bytes given, %zu needed", workspace_bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(workspace) & 255u))
    return fail(OPS3D_FDA_EINVAL, "workspace must be 256-byte aligned");
  Args a{};
  a.x = x;
  a.ldx = ld_x;
  a.g = grad_y;
  a.ldg = ld_grad_y;
  a.w = weight;
  a.out = grad_x;
  a.stats = const_cast<float *>(stats);
  a.rows = rows;
  a.C = width;
  float *part = static_cast<float *>(workspace);
  if (need && grad_weight) {
    a.part_w = part;
    part += align256((size_t)Plan(dtype, width).blocks(rows) * width * 4) / 4;
  }
  if (need && grad_bias) a.part_b = part;
  return run(dtype, weight_dtype, "layer norm backward", [&](auto t, auto w) {
    return backward<decltype(t), decltype(w)>(a, dtype, grad_weight, grad_bias, static_cast<hipStream_t>(stream));
  });
}

}  // extern "C"
