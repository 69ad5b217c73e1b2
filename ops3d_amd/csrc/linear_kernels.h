// Linear operators (gfx950): y = act(x W^T + b) + r and its gradients, one weight or one per group
// of consecutive rows.
//
// Every product here is a tile product over LDS with fp32 sums in MFMA accumulators:
//   rows kernel     y = x W^T            rows of x by rows of W, both contiguous along the sum
//   rows kernel     dx = dz W            rows of dz by columns of W (W is strided along the sum)
//   weight kernel   dW = dz^T x          both strided along the sum (the rows), split over chunks of
//                                        rows; the chunks' partial sums are joined in order
// A stage of a tile is 128 bytes of the sum's axis for every row (64 elements of 16 bits, 32 of 32).
// Operands that are contiguous along the sum lie in LDS as rows of 128 bytes and are read 16 bytes a
// lane; the others lie as they are in memory, sum axis outermost, and are read transposed
// (ds_read_tr16_b64; single words for fp32).  16-byte chunks are XOR-swizzled so that the lanes of a
// read fall on different banks.
// The weight is the first operand of the MFMA, so a lane holds 4 consecutive output columns of a row;
// the epilogue passes them through LDS, 16 rows at a time, to write whole 16-byte chunks.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ops3d_linear {

enum Act { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4 };

// Which rows use which weight.  start == nullptr: all rows use weight 0 (then B == 1, E == 1).
// Otherwise, for each of B items of S rows, group e has rows [bound(e), bound(e+1)), where bound(i)
// is start[i] held to [0, S] and made monotone, and S for i >= count.
struct Groups {
  const int64_t *start;
  int count;   // E or E + 1
  int E, B;
  int S;       // rows per item
};

struct RowsArgs {
  const void *a;          // rows operand: x, or grad_y
  const void *scale;      // act_grad multiplied into a (backward; nullptr: none), [rows, K]
  const void *w;          // weight(s)
  const void *bias;       // [E, N] or nullptr
  const void *res;        // residual or nullptr
  void *c;                // [rows, N]
  void *act_grad;         // forward: act'(z) out, [rows, N], or nullptr
  int64_t lda, ld_res;
  int64_t w_group;        // elements from one group's weight to the next
  int N, K;               // columns of c, length of the sum
  int act;
  int col_tiles;
  int row_tiles;          // bound on the number of row tiles
  int spread;             // row tiles over XCDs (see block_tile)
  Groups g;
};

struct WeightArgs {
  const void *u;          // grad_y
  const void *scale;      // act_grad or nullptr, [rows, N]
  const void *x;
  void *gw, *gb;          // [E, N, K], [E, N] or nullptr
  float *part, *part_b;   // partial sums [slots, N, K], [slots, N] (nullptr: one chunk per group)
  int64_t ldu, ldx;
  int N, K;
  int chunk;              // rows per chunk
  int n_tiles, k_tiles;
  int slots;              // bound on the number of chunks
  Groups g;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

// ---------------------------------------------------------------------------------------------
// element types
template <typename T> struct Type;
template <> struct Type<float> {
  typedef f32x4 frag;
  static constexpr int kPer16 = 4;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ frag ones() { return frag{1.f, 1.f, 1.f, 1.f}; }
};
template <> struct Type<__bf16> {
  typedef __bf16 frag __attribute__((ext_vector_type(8)));
  static constexpr int kPer16 = 8;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag ones() {
    return __builtin_bit_cast(frag, s16x8{0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80});
  }
};
template <> struct Type<_Float16> {
  typedef _Float16 frag __attribute__((ext_vector_type(8)));
  static constexpr int kPer16 = 8;
  static __device__ __forceinline__ f32x4 mma(frag a, frag b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ frag ones() {
    return __builtin_bit_cast(frag, s16x8{0x3c00, 0x3c00, 0x3c00, 0x3c00, 0x3c00, 0x3c00, 0x3c00, 0x3c00});
  }
};

// 16 bytes at any element alignment (the global memory unit takes unaligned 16-byte accesses)
struct __attribute__((packed, aligned(2))) Packed16 {
  uint32_t x, y, z, w;
};
__device__ __forceinline__ uint4 load16(const void *p) {
  const Packed16 v = *static_cast<const Packed16 *>(p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void store16(void *p, uint4 v) {
  *static_cast<Packed16 *>(p) = Packed16{v.x, v.y, v.z, v.w};
}

template <typename T> union Chunk {
  uint4 raw;
  T e[16 / sizeof(T)];
  __device__ __forceinline__ Chunk() {}
};

// The 16-byte chunk at (row, col) of a matrix of nrows x ncols; zeros outside it.
template <typename T>
__device__ __forceinline__ uint4 fetch(const T *base, int64_t ld, int row, int col, int nrows, int ncols) {
  constexpr int CH = 16 / sizeof(T);
  if (row >= nrows || col >= ncols) return make_uint4(0, 0, 0, 0);
  const T *p = base + (int64_t)row * ld + col;
  if (col + CH <= ncols) return load16(p);
  Chunk<T> c;
  c.raw = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < CH; ++i)
    if (col + i < ncols) c.e[i] = p[i];
  return c.raw;
}

// act_grad: fp32 beside fp32, otherwise 16-bit fixed point in steps of 2^-14 (act' lies in
// [-0.13, 1.13]; half a step is 3.1e-5, where bf16 would round by up to 2^-9 of the value), with
// INT16_MIN for NaN.
template <typename T> struct Deriv {
  typedef int16_t type;
  static __device__ __forceinline__ type encode(float d) {
    return d != d ? (int16_t)-32768 : (int16_t)__float2int_rn(d * 16384.f);
  }
  // u * derivative, element by element of a 16-byte chunk
  static __device__ __forceinline__ uint4 apply(uint4 u, uint4 d) {
    Chunk<T> c;
    Chunk<int16_t> s;
    c.raw = u;
    s.raw = d;
    // words with bit 15 set and bit 14 clear hold INT16_MIN: codes of derivatives are >= -2^12
    const uint32_t nan = ((d.x & ~(d.x << 1)) | (d.y & ~(d.y << 1)) | (d.z & ~(d.z << 1)) | (d.w & ~(d.w << 1))) & 0x80008000u;
#pragma unroll
    for (int i = 0; i < 8; ++i) c.e[i] = (T)((float)c.e[i] * ((float)s.e[i] * (1.f / 16384.f)));
    if (nan) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (s.e[i] == -32768) c.e[i] = (T)__builtin_nanf("");
    }
    return c.raw;
  }
};
template <> struct Deriv<float> {
  typedef float type;
  static __device__ __forceinline__ type encode(float d) { return d; }
  static __device__ __forceinline__ uint4 apply(uint4 u, uint4 d) {
    return make_uint4(__float_as_uint(__uint_as_float(u.x) * __uint_as_float(d.x)),
                      __float_as_uint(__uint_as_float(u.y) * __uint_as_float(d.y)),
                      __float_as_uint(__uint_as_float(u.z) * __uint_as_float(d.z)),
                      __float_as_uint(__uint_as_float(u.w) * __uint_as_float(d.w)));
  }
};

// ---------------------------------------------------------------------------------------------
// activations: act(z), and act'(z) in d.  FAST (16-bit outputs): one v_exp and one v_rcp; the error
// function by Abramowitz and Stegun 7.1.26 (absolute error 1.5e-7).
template <bool FAST> __device__ __forceinline__ float sigmoid(float v) {
  if (FAST) return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * v));
  return 1.f / (1.f + expf(-v));
}

template <bool FAST> __device__ __forceinline__ float activate(int act, float z, float &d) {
  switch (act) {
    case kRelu: {
      d = z <= 0.f ? 0.f : 1.f;
      return z <= 0.f ? 0.f : z;
    }
    case kGelu: {
      float phi, cdf;   // sqrt(2 pi) times the normal density, and its distribution
      if (FAST) {
        phi = __builtin_amdgcn_exp2f(-0.72134752f * z * z);
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, fabsf(z), 1.f));
        float p = fmaf(1.061405429f, t, -1.453152027f);
        p = fmaf(p, t, 1.421413741f);
        p = fmaf(p, t, -0.284496736f);
        p = fmaf(p, t, 0.254829592f);
        const float tail = 0.5f * p * t * phi;
        cdf = z > 0.f ? 1.f - tail : tail;
      } else {
        phi = expf(-0.5f * z * z);
        cdf = 0.5f * erfcf(-0.70710678f * z);
      }
      d = fmaf(z * 0.39894228f, phi, cdf);
      return z * cdf;
    }
    case kGeluTanh: {
      // 0.5 (1 + tanh v) = sigmoid(2 v)
      const float z2 = fminf(z * z, 1e18f);   // finite, for its product with s (1 - s) = 0
      const float s = sigmoid<FAST>(z * fmaf(2.f * 0.7978845608f * 0.044715f, z2, 2.f * 0.7978845608f));
      d = fmaf(z * s * (1.f - s), fmaf(6.f * 0.7978845608f * 0.044715f, z2, 2.f * 0.7978845608f), s);
      return z * s;
    }
    case kSilu: {
      const float s = sigmoid<FAST>(z);
      d = fmaf(z * s, 1.f - s, s);
      return z * s;
    }
    default: d = 1.f; return z;
  }
}

// ---------------------------------------------------------------------------------------------
// groups

// Inclusive scans over a wave.
__device__ __forceinline__ int scan_add(int v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o);
    if ((int)(threadIdx.x & 63) >= o) v += t;
  }
  return v;
}
__device__ __forceinline__ int scan_max(int v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o);
    if ((int)(threadIdx.x & 63) >= o) v = max(v, t);
  }
  return v;
}

// Segments of an item: 0 the rows before the first group, e + 1 group e, E + 1 the rows behind the
// last.  One step of a walk over them, 64 at a time, a segment per lane.
struct Segment {
  int lower, upper;   // rows
};
__device__ __forceinline__ Segment segment_at(const Groups &g, int j, int &carry) {
  int64_t v = j < g.count ? g.start[j] : (int64_t)g.S;
  v = v < 0 ? 0 : (v > g.S ? g.S : v);
  Segment s;
  s.upper = max(scan_max((int)v), carry);
  s.lower = __shfl_up(s.upper, 1);
  if ((threadIdx.x & 63) == 0) s.lower = carry;
  carry = __builtin_amdgcn_readlane(s.upper, 63);
  return s;
}

struct RowTile {
  int e;            // weight, or -1: rows of no group
  int64_t first;    // first row, over all items
  int rows;
};

// Row tile t, counted over items, segments and steps of BM rows; false: there is none.  Every wave
// walks the table by itself: E + 2 loads and two scans, no barrier and no kernel before this one.
__device__ __forceinline__ bool find_row_tile(const Groups &g, int t, int BM, RowTile &out) {
  if (!g.start) {
    const int64_t first = (int64_t)t * BM;
    if (first >= g.S) return false;
    out.e = 0;
    out.first = first;
    out.rows = min(BM, (int)(g.S - first));
    return true;
  }
  const int lane = threadIdx.x & 63;
  int b = 0;
  if (g.B > 1) {
    int carry = 0, total = 0;
    for (int base = 0; base < g.E + 2; base += 64) {
      const Segment s = segment_at(g, base + lane, carry);
      total += __builtin_amdgcn_readlane(scan_add((s.upper - s.lower + BM - 1) / BM), 63);
    }
    if (total == 0) return false;
    b = t / total;
    t -= b * total;
    if (b >= g.B) return false;
  }
  int carry = 0, before = 0;
  for (int base = 0; base < g.E + 2; base += 64) {
    const Segment s = segment_at(g, base + lane, carry);
    const int tiles = (s.upper - s.lower + BM - 1) / BM;
    const int incl = before + scan_add(tiles);
    const uint64_t m = __ballot(incl > t);
    if (m) {
      const int src = __builtin_ctzll(m);
      const int lower = __builtin_amdgcn_readlane(s.lower, src), upper = __builtin_amdgcn_readlane(s.upper, src);
      const int step = t - (__builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(tiles, src));
      const int at = lower + step * BM, j = base + src;
      out.e = j <= g.E ? j - 1 : -1;
      out.first = (int64_t)b * g.S + at;
      out.rows = min(BM, upper - at);
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

struct RowChunk {
  int e;
  int64_t first;
  int rows;
  int chunks;       // of this group, all items
  int slot;         // of this group's first chunk
};

// Chunk t of `chunk` rows, counted over groups, items and steps.  by_group: the chunks of group t
// instead (first and rows not set; false never).
__device__ __forceinline__ bool find_chunk(const Groups &g, int t, int chunk, bool by_group, RowChunk &out) {
  if (!g.start) {
    const int n = (g.S + chunk - 1) / chunk;
    out.e = 0;
    out.chunks = n;
    out.slot = 0;
    if (by_group) return true;
    if (t >= n) return false;
    out.first = (int64_t)t * chunk;
    out.rows = min(chunk, (int)(g.S - out.first));
    return true;
  }
  const int lane = threadIdx.x & 63;
  int carry = 0, before = 0;
  for (int base = 0; base < g.E + 2; base += 64) {
    const int j = base + lane;
    const Segment s = segment_at(g, j, carry);
    const int per = j >= 1 && j <= g.E ? (s.upper - s.lower + chunk - 1) / chunk : 0;   // per item
    const int n = per * g.B;
    const int incl = before + scan_add(n);
    const uint64_t m = __ballot(by_group ? j == t + 1 : incl > t);
    if (m) {
      const int src = __builtin_ctzll(m);
      out.e = base + src - 1;
      out.chunks = __builtin_amdgcn_readlane(n, src);
      out.slot = __builtin_amdgcn_readlane(incl, src) - out.chunks;
      if (by_group) return true;
      const int p = __builtin_amdgcn_readlane(per, src), lower = __builtin_amdgcn_readlane(s.lower, src);
      const int r = t - out.slot, b = r / p, at = lower + (r - b * p) * chunk;
      out.first = (int64_t)b * g.S + at;
      out.rows = min(chunk, __builtin_amdgcn_readlane(s.upper, src) - at);
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

// ---------------------------------------------------------------------------------------------
// A stage of an operand tile of R rows (of the output's side): loaded to registers, then to LDS.
// STRIDED: the sum's axis is the matrix's row axis.
template <typename T, int R, int NT, bool STRIDED, bool SCALE> struct Stage {
  static constexpr int CH = 16 / (int)sizeof(T);      // elements of a chunk
  static constexpr int KC = 128 / (int)sizeof(T);     // sum elements of a stage
  static constexpr int NC = R / CH;                   // chunks of a matrix row (STRIDED)
  static constexpr int NL = R * 8 / NT;               // chunks per thread
  static constexpr int kBytes = R * 128;
  static_assert(R * 8 % NT == 0, "chunks divide over the threads");
  uint4 v[NL], d[SCALE ? NL : 1];

  // base: the tile's first element; rows, cols: what is left of the matrix from there
  __device__ __forceinline__ void load(const T *base, int64_t ld, const void *scale, int64_t ld_scale, int rows, int cols,
                                       int k0) {
    typedef typename Deriv<T>::type D;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = threadIdx.x + i * NT;
      const int row = STRIDED ? k0 + c / NC : c >> 3, col = STRIDED ? c % NC * CH : k0 + (c & 7) * CH;
      v[i] = fetch(base, ld, row, col, rows, cols);
      if (SCALE) d[i] = fetch(static_cast<const D *>(scale), ld_scale, row, col, rows, cols);
    }
  }
  __device__ __forceinline__ void store(char *lds) const {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int c = threadIdx.x + i * NT;
      const int row = STRIDED ? c / NC : c >> 3, col = STRIDED ? c % NC : c & 7;
      *reinterpret_cast<uint4 *>(lds + address(row, col)) = SCALE ? Deriv<T>::apply(v[i], d[i]) : v[i];
    }
  }
  // byte address of a 16-byte chunk
  static __device__ __forceinline__ int address(int row, int col) {
    if (!STRIDED) return row * 128 + ((col ^ (row & 7)) << 4);
    return row * (R * (int)sizeof(T)) + ((col ^ (sizeof(T) == 2 ? (row & 3) << 1 : ((row >> 2) & 3) << 2)) << 4);
  }
  // MFMA operand of output rows r0 .. r0 + 15, half `step` of the stage
  static __device__ __forceinline__ typename Type<T>::frag frag(const char *lds, int r0, int step) {
    const int lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
    if constexpr (!STRIDED) {
      return __builtin_bit_cast(typename Type<T>::frag, *reinterpret_cast<const uint4 *>(lds + address(r0 + i, step * 4 + q)));
    } else if constexpr (sizeof(T) == 2) {
      // 16 lanes read 4 matrix rows of 16 elements and get them transposed: lane i column r0 + i
      s16x4 h[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const char *at = lds + address(step * 32 + q * 8 + p * 4 + (i >> 2), (r0 >> 3) + ((i & 3) >> 1)) + (i & 1) * 8;
        h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4 *)(const_cast<char *>(at)));
      }
      return __builtin_bit_cast(typename Type<T>::frag, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      f32x4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *reinterpret_cast<const float *>(lds + address(step * 16 + q * 4 + j, (r0 + i) >> 2) + (i & 3) * 4);
      return __builtin_bit_cast(typename Type<T>::frag, f);
    }
  }
};

// blockIdx -> (row tile, column tile).  spread: the column tiles of a row tile run one after another
// on one XCD, whose L2 then holds the row tile (blocks go to XCD blockIdx % 8); used from 64 row tiles
// on, where every XCD gets its share of them.
__device__ __forceinline__ void block_tile(int bid, int col_tiles, int spread, int &rt, int &ct) {
  if (spread) {
    const int r = bid >> 3;
    ct = r % col_tiles;
    rt = r / col_tiles * 8 + (bid & 7);
  } else {
    ct = bid % col_tiles;
    rt = bid / col_tiles;
  }
}

// Cross-lane traffic through LDS inside one wave: LDS accesses of a wave stay in order; this keeps
// the compiler from moving them.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------------------------------------
// c = epilogue(a w^T) (WSTR = false, w [N, K]) or a w (WSTR = true, w [K, N]) over tiles of BM rows
// and BN columns, WR x WC waves.
template <typename T, int BM, int BN, int WR, int WC, bool WSTR, bool SCALE, bool EPI>
__global__ __launch_bounds__(64 * WR *WC) void rows_kernel(RowsArgs p) {
  constexpr int NT = 64 * WR * WC, TM = BM / WR, TN = BN / WC, MI = TM / 16, NI = TN / 16;
  constexpr int CH = 16 / (int)sizeof(T);
  typedef Stage<T, BM, NT, false, SCALE> SA;
  typedef Stage<T, BN, NT, WSTR, false> SB;
  constexpr int kPad = TN + 4;   // floats of a row of the epilogue's buffer: rows 16 bytes off each other's banks
  constexpr int kEpi = WR * WC * 16 * kPad * 4;
  __shared__ __attribute__((aligned(16))) char lds[SA::kBytes + SB::kBytes > kEpi ? SA::kBytes + SB::kBytes : kEpi];

  int rt, ct;
  block_tile(blockIdx.x, p.col_tiles, p.spread, rt, ct);
  if (rt >= p.row_tiles) return;
  RowTile tile;
  if (!find_row_tile(p.g, rt, BM, tile)) return;
  const int n0 = ct * BN, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int wr = wave / WC, wc = wave % WC;

  f32x4 acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (tile.e >= 0) {
    const T *a = static_cast<const T *>(p.a) + tile.first * p.lda;
    const void *scale = SCALE ? static_cast<const typename Deriv<T>::type *>(p.scale) + tile.first * p.K : nullptr;
    const T *w = static_cast<const T *>(p.w) + tile.e * p.w_group + (WSTR ? (int64_t)n0 : (int64_t)n0 * p.K);
    const int64_t ldw = WSTR ? p.N : p.K;
    const int wrows = WSTR ? p.K : p.N - n0, wcols = WSTR ? p.N - n0 : p.K;
    SA sa;
    SB sb;
    sa.load(a, p.lda, scale, p.K, tile.rows, p.K, 0);
    sb.load(w, ldw, nullptr, 0, wrows, wcols, 0);
    for (int k0 = 0; k0 < p.K; k0 += SA::KC) {
      __syncthreads();
      sa.store(lds);
      sb.store(lds + SA::kBytes);
      __syncthreads();
      if (k0 + SA::KC < p.K) {
        sa.load(a, p.lda, scale, p.K, tile.rows, p.K, k0 + SA::KC);
        sb.load(w, ldw, nullptr, 0, wrows, wcols, k0 + SA::KC);
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        typename Type<T>::frag fb[NI];
#pragma unroll
        for (int n = 0; n < NI; ++n) fb[n] = SB::frag(lds + SA::kBytes, wc * TN + n * 16, s);
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const typename Type<T>::frag fa = SA::frag(lds, wr * TM + m * 16, s);
#pragma unroll
          for (int n = 0; n < NI; ++n) acc[m][n] = Type<T>::mma(fb[n], fa, acc[m][n]);
        }
      }
    }
    __syncthreads();
  }

  // lane (i, q) of acc[m][n]: row m * 16 + i, columns n * 16 + 4 q .. + 3
  float *buf = reinterpret_cast<float *>(lds) + wave * 16 * kPad;
  constexpr int PC = TN / CH;                     // chunks of a row
  constexpr int PN = 16 * PC / 64;                // chunks per lane and 16 rows
  static_assert(64 % PC == 0 && 16 * PC % 64 == 0, "a lane keeps its columns");
  const int c0 = lane % PC * CH, col = n0 + wc * TN + c0, left = p.N - col;
  float bias[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) bias[i] = 0.f;
  if (EPI && p.bias && tile.e >= 0 && left > 0) {
    Chunk<T> b;
    b.raw = fetch(static_cast<const T *>(p.bias) + (int64_t)tile.e * p.N, 0, 0, col, 1, p.N);
#pragma unroll
    for (int i = 0; i < CH; ++i) bias[i] = (float)b.e[i];
  }
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    if (m) wave_fence();
#pragma unroll
    for (int n = 0; n < NI; ++n) *reinterpret_cast<f32x4 *>(buf + (lane & 15) * kPad + n * 16 + (lane >> 4) * 4) = acc[m][n];
    wave_fence();
#pragma unroll
    for (int t = 0; t < PN; ++t) {
      const int r = t * (64 / PC) + lane / PC, row = wr * TM + m * 16 + r;
      if (row >= tile.rows || left <= 0) continue;
      const int64_t grow = tile.first + row;
      float z[CH];
#pragma unroll
      for (int i = 0; i < CH; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(buf + r * kPad + c0 + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) z[i + j] = v[j];
      }
      Chunk<T> out;
      if (EPI && tile.e >= 0) {
        typedef typename Deriv<T>::type D;
        D der[CH];
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          float d;
          z[i] = activate<sizeof(T) == 2>(p.act, z[i] + bias[i], d);
          der[i] = Deriv<T>::encode(d);
        }
        if (p.act_grad) {
          D *dp = static_cast<D *>(p.act_grad) + grow * p.N + col;
          if (left >= CH) {
            store16(dp, __builtin_bit_cast(uint4, der));
          } else {
#pragma unroll
            for (int i = 0; i < CH; ++i)
              if (i < left) dp[i] = der[i];
          }
        }
        if (p.res) {
          Chunk<T> rr;
          rr.raw = fetch(static_cast<const T *>(p.res) + grow * p.ld_res, 0, 0, col, 1, p.N);
#pragma unroll
          for (int i = 0; i < CH; ++i) z[i] += (float)rr.e[i];
        }
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) out.e[i] = (T)z[i];
      T *cp = static_cast<T *>(p.c) + grow * p.N + col;
      if (left >= CH) {
        store16(cp, out.raw);
      } else {
#pragma unroll
        for (int i = 0; i < CH; ++i)
          if (i < left) cp[i] = out.e[i];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows: the weight's bytes bound it.  A block takes 16 columns of up to 16 RT rows; its waves
// share the sum, read the weight straight into MFMA operands (each byte once) and join their sums
// through LDS.
template <typename T, int RT, int NW>
__global__ __launch_bounds__(64 * NW) void few_rows_kernel(RowsArgs p) {
  constexpr int CH = 16 / (int)sizeof(T), KS = 4 * CH;   // sum elements of a step: 16 bytes a lane, 4 lanes a row
  __shared__ f32x4 red[NW][RT][64];
  int rt, ct;
  block_tile(blockIdx.x, p.col_tiles, 0, rt, ct);
  RowTile tile;
  if (!find_row_tile(p.g, rt, 16 * RT, tile)) return;
  const int n0 = ct * 16, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  f32x4 acc[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tile.e >= 0) {
    const T *a = static_cast<const T *>(p.a) + tile.first * p.lda;
    const T *w = static_cast<const T *>(p.w) + tile.e * p.w_group + (int64_t)n0 * p.K;
    constexpr int U = RT <= 2 ? 4 : 2;   // steps in flight
    for (int k0 = wave * KS; k0 < p.K; k0 += NW * KS * U) {
      uint4 fw[U], fa[U][RT];
#pragma unroll
      for (int s = 0; s < U; ++s) {
        const int k = k0 + s * NW * KS + q * CH;
        fw[s] = fetch(w, p.K, i, k, p.N - n0, p.K);
#pragma unroll
        for (int m = 0; m < RT; ++m) fa[s][m] = fetch(a, p.lda, m * 16 + i, k, tile.rows, p.K);
      }
#pragma unroll
      for (int s = 0; s < U; ++s)
#pragma unroll
        for (int m = 0; m < RT; ++m)
          acc[m] = Type<T>::mma(__builtin_bit_cast(typename Type<T>::frag, fw[s]),
                                __builtin_bit_cast(typename Type<T>::frag, fa[s][m]), acc[m]);
    }
  }
#pragma unroll
  for (int m = 0; m < RT; ++m) red[wave][m][lane] = acc[m];
  __syncthreads();
  for (int t = threadIdx.x; t < RT * 64; t += 64 * NW) {
    const int m = t >> 6, l = t & 63, row = m * 16 + (l & 15), col = n0 + (l >> 4) * 4;
    if (row >= tile.rows) continue;
    f32x4 z = red[0][m][l];
#pragma unroll
    for (int w = 1; w < NW; ++w) z += red[w][m][l];
    const int64_t grow = tile.first + row;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (col + j >= p.N) continue;
      float y = z[j];
      if (tile.e >= 0) {
        if (p.bias) y += (float)static_cast<const T *>(p.bias)[(int64_t)tile.e * p.N + col + j];
        float d;
        y = activate<sizeof(T) == 2>(p.act, y, d);
        if (p.act_grad) static_cast<typename Deriv<T>::type *>(p.act_grad)[grow * p.N + col + j] = Deriv<T>::encode(d);
        if (p.res) y += (float)static_cast<const T *>(p.res)[grow * p.ld_res + col + j];
      }
      static_cast<T *>(p.c)[grow * p.N + col + j] = (T)y;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// gw = dz^T x, gb = sum of dz over the rows of a chunk; a chunk that is its group's only one writes
// the results, the others their partial sums.
template <typename T, int BM, int BN, int WR, int WC, bool SCALE>
__global__ __launch_bounds__(64 * WR *WC) void weight_kernel(WeightArgs p) {
  constexpr int NT = 64 * WR * WC, TM = BM / WR, TN = BN / WC, MI = TM / 16, NI = TN / 16;
  typedef Stage<T, BM, NT, true, SCALE> SU;
  typedef Stage<T, BN, NT, true, false> SX;
  __shared__ __attribute__((aligned(16))) char lds[SU::kBytes + SX::kBytes];
  int slot, ct;
  block_tile(blockIdx.x, p.n_tiles * p.k_tiles, 1, slot, ct);
  if (slot >= p.slots) return;
  RowChunk ch;
  if (!find_chunk(p.g, slot, p.chunk, false, ch)) return;
  const int n0 = ct / p.k_tiles * BM, k0 = ct % p.k_tiles * BN;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wr = wave / WC, wc = wave % WC;
  const bool with_b = p.gb && k0 == 0 && wc == 0;   // column sums as products with ones

  f32x4 acc[MI][NI], accb[MI];
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    accb[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const T *u = static_cast<const T *>(p.u) + ch.first * p.ldu + n0;
  const void *scale = SCALE ? static_cast<const typename Deriv<T>::type *>(p.scale) + ch.first * p.N + n0 : nullptr;
  const T *x = static_cast<const T *>(p.x) + ch.first * p.ldx + k0;
  SU su;
  SX sx;
  su.load(u, p.ldu, scale, p.N, ch.rows, p.N - n0, 0);
  sx.load(x, p.ldx, nullptr, 0, ch.rows, p.K - k0, 0);
  for (int r0 = 0; r0 < ch.rows; r0 += SU::KC) {
    __syncthreads();
    su.store(lds);
    sx.store(lds + SU::kBytes);
    __syncthreads();
    if (r0 + SU::KC < ch.rows) {
      su.load(u, p.ldu, scale, p.N, ch.rows, p.N - n0, r0 + SU::KC);
      sx.load(x, p.ldx, nullptr, 0, ch.rows, p.K - k0, r0 + SU::KC);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      typename Type<T>::frag fx[NI];
#pragma unroll
      for (int n = 0; n < NI; ++n) fx[n] = SX::frag(lds + SU::kBytes, wc * TN + n * 16, s);
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const typename Type<T>::frag fu = SU::frag(lds, wr * TM + m * 16, s);
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] = Type<T>::mma(fx[n], fu, acc[m][n]);
        if (with_b) accb[m] = Type<T>::mma(Type<T>::ones(), fu, accb[m]);
      }
    }
  }
  // lane (i, q) of acc[m][n]: row n0 + m * 16 + i of gw, columns k0 + n * 16 + 4 q .. + 3
  const bool direct = ch.chunks == 1;
  const int i = lane & 15, q = lane >> 4;
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int row = n0 + wr * TM + m * 16 + i;
    if (row >= p.N) continue;
#pragma unroll
    for (int n = 0; n < NI && p.gw; ++n) {
      const int col = k0 + wc * TN + n * 16 + q * 4;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (col + j >= p.K) continue;
        if (direct) static_cast<T *>(p.gw)[((int64_t)ch.e * p.N + row) * p.K + col + j] = (T)acc[m][n][j];
        else p.part[((int64_t)slot * p.N + row) * p.K + col + j] = acc[m][n][j];
      }
    }
    if (with_b && q == 0) {
      if (direct) static_cast<T *>(p.gb)[(int64_t)ch.e * p.N + row] = (T)accb[m][0];
      else p.part_b[(int64_t)slot * p.N + row] = accb[m][0];
    }
  }
}

// Sums the chunks' partial results in order; zeros for groups without rows.  Blocks of 64 elements,
// four threads an element, each a quarter of the slots.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(WeightArgs p) {
  __shared__ float red[4][64];
  const int e = blockIdx.y;
  RowChunk ch;
  find_chunk(p.g, e, p.chunk, true, ch);
  if (ch.chunks == 1) return;
  const int64_t nk = p.gw ? (int64_t)p.N * p.K : 0, total = nk + (p.gb ? p.N : 0);
  const int lane = threadIdx.x & 63, part = threadIdx.x >> 6;
  const int per = (ch.chunks + 3) / 4, s0 = part * per, s1 = min(ch.chunks, s0 + per);
  for (int64_t base = (int64_t)blockIdx.x * 64; base < total; base += (int64_t)gridDim.x * 64) {
    const int64_t at = base + lane;
    float sum = 0.f;
    if (at < total) {
      const bool b = at >= nk;
      const float *src = b ? p.part_b + (int64_t)ch.slot * p.N + (at - nk) : p.part + (int64_t)ch.slot * nk + at;
      const int64_t step = b ? p.N : nk;
#pragma unroll 8
      for (int s = s0; s < s1; ++s) sum += src[s * step];
    }
    red[part][lane] = sum;
    __syncthreads();
    if (part == 0 && at < total) {
      const float r = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
      if (at < nk) static_cast<T *>(p.gw)[(int64_t)e * nk + at] = (T)r;
      else static_cast<T *>(p.gb)[(int64_t)e * p.N + (at - nk)] = (T)r;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------
// launches

inline int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Row tiles of BM rows at most: every segment may end inside one.
inline int64_t max_row_tiles(const Groups &g, int BM) {
  if (!g.start) return ceil_div(g.S, BM);
  return (int64_t)g.B * (g.S / BM + g.E + 2);
}

template <typename K> inline hipError_t launch(K kernel, int64_t grid, int threads, hipStream_t st, const RowsArgs &p) {
  if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), 0, st, p);
  return hipGetLastError();
}

template <typename T, int BM, int BN, int WR, int WC, bool WSTR, bool SCALE, bool EPI>
inline hipError_t launch_rows(RowsArgs p, hipStream_t st) {
  const int64_t rt = max_row_tiles(p.g, BM);
  p.row_tiles = (int)rt;
  p.col_tiles = ceil_div(p.N, BN);
  p.spread = rt >= 64;
  const int64_t grid = (p.spread ? (rt + 7) / 8 * 8 : rt) * p.col_tiles;
  return launch(rows_kernel<T, BM, BN, WR, WC, WSTR, SCALE, EPI>, grid, 64 * WR * WC, st, p);
}

template <typename T, int RT, int NW> inline hipError_t launch_few(RowsArgs p, hipStream_t st) {
  const int64_t rt = max_row_tiles(p.g, 16 * RT);
  p.row_tiles = (int)rt;
  p.col_tiles = ceil_div(p.N, 16);
  return launch(few_rows_kernel<T, RT, NW>, rt * p.col_tiles, 64 * NW, st, p);
}

template <typename T, bool WSTR, bool SCALE, bool EPI> inline hipError_t launch_tiles(const RowsArgs &p, hipStream_t st) {
  const int64_t rows = (int64_t)p.g.B * p.g.S;
  if ((rows + 127) / 128 * ceil_div(p.N, 128) >= 256) return launch_rows<T, 128, 128, 2, 2, WSTR, SCALE, EPI>(p, st);
  return launch_rows<T, 64, 64, 2, 2, WSTR, SCALE, EPI>(p, st);
}

template <typename T> hipError_t forward(const RowsArgs &p, hipStream_t st) {
  const int64_t per_group = (int64_t)p.g.B * p.g.S / p.g.E;
  if (per_group <= 16) return p.K >= 2048 ? launch_few<T, 1, 8>(p, st) : launch_few<T, 1, 4>(p, st);
  if (per_group <= 32) return p.K >= 2048 ? launch_few<T, 2, 8>(p, st) : launch_few<T, 2, 4>(p, st);
  if (per_group <= 64) return p.K >= 2048 ? launch_few<T, 4, 8>(p, st) : launch_few<T, 4, 4>(p, st);
  return launch_tiles<T, false, false, true>(p, st);
}

template <typename T> hipError_t grad_x(const RowsArgs &p, hipStream_t st) {
  return p.scale ? launch_tiles<T, true, true, false>(p, st) : launch_tiles<T, true, false, false>(p, st);
}

constexpr int kWeightTile = 128;

// Rows per chunk of the weight kernel and the number of chunks; the workspace follows from it.
struct ChunkPlan {
  int chunk;
  int64_t slots;
  bool joined;   // a group may have several chunks
  ChunkPlan(int esize, bool grouped, int B, int64_t S, int E, int N, int K) {
    const int kc = 128 / esize;
    const int64_t tiles = (int64_t)ceil_div(N, kWeightTile) * ceil_div(K, kWeightTile), rows = (int64_t)B * S;
    int64_t want = 512 / tiles;
    if (want > rows / 256) want = rows / 256;
    if (want <= E) want = 1;
    chunk = (int)((S + kc - 1) / kc * kc);
    if (want > 1) chunk = (int)((rows / want + kc - 1) / kc * kc);
    if (chunk < kc) chunk = kc;
    slots = grouped ? (int64_t)B * (S / chunk + E) : ceil_div(S, chunk);
    joined = grouped ? B > 1 || chunk < S : slots > 1;
  }
};

template <typename T> hipError_t grad_weight(const WeightArgs &q, bool joined, hipStream_t st) {
  WeightArgs p = q;
  p.n_tiles = ceil_div(p.N, kWeightTile);
  p.k_tiles = p.gw ? ceil_div(p.K, kWeightTile) : 1;
  const int64_t grid = ((int64_t)p.slots + 7) / 8 * 8 * p.n_tiles * p.k_tiles;
  if (grid > 0x7fffffff) return hipErrorInvalidConfiguration;
  if (grid > 0) {
    if (p.scale) hipLaunchKernelGGL((weight_kernel<T, kWeightTile, kWeightTile, 2, 2, true>), dim3((unsigned)grid), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((weight_kernel<T, kWeightTile, kWeightTile, 2, 2, false>), dim3((unsigned)grid), dim3(256), 0, st, p);
  }
  if (joined || p.g.start || !p.slots) {
    const int64_t total = (p.gw ? (int64_t)p.N * p.K : 0) + (p.gb ? p.N : 0);
    const int64_t want = (total + 63) / 64, most = joined ? 2048 : 64;
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(want < most ? want : most), p.g.E), dim3(256), 0, st, p);
  }
  return hipGetLastError();
}

// one translation unit per type
extern template hipError_t forward<float>(const RowsArgs &, hipStream_t);
extern template hipError_t forward<_Float16>(const RowsArgs &, hipStream_t);
extern template hipError_t forward<__bf16>(const RowsArgs &, hipStream_t);
extern template hipError_t grad_x<float>(const RowsArgs &, hipStream_t);
extern template hipError_t grad_x<_Float16>(const RowsArgs &, hipStream_t);
extern template hipError_t grad_x<__bf16>(const RowsArgs &, hipStream_t);
extern template hipError_t grad_weight<float>(const WeightArgs &, bool, hipStream_t);
extern template hipError_t grad_weight<_Float16>(const WeightArgs &, bool, hipStream_t);
extern template hipError_t grad_weight<__bf16>(const WeightArgs &, bool, hipStream_t);

}  // namespace ops3d_linear
