// Linear operators (gfx950): y = act(x W^T + b) + r and its gradients, one weight or one per group
// of consecutive rows.
//
// Every product here is a tile product over LDS with fp32 sums in MFMA accumulators:
//   rows kernel     y = x W^T            rows of x by rows of W, both contiguous along the sum
//   rows kernel     dx = dz W            rows of dz by columns of W (W is strided along the sum)
//   weight kernel   dW = dz^T x          both strided along the sum (the rows), split over chunks of
//                                        rows; the chunks' partial sums are joined in order
// but for two kinds of sizes, which the bytes bound:
//   stream kernel   y or dx              many rows, a sum of 128 or 256: the weight stays in registers
//   few rows        y                    64 rows a group at most: the weight goes straight to registers
// A stage of a tile is 128 bytes of the sum's axis for every row (64 elements of 16 bits, 32 of 32).
// Operands that are contiguous along the sum lie in LDS as rows of 128 bytes and are read 16 bytes a
// lane; the others lie as they are in memory, sum axis outermost, and are read transposed
// (ds_read_tr16_b64; single words for fp32).  16-byte chunks are XOR-swizzled so that the lanes of a
// read fall on different banks.
// The weight is the first operand of the MFMA, so a lane holds 4 consecutive output columns of a row, or
// 8 of two results (column_of): whole 16-byte chunks, and the epilogue stays in registers.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

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
  void *dz;               // backward with scale: a * scale out, [rows, K], or nullptr
  int64_t lda, ld_res;
  int64_t w_group;        // elements from one group's weight to the next
  int N, K;               // columns of c, length of the sum
  int act;
  int col_tiles;
  int row_tiles;          // bound on the number of row tiles
  int spread;             // row tiles over XCDs (see block_tile)
  int splits, per_split;  // parts of the sum, and elements of each (SPLIT kernels)
  float *part;            // their sums [splits, rows, N]
  int64_t rows;           // of all items
  unsigned block0;        // blocks in launches before this one
  Groups g;
};

struct WeightArgs {
  const void *u;          // dz: grad_y, or grad_y * act_grad
  const void *x;
  void *gw, *gb;          // [E, N, K], [E, N] or nullptr
  float *part, *part_b;   // partial sums [slots, N, K], [slots, N] (nullptr: one chunk per group)
  int64_t ldu, ldx;
  int N, K;
  int chunk, items;       // rows of an item, and items, per chunk
  int n_tiles, k_tiles;
  int slots;              // bound on the number of chunks
  unsigned block0;        // as RowsArgs'
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

// the same past the caches, for what is next read a whole backward pass away
__device__ __forceinline__ void store16_streaming(void *p, uint4 v) {
  typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(words{v.x, v.y, v.z, v.w}, static_cast<words *>(p));
}

template <typename T> union Chunk {
  uint4 raw;
  T e[16 / sizeof(T)];
  __device__ __forceinline__ Chunk() {}
};

// The first n elements of the chunk at p, zeros behind them; not unrolled: the rare end of a row.
template <typename T> __device__ __forceinline__ uint4 load_part(const T *p, int n) {
  Chunk<T> c;
  c.raw = make_uint4(0, 0, 0, 0);
#pragma unroll 1
  for (int i = n - 1; i >= 0; --i) {
    if (sizeof(T) == 2) {
      c.raw.w = (c.raw.w << 16) | (c.raw.z >> 16);
      c.raw.z = (c.raw.z << 16) | (c.raw.y >> 16);
      c.raw.y = (c.raw.y << 16) | (c.raw.x >> 16);
      c.raw.x <<= 16;
    } else {
      c.raw = make_uint4(0, c.raw.x, c.raw.y, c.raw.z);
    }
    c.raw.x |= sizeof(T) == 2 ? *reinterpret_cast<const uint16_t *>(p + i) : *reinterpret_cast<const uint32_t *>(p + i);
  }
  return c.raw;
}
// The first n elements of a chunk to p.
template <typename T> __device__ __forceinline__ void store_part(T *p, uint4 v, int n) {
#pragma unroll 1
  for (int i = 0; i < n; ++i) {
    if (sizeof(T) == 2) {
      *reinterpret_cast<uint16_t *>(p + i) = (uint16_t)v.x;
      v.x = (v.x >> 16) | (v.y << 16);
      v.y = (v.y >> 16) | (v.z << 16);
      v.z = (v.z >> 16) | (v.w << 16);
      v.w >>= 16;
    } else {
      *reinterpret_cast<uint32_t *>(p + i) = v.x;
      v = make_uint4(v.y, v.z, v.w, 0);
    }
  }
}

// The 16-byte chunk at (row, col) of a matrix of nrows x ncols; zeros outside it.  A chunk that ends
// outside is cut from the row's last 16 bytes.
template <typename T>
__device__ __forceinline__ uint4 fetch(const T *base, int64_t ld, int row, int col, int nrows, int ncols) {
  constexpr int CH = 16 / (int)sizeof(T);
  if (row >= nrows || col >= ncols) return make_uint4(0, 0, 0, 0);
  const T *p = base + (int64_t)row * ld;
  if (col + CH <= ncols) return load16(p + col);
  if (ncols < CH) return load_part(p + col, ncols - col);
  const uint4 v = load16(p + ncols - CH);
  const int bits = (col + CH - ncols) * 8 * (int)sizeof(T);   // 16 .. 112
  const uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
  const uint64_t a = bits < 64 ? lo >> bits | hi << (64 - bits) : hi >> (bits - 64), b = bits < 64 ? hi >> bits : 0;
  return make_uint4((uint32_t)a, (uint32_t)(a >> 32), (uint32_t)b, (uint32_t)(b >> 32));
}

// A chunk of a row with `left` elements left.
template <typename T, bool STREAM = false> __device__ __forceinline__ void store_chunk(T *p, uint4 v, int left) {
  if (left < 16 / (int)sizeof(T)) store_part(p, v, left);
  else if (STREAM) store16_streaming(p, v);
  else store16(p, v);
}

// act_grad: fp32 beside fp32, otherwise 16 bits.  act' lies in [-0.13, 1.13], and a saturated unit's is
// small in every row, so that errors of one sign add up in its gradients: below 1/8 the code is the fp16
// number (half a step is 2^-11 of the value, 2^-25 at least), from there on steps of 2^-14 (half a step is
// 2^-12 of the value at most, 2^-15 near 1; 0 and 1 are exact).  Codes grow with the value, 0x3000 is 1/8 in
// both; NaN is kNan, fp16's with the sign.
template <typename T> struct Deriv {
  typedef int16_t type;
  static constexpr uint32_t kNan = 0xfe00;
  // codes of two values: up to 1/8 as fp16, the steps above added.  v_cvt_pknorm_u16 takes [0, 1] to
  // [0, 65535], rounded to nearest, and what is below to 0.
  static __device__ __forceinline__ uint32_t encode2(float d0, float d1) {
    typedef uint16_t codes __attribute__((ext_vector_type(2)));
    typedef _Float16 halves __attribute__((ext_vector_type(2)));
    constexpr float c = 16384.f / 65535.f;
    const codes low = __builtin_bit_cast(codes, halves{(_Float16)fminf(d0, 0.125f), (_Float16)fminf(d1, 0.125f)});
    const codes steps =
        __builtin_bit_cast(codes, __builtin_amdgcn_cvt_pknorm_u16(fmaf(c, d0, -0.125f * c), fmaf(c, d1, -0.125f * c)));
    return __builtin_bit_cast(uint32_t, low + steps);
  }
  static __device__ __forceinline__ uint4 encode(const float (&d)[8]) {
    uint32_t w[4];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = encode2(d[2 * i], d[2 * i + 1]);
      sum += d[2 * i] + d[2 * i + 1];
    }
    if (sum != sum) {   // derivatives are finite otherwise, and so is their sum
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (d[2 * i] != d[2 * i]) w[i] = (w[i] & 0xffff0000u) | kNan;
        if (d[2 * i + 1] != d[2 * i + 1]) w[i] = (w[i] & 0xffffu) | kNan << 16;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ type encode1(float d) { return (int16_t)(d != d ? kNan : encode2(d, d) & 0xffff); }
  // u * derivative, element by element of a 16-byte chunk
  static __device__ __forceinline__ uint4 apply(uint4 u, uint4 d) {
    typedef int16_t codes __attribute__((ext_vector_type(8)));
    typedef _Float16 halves __attribute__((ext_vector_type(8)));
    Chunk<T> c;
    c.raw = u;
    const codes s = __builtin_bit_cast(codes, d), edge = 0x3000;
    const halves low = __builtin_bit_cast(halves, __builtin_elementwise_min(s, edge));
    const codes steps = __builtin_elementwise_max(s, edge) - edge;
#pragma unroll
    for (int i = 0; i < 8; ++i) c.e[i] = (T)((float)c.e[i] * fmaf((float)steps[i], 1.f / 16384.f, (float)low[i]));
    return c.raw;
  }
};
template <> struct Deriv<float> {
  typedef float type;
  static __device__ __forceinline__ uint4 encode(const float (&d)[4]) {
    return make_uint4(__float_as_uint(d[0]), __float_as_uint(d[1]), __float_as_uint(d[2]), __float_as_uint(d[3]));
  }
  static __device__ __forceinline__ type encode1(float d) { return d; }
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
      if (FAST) {
        // tail = P(X > |z|), w = |z| times the density: act = max(z, 0) - |z| tail, and act' is
        // tail - w below zero and 1 minus that above
        const float e = __builtin_amdgcn_exp2f(-0.72134752f * z * z), a = fminf(fabsf(z), 1e4f);   // finite: e = 0 there
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678f, a, 1.f));
        float p = fmaf(0.5f * 1.061405429f, t, 0.5f * -1.453152027f);
        p = fmaf(p, t, 0.5f * 1.421413741f);
        p = fmaf(p, t, 0.5f * -0.284496736f);
        p = fmaf(p, t, 0.5f * 0.254829592f);
        const float tail = p * t * e;
        const float g = fmaf(-0.39894228f * a, e, tail);
        d = z > 0.f ? 1.f - g : g;
        return fmaf(-a, tail, z > 0.f ? z : 0.f);
      }
      const float phi = expf(-0.5f * z * z), cdf = 0.5f * erfcf(-0.70710678f * z);
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

// The row tiles of one segment of one item: tiles lo .. hi - 1, of `rows` rows from `first` on.
struct SegmentTiles {
  int e, lo, hi, rows;
  int64_t first;
};

// The segment of row tile t, counted over items, segments and steps of BM rows; false: there is none.
// Every wave walks the table by itself: E + 2 loads and two scans, no barrier and no kernel before
// this one.
__device__ __forceinline__ bool find_segment(const Groups &g, int t, int BM, SegmentTiles &out) {
  if (!g.start) {
    out = SegmentTiles{0, 0, (g.S + BM - 1) / BM, g.S, 0};
    return t < out.hi;
  }
  const int lane = threadIdx.x & 63;
  int b = 0, skipped = 0;
  if (g.B > 1) {
    int carry = 0, total = 0;
    for (int base = 0; base < g.E + 2; base += 64) {
      const Segment s = segment_at(g, base + lane, carry);
      total += __builtin_amdgcn_readlane(scan_add((s.upper - s.lower + BM - 1) / BM), 63);
    }
    if (total == 0) return false;
    b = t / total;
    skipped = b * total;
    if (b >= g.B) return false;
  }
  int carry = 0, before = skipped;
  for (int base = 0; base < g.E + 2; base += 64) {
    const Segment s = segment_at(g, base + lane, carry);
    const int tiles = (s.upper - s.lower + BM - 1) / BM;
    const int incl = before + scan_add(tiles);
    const uint64_t m = __ballot(incl > t);
    if (m) {
      const int src = __builtin_ctzll(m), j = base + src;
      const int lower = __builtin_amdgcn_readlane(s.lower, src);
      out.e = j <= g.E ? j - 1 : -1;
      out.hi = __builtin_amdgcn_readlane(incl, src);
      out.lo = out.hi - __builtin_amdgcn_readlane(tiles, src);
      out.rows = __builtin_amdgcn_readlane(s.upper, src) - lower;
      out.first = (int64_t)b * g.S + lower;
      return true;
    }
    before = __builtin_amdgcn_readlane(incl, 63);
  }
  return false;
}

__device__ __forceinline__ bool find_row_tile(const Groups &g, int t, int BM, RowTile &out) {
  SegmentTiles s;
  if (!find_segment(g, t, BM, s)) return false;
  const int at = (t - s.lo) * BM;
  out = RowTile{s.e, s.first + at, min(BM, s.rows - at)};
  return true;
}

struct RowChunk {
  int e;
  int64_t first;
  int rows, items;  // rows from `first` on, and the same of the items - 1 next items
  int chunks;       // of this group, all items
  int slot;         // of this group's first chunk
};

// Chunk t of `chunk` rows of each of `items` items, counted over groups, runs of items and steps; a group
// without rows has one of no rows in each run, which writes its zeros.  by_group: the chunks of group t
// instead (first, rows and items not set; false never).
__device__ __forceinline__ bool find_chunk(const Groups &g, int t, int chunk, int items, bool by_group, RowChunk &out) {
  if (!g.start) {
    const int n = max(1, (g.S + chunk - 1) / chunk);
    out.e = 0;
    out.chunks = n;
    out.slot = 0;
    if (by_group) return true;
    if (t >= n) return false;
    out.first = (int64_t)t * chunk;
    out.rows = min(chunk, (int)(g.S - out.first));
    out.items = 1;
    return true;
  }
  const int lane = threadIdx.x & 63;
  int carry = 0, before = 0;
  for (int base = 0; base < g.E + 2; base += 64) {
    const int j = base + lane;
    const Segment s = segment_at(g, j, carry);
    const int per = j >= 1 && j <= g.E ? max(1, (s.upper - s.lower + chunk - 1) / chunk) : 0;   // per run of items
    const int n = per * ((g.B + items - 1) / items);
    const int incl = before + scan_add(n);
    const uint64_t m = __ballot(by_group ? j == t + 1 : incl > t);
    if (m) {
      const int src = __builtin_ctzll(m);
      out.e = base + src - 1;
      out.chunks = __builtin_amdgcn_readlane(n, src);
      out.slot = __builtin_amdgcn_readlane(incl, src) - out.chunks;
      if (by_group) return true;
      const int p = __builtin_amdgcn_readlane(per, src), lower = __builtin_amdgcn_readlane(s.lower, src);
      const int r = t - out.slot, run = r / p, b = run * items, at = lower + (r - run * p) * chunk;
      out.first = (int64_t)b * g.S + at;
      out.items = min(items, g.B - b);
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
template <typename T, int R, int NT, bool STRIDED> struct Stage {
  static constexpr int CH = 16 / (int)sizeof(T);      // elements of a chunk
  static constexpr int KC = 128 / (int)sizeof(T);     // sum elements of a stage
  static constexpr int NC = R / CH;                   // chunks of a matrix row (STRIDED)
  static constexpr int NL = R * 8 / NT;               // chunks per thread
  static constexpr int kBytes = R * 128;
  static_assert(R * 8 % NT == 0, "chunks divide over the threads");

  // matrix row and column of chunk i of this thread, from the tile's first element, in stage 0
  static __device__ __forceinline__ int row_of(int i) {
    const int c = threadIdx.x + i * NT;
    return STRIDED ? c / NC : c >> 3;
  }
  static __device__ __forceinline__ int col_of(int i) {
    const int c = threadIdx.x + i * NT;
    return STRIDED ? c % NC * CH : (c & 7) * CH;
  }
  static constexpr int kRowStep = STRIDED ? NT / NC : NT / 8;   // matrix rows between a thread's chunks
  static constexpr int kRowBytes = STRIDED ? R * (int)sizeof(T) : 128;

  // Chunks of one stage.  base: the tile's first element; rows, cols: what is left of the matrix from
  // there; k0: sum elements before this stage.  A stage of a whole tile takes 16-byte loads at one
  // 32-bit offset a thread and scalar bases.  One that lacks some of the output's side reads the last
  // row for it, or, STRIDED, its columns' last chunk, whose end may lie in the next row, so not in the
  // matrix's last row (the results of such rows and columns are not stored).  Others go chunk by chunk
  // with zeros outside.
  template <typename E>
  static __device__ __forceinline__ void load(uint4 (&v)[NL], const E *base, int64_t ld, int rows, int cols, int k0) {
    const E *at = base + (STRIDED ? (int64_t)k0 * ld : (int64_t)k0);
    const bool inside = k0 + KC <= (STRIDED ? rows : cols) && ld < (1 << 22);
    if (inside && (STRIDED ? cols : rows) >= R) {
      const uint32_t off = row_of(0) * (int)ld + col_of(0);
#pragma unroll
      for (int i = 0; i < NL; ++i) v[i] = load16(at + (int64_t)i * kRowStep * ld + off);
    } else if (inside && (!STRIDED || (k0 + KC < rows && ld >= CH))) {
      int last = STRIDED ? (cols - 1) / CH * CH : rows - 1;
      asm volatile("" : "+v"(last));   // the offsets are formed here, not in every block before its loop
#pragma unroll
      for (int i = 0; i < NL; ++i)
        v[i] = STRIDED ? load16(at + (uint32_t)(row_of(i) * (int)ld + min(col_of(i), last)))
                       : load16(at + (uint32_t)(min(row_of(i), last) * (int)ld + col_of(i)));
    } else {
      int zero = 0;
      asm volatile("" : "+v"(zero));
#pragma unroll
      for (int i = 0; i < NL; ++i)
        v[i] = fetch(base, ld, row_of(i) + (STRIDED ? k0 : zero), col_of(i) + (STRIDED ? zero : k0), rows, cols);
    }
  }
  static __device__ __forceinline__ void store(char *lds, const uint4 (&v)[NL]) {
    if constexpr (kRowStep % 16 == 0) {   // the swizzle looks at the row's lower 4 bits
      char *at = lds + address(row_of(0), col_of(0) / CH);
#pragma unroll
      for (int i = 0; i < NL; ++i) *reinterpret_cast<uint4 *>(at + i * kRowStep * kRowBytes) = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < NL; ++i) *reinterpret_cast<uint4 *>(lds + address(row_of(i), col_of(i) / CH)) = v[i];
    }
  }
  // Byte address of a 16-byte chunk.  Rows of 128 bytes: 8 rows that follow each other, and 8 that a lane
  // octet reads in the order of column_of (4 h + 0 .. 3 of two groups of 8), fall on 8 different chunks.
  // STRIDED: the 4 matrix rows that 16 lanes read (fp32: the rows that the lane quarters read) fall on
  // different chunks, for columns that follow each other and for those of column_of.
  static __device__ __forceinline__ int swizzle(int row) {
    if (!STRIDED) return (row & 3) | (((row >> 2) ^ (row >> 3)) & 1) << 2;
    return (sizeof(T) == 2 ? row & 3 : (row >> 2) & 3) << (sizeof(T) == 4 || NC >= 16 ? 2 : 1);
  }
  static __device__ __forceinline__ int address(int row, int col) { return row * kRowBytes + ((col ^ swizzle(row)) << 4); }

  // A stage inside the matrix straight to LDS, without registers between: an instruction of a wave fills
  // 1024 bytes in lane order, so the lane at a place loads the chunk that the swizzle puts there.  Needs
  // rows that start at 16-byte boundaries and, STRIDED, cols a multiple of CH; sides beyond the matrix
  // read its last row or chunk (their results are not stored).
  static __device__ __forceinline__ void load_lds(char *lds, const T *base, int64_t ld, int rows, int cols, int k0) {
    constexpr int kRowChunks = kRowBytes / 16;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const T *at = base + (STRIDED ? (int64_t)k0 * ld : (int64_t)k0);
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int slot = (wave * NL + j) * 64 + lane, row = slot / kRowChunks, col = ((slot % kRowChunks) ^ swizzle(row)) * CH;
      const uint32_t off = STRIDED ? (uint32_t)(row * (int)ld + min(col, cols - CH))
                                   : (uint32_t)(min(row, rows - 1) * (int)ld + col);
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(at + off),
                                       (__attribute__((address_space(3))) void *)(lds + (wave * NL + j) * 1024), 16, 0, 0);
    }
  }
  // A stage that ends inside the matrix, chunk by chunk with zeros behind it.
  static __device__ __forceinline__ void load_end(char *lds, const T *base, int64_t ld, int rows, int cols, int k0) {
#pragma unroll 1
    for (int c = threadIdx.x; c < R * 8; c += NT) {
      const int row = STRIDED ? c / NC : c >> 3, col = STRIDED ? c % NC : c & 7;
      *reinterpret_cast<uint4 *>(lds + address(row, col)) =
          fetch(base, ld, row + (STRIDED ? k0 : 0), col * CH + (STRIDED ? 0 : k0), rows, cols);
    }
  }
  static __device__ __forceinline__ void load_either(char *lds, const T *base, int64_t ld, int rows, int cols, int k0) {
    if (k0 + KC <= (STRIDED ? rows : cols)) load_lds(lds, base, ld, rows, cols, k0);
    else load_end(lds, base, ld, rows, cols, k0);
  }
  // MFMA operand, half `step` of the stage, of 16 output rows: r0 + row(i) for lane index i
  template <typename F> static __device__ __forceinline__ typename Type<T>::frag frag(const char *lds, int step, F row, int lane) {
    const int i = lane & 15, q = lane >> 4;
    if constexpr (!STRIDED) {
      return __builtin_bit_cast(typename Type<T>::frag, *reinterpret_cast<const uint4 *>(lds + address(row(i), step * 4 + q)));
    } else if constexpr (sizeof(T) == 2) {
      // 16 lanes read 4 matrix rows of 16 elements, 4 elements a lane, and get them transposed: lane i
      // has the elements that lanes i / 4, 4 + i / 4, .. read at place i % 4
      s16x4 h[2];
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int c = row((i & 3) * 4);
        const char *at = lds + address(step * 32 + q * 8 + p * 4 + (i >> 2), c >> 3) + (c & 7) * 2;
        h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4 *)(const_cast<char *>(at)));
      }
      return __builtin_bit_cast(typename Type<T>::frag, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      f32x4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *reinterpret_cast<const float *>(lds + address(step * 16 + q * 4 + j, row(i) >> 2) + (row(i) & 3) * 4);
      return __builtin_bit_cast(typename Type<T>::frag, f);
    }
  }
};

// The output columns of the MFMA rows: a lane holds rows 4 q .. 4 q + 3 of each 16-row result.  In 16
// bits results 2 t and 2 t + 1 take columns 32 t + 8 q .. + 3 and .. + 4 .. + 7, so that a lane holds 8
// consecutive columns, a 16-byte chunk; in fp32 4 columns are one already.
template <typename T> __device__ __forceinline__ int column_of(int n, int i) {
  if (sizeof(T) == 4) return n * 16 + i;
  return (n >> 1) * 32 + (i >> 2) * 8 + (n & 1) * 4 + (i & 3);
}

// block -> (row tile, column tile).  spread: the column tiles of a row tile run one after another
// on one XCD, whose L2 then holds the row tile (blocks go to XCD block % 8); used from 64 row tiles
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

// The results of a wave: rows r0 + 16 m + lane & 15 of the tile, columns col0 + column_of of acc[m][..],
// with activation and residual.  FULL: all inside.  A row's chunks follow one another, so that the
// 64-byte pieces of a line are stored together (and 22 % faster than column by column, 73728 x 1024
// bf16 with act_grad); act_grad goes past the caches (120 -> 95 us there).
template <typename T, int MI, int NI, bool EPI, int ACT, bool FULL>
__device__ __forceinline__ void store_results(const RowsArgs &p, const f32x4 (&acc)[MI][NI], const RowTile &tile, int r0,
                                              int col0, int lane) {
  constexpr int CH = 16 / (int)sizeof(T), NP = CH / 4;   // MFMA results that make up a chunk of columns
  constexpr int NC = NI / NP;
  typedef typename Deriv<T>::type D;
  const int row0 = r0 + (lane & 15), c0 = (lane >> 4) * CH;
  const int64_t at = tile.first * p.N + col0;                    // uniform
  const uint32_t off = (uint32_t)row0 * (uint32_t)p.N + c0;      // the rest: below 256 rows of 2^24
  const T *res = EPI && p.res ? static_cast<const T *>(p.res) + tile.first * p.ld_res + col0 : nullptr;
  const int64_t off_res = row0 * p.ld_res + c0;
  uint4 r[NC];
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    if (!FULL && row0 + m * 16 >= tile.rows) continue;
    if (EPI && res) {   // of these 16 rows, all on their way before the first is waited for
#pragma unroll
      for (int t = 0; t < NC; ++t) {
        const T *from = res + (int64_t)m * 16 * p.ld_res + t * NP * 16 + off_res;
        r[t] = FULL ? load16(from) : fetch(from, 0, 0, 0, 1, p.N - col0 - c0 - t * NP * 16);
      }
    }
#pragma unroll
    for (int t = 0; t < NC; ++t) {
      const int cols = t * NP * 16, left = FULL ? CH : p.N - col0 - c0 - cols;
      if (!FULL && left <= 0) continue;
      const int64_t to = at + (int64_t)m * 16 * p.N + cols;      // uniform
      float z[CH], d[CH];
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        z[i] = acc[m][t * NP + i / 4][i & 3];
        if (EPI) z[i] = activate<sizeof(T) == 2>(ACT, z[i], d[i]);
      }
      if (EPI && ACT != kNone && p.act_grad) store_chunk<D, true>(static_cast<D *>(p.act_grad) + to + off, Deriv<T>::encode(d), left);
      if (EPI && res) {
        Chunk<T> c;
        c.raw = r[t];
#pragma unroll
        for (int i = 0; i < CH; ++i) z[i] += (float)c.e[i];
      }
      Chunk<T> out;
#pragma unroll
      for (int i = 0; i < CH; ++i) out.e[i] = (T)z[i];
      store_chunk<T>(static_cast<T *>(p.c) + to + off, out.raw, left);
      __builtin_amdgcn_sched_barrier(0);   // chunk by chunk: together they would not fit the registers
    }
  }
}
template <typename T, int MI, int NI, bool EPI, bool FULL>
__device__ __forceinline__ void finish_tile(const RowsArgs &p, const f32x4 (&acc)[MI][NI], const RowTile &tile, int r0, int col0,
                                            int lane) {
  if constexpr (!EPI) {
    store_results<T, MI, NI, false, kNone, FULL>(p, acc, tile, r0, col0, lane);
  } else if (tile.e < 0) {
    store_results<T, MI, NI, false, kNone, FULL>(p, acc, tile, r0, col0, lane);
  } else {
    switch (p.act) {
      case kRelu: store_results<T, MI, NI, true, kRelu, FULL>(p, acc, tile, r0, col0, lane); break;
      case kGelu: store_results<T, MI, NI, true, kGelu, FULL>(p, acc, tile, r0, col0, lane); break;
      case kGeluTanh: store_results<T, MI, NI, true, kGeluTanh, FULL>(p, acc, tile, r0, col0, lane); break;
      case kSilu: store_results<T, MI, NI, true, kSilu, FULL>(p, acc, tile, r0, col0, lane); break;
      default: store_results<T, MI, NI, true, kNone, FULL>(p, acc, tile, r0, col0, lane); break;
    }
  }
}

// The results of a wave as one part of a split sum.
template <typename T, int MI, int NI>
__device__ __forceinline__ void store_parts(const RowsArgs &p, const f32x4 (&acc)[MI][NI], const RowTile &tile, int r0,
                                            int col0, int part) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int row = r0 + m * 16 + (lane & 15);
    if (row >= tile.rows) continue;
#pragma unroll
    for (int n = 0; n < NI; ++n) {
      const int col = col0 + column_of<T>(n, (lane >> 4) * 4);
      if (col < p.N)
        store_chunk<float>(p.part + (part * p.rows + tile.first + row) * p.N + col, __builtin_bit_cast(uint4, acc[m][n]), p.N - col);
    }
  }
}

// ---------------------------------------------------------------------------------------------
// c = epilogue(a w^T) (WSTR = false, w [N, K]) or a w (WSTR = true, w [K, N]) over tiles of BM rows
// and BN columns, WR x WC waves.  SCALE: a is grad_y * act_grad, and the first column's tiles store
// it for the weights' gradients.  SPLIT: a block sums a part of the sum's axis only and stores it for
// split_join_kernel, where the tiles alone do not fill the CUs.
// U stages are loaded and multiplied at a time.  DMA: loads go straight to LDS (rows at 16-byte
// boundaries); nothing is loaded ahead, but without registers for it more blocks fit a CU, which wait in
// turn (4096^3 bf16, same run: 128 x 256 136 us, 128 x 128 144; through registers and a stage ahead 256 x 256
// 159, 128 x 128 189; 130 to 136 from run to run, where a library's bare product takes 94).
// What bounds it: at long sums the wait for a stage's loads, which the blocks of a CU hide from one another
// (half of the wave cycles wait, for 4096^3); at 73728 x 256 -> 1024 with an act_grad (97 to 125
// us) the stores, of 300 MB, and the activation's arithmetic.  Otherwise loads go through registers, the
// next stages' while these are multiplied; so does the scaled operand always.  That is rounded to T, as the
// matrix units take no more, and stored so: dW and db sum the same dz.
template <typename T, int BM, int BN, int WR, int WC, int U, bool DMA, int OCC, bool WSTR, bool SCALE, bool EPI, bool SPLIT>
__global__ __launch_bounds__(64 * WR *WC) __attribute__((amdgpu_waves_per_eu(OCC))) void rows_kernel(RowsArgs p) {
  constexpr int NT = 64 * WR * WC, TM = BM / WR, TN = BN / WC, MI = TM / 16, NI = TN / 16;
  typedef Stage<T, BM, NT, false> SA;
  typedef Stage<T, BN, NT, WSTR> SB;
  typedef typename Deriv<T>::type D;
  constexpr int kStage = SA::kBytes + SB::kBytes;
  __shared__ __attribute__((aligned(16))) char lds[U * kStage];

  const int block = blockIdx.x + p.block0, part = SPLIT ? block % p.splits : 0;
  int rt, ct;
  block_tile(SPLIT ? block / p.splits : block, p.col_tiles, p.spread, rt, ct);
  if (rt >= p.row_tiles) return;
  RowTile tile;
  if (!find_row_tile(p.g, rt, BM, tile)) return;
  const int n0 = ct * BN, wave = threadIdx.x >> 6, q = (threadIdx.x & 63) >> 4;
  const int wr = wave / WC, wc = wave % WC;

  f32x4 acc[MI][NI];   // lane (i, q) of [m][n]: row 16 m + i, columns column_of(n, 4 q) .. + 3
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (tile.e >= 0) {
    const T *a = static_cast<const T *>(p.a) + tile.first * p.lda;
    const D *scale = SCALE ? static_cast<const D *>(p.scale) + tile.first * p.K : nullptr;
    T *dz = SCALE && ct == 0 && p.dz ? static_cast<T *>(p.dz) + tile.first * p.K : nullptr;
    const T *w = static_cast<const T *>(p.w) + tile.e * p.w_group + (WSTR ? (int64_t)n0 : (int64_t)n0 * p.K);
    const int64_t ldw = WSTR ? p.N : p.K;
    const int wrows = WSTR ? p.K : p.N - n0, wcols = WSTR ? p.N - n0 : p.K;
    const int first = SPLIT ? part * p.per_split : 0, end = SPLIT ? min(p.K, first + p.per_split) : p.K;
    constexpr int kStep = U * SA::KC;
    constexpr bool kRegA = !DMA || SCALE;
    uint4 va[kRegA ? U : 1][kRegA ? SA::NL : 1], vd[SCALE ? U : 1][SCALE ? SA::NL : 1], vb[DMA ? 1 : U][DMA ? 1 : SB::NL];
    const auto load = [&](int k0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u && k0 + u * SA::KC >= end) break;
        if constexpr (kRegA) SA::load(va[u], a, p.lda, tile.rows, p.K, k0 + u * SA::KC);
        if constexpr (SCALE) SA::load(vd[u], scale, p.K, tile.rows, p.K, k0 + u * SA::KC);
        if constexpr (!DMA) SB::load(vb[u], w, ldw, wrows, wcols, k0 + u * SA::KC);
      }
    };
    if (kRegA) load(first);
    for (int k0 = first; k0 < end; k0 += kStep) {
      if (k0 > first) __syncthreads();
      if constexpr (DMA) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (u && k0 + u * SA::KC >= end) break;
          if constexpr (!SCALE) SA::load_either(lds + u * kStage, a, p.lda, tile.rows, p.K, k0 + u * SA::KC);
          SB::load_either(lds + u * kStage + SA::kBytes, w, ldw, wrows, wcols, k0 + u * SA::KC);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u && k0 + u * SA::KC >= end) break;
        if constexpr (SCALE) {
#pragma unroll
          for (int i = 0; i < SA::NL; ++i) {
            va[u][i] = Deriv<T>::apply(va[u][i], vd[u][i]);
            const int row = SA::row_of(i), col = k0 + u * SA::KC + SA::col_of(i), left = p.K - col;
            if (dz && row < tile.rows && left > 0) store_chunk<T>(dz + (int64_t)row * p.K + col, va[u][i], left);
          }
        }
        if constexpr (kRegA) SA::store(lds + u * kStage, va[u]);
        if constexpr (!DMA) SB::store(lds + u * kStage + SA::kBytes, vb[u]);
      }
      if (DMA) __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's loads are in LDS
      if (kRegA && k0 + kStep < end) load(k0 + kStep);
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 2 * U; ++s) {
        if (s >= 2 && k0 + (s >> 1) * SA::KC >= end) break;
        const char *const la = lds + (s >> 1) * kStage, *const lb = la + SA::kBytes;
        typename Type<T>::frag fb[NI];
#pragma unroll
        for (int n = 0; n < NI; ++n)
          fb[n] = SB::frag(lb, s & 1, [&](int i) { return wc * TN + column_of<T>(n, i); }, threadIdx.x & 63);
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const typename Type<T>::frag fa = SA::frag(la, s & 1, [&](int i) { return wr * TM + m * 16 + i; }, threadIdx.x & 63);
#pragma unroll
          for (int n = 0; n < NI; ++n) acc[m][n] = Type<T>::mma(fb[n], fa, acc[m][n]);
        }
      }
    }
  }

  if constexpr (SPLIT) {
    if (tile.e >= 0) store_parts<T, MI, NI>(p, acc, tile, wr * TM, n0 + wc * TN, part);
    return;
  }
  if (EPI && p.bias && tile.e >= 0) {
    constexpr int CH = 16 / (int)sizeof(T), NP = CH / 4;
#pragma unroll
    for (int t = 0; t < NI / NP; ++t) {
      Chunk<T> b;
      b.raw = fetch(static_cast<const T *>(p.bias) + (int64_t)tile.e * p.N, 0, 0, n0 + wc * TN + t * NP * 16 + q * CH, 1, p.N);
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int i = 0; i < CH; ++i) acc[m][t * NP + i / 4][i & 3] += (float)b.e[i];
    }
  }
  if (tile.rows >= BM && n0 + BN <= p.N) finish_tile<T, MI, NI, EPI, true>(p, acc, tile, wr * TM, n0 + wc * TN, threadIdx.x & 63);
  else finish_tile<T, MI, NI, EPI, false>(p, acc, tile, wr * TM, n0 + wc * TN, threadIdx.x & 63);
}

// ---------------------------------------------------------------------------------------------
// Many rows, a short sum (16-bit types, K = 64 KS, no scale), as projections of whole volumes are: bound by
// the rows' bytes.  The tile kernel reads its operands through LDS once for every 128 columns or rows,
// waits for every stage of every tile and has no more than its LDS's bytes under way (598016 x 256 ->
// 1024 570 to 690 us).  Here a block of 8 waves stays on its CU with 256 columns of the weight in
// registers (64 a wave: 32 KS registers) and walks over tiles of 64 rows: loads to a ring of four tiles in
// LDS run two to three tiles ahead of the products, one barrier a tile, and results go out meanwhile
// (390 to 450 us; with 256 columns 114 to 123, 171 in tiles, where the bytes alone take 118).
// A segment's last tile is its last 64 rows, and the last columns are the last 256: what two blocks
// compute they write alike, and every tile is whole.
//
// Order of a wave's memory operations, which complete in order: loads of tile i (KS of them), results of
// tile i - 3, loads of tile i + 1, results of i - 2, loads of i + 2, results of i - 1.  So when all but the
// newest 2 KS operations are done, the loads of tile i are, with results to store or without.  A residual's
// loads come behind those of tile i + 3, so waiting for them waits for these too; it costs no more than its
// bytes (598016 x 256 -> 256 bf16 123 us, 173 with a residual, 177 in bytes).  Behind the
// barrier every wave's are, and every wave has read tile i - 1 (the reads' results are waited for where
// they are read), whose place tile i + 3 takes.  Behind the last tile it is loaded again, so the counts
// hold, and all loads are waited for before a segment ends.
// The operands are read in assembly with the wait in the same statement: for its own reads of LDS the
// compiler waits for all loads to LDS under way.
template <int OFF> __device__ __forceinline__ void read_rows(f32x4 (&x)[4], uint32_t even, uint32_t odd) {
  asm volatile(
      "ds_read_b128 %0, %4 offset:%6\n\tds_read_b128 %1, %4 offset:%7\n\t"
      "ds_read_b128 %2, %5 offset:%6\n\tds_read_b128 %3, %5 offset:%7\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3])
      : "v"(even), "v"(odd), "n"(OFF), "n"(OFF + 16 * 128)
      : "memory");
}

template <typename T, int KS, bool WSTR, bool EPI, int ACT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void stream_kernel(RowsArgs p) {
  constexpr int BM = 64, NB = 256, NI = 4, ST = 2 * KS;
  typedef Stage<T, NB, 512, WSTR> SB;
  typedef Stage<T, BM, 512, false> SA;
  constexpr int kTile = KS * SA::kBytes;
  static_assert(KS * SB::kBytes == 4 * kTile, "the weight's columns pass through the ring");
  static_assert(SA::NL == 1, "a stage of rows is one load a thread");
  __shared__ __attribute__((aligned(16))) char lds[4 * kTile];
  const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, ct = slot % p.col_tiles;
  const int groups = gridDim.x / 8 / p.col_tiles * 8;
  const int n0 = min(ct * NB, p.N - NB);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, q = lane >> 4;
  const int wr = wave >> 2, col0 = n0 + (wave & 3) * 64;   // the wave has 32 rows and 64 columns of a tile
  const int64_t ldw = WSTR ? p.N : p.K;
  // LDS addresses of this lane's operands of tile 0: even and odd steps of 32
  const uint32_t ring = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
  const uint32_t even = ring + SA::address(wr * 32 + li, q), odd = ring + SA::address(wr * 32 + li, 4 + q);

  int rt = slot / p.col_tiles * 8 + xcd;
  while (rt < p.row_tiles) {
    SegmentTiles seg;
    if (!find_segment(p.g, rt, BM, seg)) return;
    // first row of tile t of the segment
    const auto first_row = [&](int t) { return seg.first + max(0, min((t - seg.lo) * BM, seg.rows - BM)); };
    const auto load_tile = [&](int t, int buf) {
      const T *a = static_cast<const T *>(p.a) + first_row(t) * p.lda;
#pragma unroll
      for (int k = 0; k < KS; ++k) SA::load_lds(lds + buf * kTile + k * SA::kBytes, a, p.lda, min(seg.rows, BM), p.K, k * 64);
    };
    if (seg.e < 0) {
      for (; rt < seg.hi; rt += groups) {
        f32x4 zero[2][NI];
#pragma unroll
        for (int n = 0; n < NI; ++n) zero[0][n] = zero[1][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        const RowTile tile{-1, first_row(rt), min(seg.rows, BM)};
        store_results<T, 2, NI, false, kNone, false>(p, zero, tile, wr * 32, col0, lane);
      }
      continue;
    }

    // the weight's columns, through the ring, and the bias
    const T *w = static_cast<const T *>(p.w) + seg.e * p.w_group + (WSTR ? (int64_t)n0 : (int64_t)n0 * p.K);
    typename Type<T>::frag fw[NI][ST];
    uint4 bias[2];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KS; ++k) SB::load_lds(lds + k * SB::kBytes, w, ldw, WSTR ? p.K : NB, WSTR ? NB : p.K, k * 64);
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int s = 0; s < ST; ++s)
        fw[n][s] = SB::frag(lds + (s >> 1) * SB::kBytes, s & 1, [&](int i) { return (wave & 3) * 64 + column_of<T>(n, i); }, lane);
    if constexpr (EPI)
#pragma unroll
      for (int t = 0; t < 2; ++t)
        bias[t] = p.bias ? load16(static_cast<const T *>(p.bias) + (int64_t)seg.e * p.N + col0 + t * 32 + q * 8) : make_uint4(0, 0, 0, 0);
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0): the weight is read, the ring free
    __syncthreads();

    const int last = rt + (seg.hi - 1 - rt) / groups * groups;   // this block's last tile of the segment
#pragma unroll
    for (int j = 0; j < 3; ++j) load_tile(min(rt + j * groups, last), j);
    for (int buf = 0; rt < seg.hi; rt += groups, buf = (buf + 1) & 3) {
      __builtin_amdgcn_s_waitcnt(0x0f70 | (2 * KS));   // vmcnt(2 KS)
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      load_tile(min(rt + 3 * groups, last), (buf + 3) & 3);
      f32x4 acc[2][NI];
#pragma unroll
      for (int n = 0; n < NI; ++n) acc[0][n] = acc[1][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      const auto products = [&](auto stage) {
        constexpr int S = decltype(stage)::value;
        f32x4 x[4];
        read_rows<S * SA::kBytes>(x, even + buf * kTile, odd + buf * kTile);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int m = 0; m < 2; ++m)
              acc[m][n] = Type<T>::mma(fw[n][S * 2 + s], __builtin_bit_cast(typename Type<T>::frag, x[s * 2 + m]), acc[m][n]);
      };
      products(std::integral_constant<int, 0>());
      if constexpr (KS > 1) products(std::integral_constant<int, 1>());
      if constexpr (KS > 2) products(std::integral_constant<int, 2>());
      if constexpr (KS > 3) products(std::integral_constant<int, 3>());
      if constexpr (EPI)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          Chunk<T> b;
          b.raw = bias[t];
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[m][t * 2 + i / 4][i & 3] += (float)b.e[i];
        }
      // what depends on the lane is formed again for every tile: kept over the loop it would not fit
      // beside the weight
      int l = lane;
      asm volatile("" : "+v"(l));
      const RowTile tile{seg.e, first_row(rt), min(seg.rows, BM)};
      if (seg.rows >= BM) store_results<T, 2, NI, EPI, ACT, true>(p, acc, tile, wr * 32, col0, l);
      else store_results<T, 2, NI, EPI, ACT, false>(p, acc, tile, wr * 32, col0, l);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): no load to LDS is under way
  }
}

// Joins the parts of split sums in order, with the epilogue; zeros for rows of no group.  A block has 16
// rows and 64 columns.
constexpr int kJoinThreads = 128;
template <typename T, bool EPI> __global__ __launch_bounds__(kJoinThreads) void split_join_kernel(RowsArgs p) {
  constexpr int CH = 16 / (int)sizeof(T), PC = 64 / CH;
  typedef typename Deriv<T>::type D;
  RowTile tile;
  const int block = blockIdx.x + p.block0;
  if (!find_row_tile(p.g, block / p.col_tiles, 16, tile)) return;
  const int n0 = block % p.col_tiles * 64;
  for (int c = threadIdx.x; c < 16 * PC; c += kJoinThreads) {
    const int row = c / PC, col = n0 + c % PC * CH, left = p.N - col;
    if (row >= tile.rows || left <= 0) continue;
    const int64_t at = (tile.first + row) * p.N + col;
    float z[CH], d[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i) z[i] = 0.f;
    if (tile.e >= 0) {
#pragma unroll 4
      for (int s = 0; s < p.splits; ++s) {
        const float *src = p.part + s * p.rows * p.N + at;
#pragma unroll
        for (int i = 0; i < CH; i += 4) {
          const uint4 v = fetch(src + i, 0, 0, 0, 1, left - i);
          z[i] += __uint_as_float(v.x);
          z[i + 1] += __uint_as_float(v.y);
          z[i + 2] += __uint_as_float(v.z);
          z[i + 3] += __uint_as_float(v.w);
        }
      }
      if (EPI) {
        if (p.bias) {
          Chunk<T> b;
          b.raw = fetch(static_cast<const T *>(p.bias) + (int64_t)tile.e * p.N, 0, 0, col, 1, p.N);
#pragma unroll
          for (int i = 0; i < CH; ++i) z[i] += (float)b.e[i];
        }
#pragma unroll
        for (int i = 0; i < CH; ++i) z[i] = activate<sizeof(T) == 2>(p.act, z[i], d[i]);
        if (p.act_grad) store_chunk<D, true>(static_cast<D *>(p.act_grad) + at, Deriv<T>::encode(d), left);
        if (p.res) {
          Chunk<T> r;
          r.raw = fetch(static_cast<const T *>(p.res) + (tile.first + row) * p.ld_res, 0, 0, col, 1, p.N);
#pragma unroll
          for (int i = 0; i < CH; ++i) z[i] += (float)r.e[i];
        }
      }
    }
    Chunk<T> out;
#pragma unroll
    for (int i = 0; i < CH; ++i) out.e[i] = (T)z[i];
    store_chunk<T>(static_cast<T *>(p.c) + at, out.raw, left);
  }
}

// ---------------------------------------------------------------------------------------------
// Few rows: the weight's bytes bound it.  A block takes 16 columns of up to 16 RT rows; its waves
// share the sum, read the weight straight into MFMA operands (each byte once) and join their sums
// through LDS.  8 x 4096 -> 4096 bf16 9 to 10 us (33.5 MB); 96 rows in 64 groups 1024 -> 2048 36 to 39 (the
// weights of the 46 or so groups that have rows, 190 MB, at HBM's rate); one row of 256 4.2, a launch and
// a round of loads.  16 waves a block were not faster.
template <typename T, int RT, int NW>
__global__ __launch_bounds__(64 * NW) void few_rows_kernel(RowsArgs p) {
  constexpr int CH = 16 / (int)sizeof(T), KS = 4 * CH;   // sum elements of a step: 16 bytes a lane, 4 lanes a row
  __shared__ f32x4 red[NW][RT][64];
  int rt, ct;
  block_tile(blockIdx.x + p.block0, p.col_tiles, 0, rt, ct);
  RowTile tile;
  if (!find_row_tile(p.g, rt, 16 * RT, tile)) return;
  const int n0 = ct * 16, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  f32x4 acc[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (tile.e >= 0) {
    const T *a = static_cast<const T *>(p.a) + tile.first * p.lda;
    const T *w = static_cast<const T *>(p.w) + tile.e * p.w_group + (int64_t)n0 * p.K;
    constexpr int U = RT <= 2 ? 4 : 2;   // steps in flight a wave
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
        if (p.act_grad) static_cast<typename Deriv<T>::type *>(p.act_grad)[grow * p.N + col + j] = Deriv<T>::encode1(d);
        if (p.res) y += (float)static_cast<const T *>(p.res)[grow * p.ld_res + col + j];
      }
      static_cast<T *>(p.c)[grow * p.N + col + j] = (T)y;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// RING's operands of 32 rows of a stage: results 2 t + h, H bytes apart, in halves of 4 rows of 256 bytes
// (Stage::frag), read in assembly with the wait in the same statement, as the compiler waits for all loads
// to LDS under way before its own reads.
template <int OFF, int H> __device__ __forceinline__ void read_columns(s16x4 (&v)[8], const uint32_t (&at)[2], uint32_t stage) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%10\n\tds_read_b64_tr_b16 %1, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%12\n\tds_read_b64_tr_b16 %3, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %9 offset:%10\n\tds_read_b64_tr_b16 %5, %9 offset:%11\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%12\n\tds_read_b64_tr_b16 %7, %9 offset:%13\n\ts_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(at[0] + stage), "v"(at[1] + stage), "n"(OFF), "n"(OFF + 1024), "n"(OFF + H), "n"(OFF + 1024 + H)
      : "memory");
}

// gw = dz^T x, gb = sum of dz over the rows of a chunk; a chunk that is its group's only one writes
// the results, the others their partial sums.  Column sums come with the products, as one more operand of
// ones: in fp32 registers beside the loads they were slower.
// RUNS: chunks of several items, a kernel of its own as the walk over them takes registers (127 -> 135 in
// 128 x 128, which is a wave a SIMD less).
// RING (16-bit types, 128 x 128, chunks of 512 rows and more): two stages in LDS, the next one's loads under
// way during the products; two blocks a CU, which is what there is of long chunks.  Order of a wave's memory
// operations: loads of stages i, i + 1, so all but the newest kLoads done means that stage i is there; the
// barrier behind it says so for every wave, the one behind the products that its place is free.
// Single-buffered, with up to four blocks a CU, and with the ring: 73728 rows of 256 x 256 in bf16 24 and 21
// us (75 MB: 15), 256 x 1024 75 and 64, 598016 rows in three groups 182 and 160 (612 MB: 118; it fetches
// 744 MB, 4.6 TB/s, which bounds it); join_kernel adds 6, 7 and 11.  Chunks of 256 rows (16411 rows in 64
// groups, 512 x 1024 fp16): 53 without, 56 with.
template <typename T, int BM, int BN, int WR, int WC, bool DMA, bool RUNS, bool RING, int OCC>
__global__ __launch_bounds__(64 * WR *WC) __attribute__((amdgpu_waves_per_eu(OCC))) void weight_kernel(WeightArgs p) {
  constexpr int NT = 64 * WR * WC, TM = BM / WR, TN = BN / WC, MI = TM / 16, NI = TN / 16;
  typedef Stage<T, BM, NT, true> SU;
  typedef Stage<T, BN, NT, true> SX;
  constexpr int kStage = SU::kBytes + SX::kBytes;
  static_assert(!RING || (DMA && !RUNS && sizeof(T) == 2), "whole items, 16-byte rows, transposing reads");
  __shared__ __attribute__((aligned(16))) char lds[(RING ? 2 : 1) * kStage];
  int slot, ct;
  block_tile(blockIdx.x + p.block0, p.n_tiles * p.k_tiles, 1, slot, ct);
  if (slot >= p.slots) return;
  RowChunk ch;
  if (!find_chunk(p.g, slot, p.chunk, p.items, false, ch)) return;
  const int n0 = ct / p.k_tiles * BM, k0 = ct % p.k_tiles * BN;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, wr = wave / WC, wc = wave % WC;
  const bool with_b = p.gb && k0 == 0 && wc == 0;   // column sums as products with ones

  f32x4 acc[MI][NI], accb[MI];
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    accb[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const auto add = [&](int64_t first) {
    const T *u = static_cast<const T *>(p.u) + first * p.ldu + n0;
    const T *x = static_cast<const T *>(p.x) + first * p.ldx + k0;
    if constexpr (RING) {
      constexpr int kLoads = SU::NL + SX::NL;
      static_assert(SU::kRowBytes == 256 && SX::kRowBytes == 256 && MI == 4 && NI == 4, "read_columns");
      const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds;
      const int i = lane & 15, row = (lane >> 4) * 8 + (i >> 2);
      uint32_t au[2], ax[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        au[t] = base + SU::address(row, (wr * TM + t * 32) / 8 + ((i & 3) >> 1)) + (i & 1) * 8;
        ax[t] = base + SU::kBytes + SX::address(row, (wc * TN + t * 32) / 8 + (i & 3));
      }
      const auto load = [&](int st) {
        char *const to = lds + (st & 1) * kStage;
        SU::load_lds(to, u, p.ldu, ch.rows, p.N - n0, st * SU::KC);
        SX::load_lds(to + SU::kBytes, x, p.ldx, ch.rows, p.K - k0, st * SU::KC);
      };
      const auto half = [&](auto step, uint32_t stage) {
        constexpr int OFF = decltype(step)::value * 32 * 256;
        typedef typename Type<T>::frag F;
        s16x4 vx[8], vu[8];
        read_columns<OFF, 8>(vx, ax, stage);     // column_of
        read_columns<OFF, 32>(vu, au, stage);
        const auto frag = [](const s16x4 (&v)[8], int n) {
          return __builtin_bit_cast(F, __builtin_shufflevector(v[2 * n], v[2 * n + 1], 0, 1, 2, 3, 4, 5, 6, 7));
        };
#pragma unroll
        for (int m = 0; m < MI; ++m) {
          const F fu = frag(vu, m);
#pragma unroll
          for (int n = 0; n < NI; ++n) acc[m][n] = Type<T>::mma(frag(vx, n), fu, acc[m][n]);
          if (with_b) accb[m] = Type<T>::mma(Type<T>::ones(), fu, accb[m]);
        }
      };
      const auto products = [&](int st) {
        half(std::integral_constant<int, 0>(), (st & 1) * kStage);
        half(std::integral_constant<int, 1>(), (st & 1) * kStage);
      };
      const auto barrier = [] {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      };
      const int whole = ch.rows / SU::KC;
      if (whole > 0) load(0);
      if (whole > 1) load(1);
      for (int st = 0; st < whole; ++st) {
        if (st + 1 < whole) __builtin_amdgcn_s_waitcnt(0x0f70 | kLoads);   // vmcnt(kLoads): stage st is here
        else __builtin_amdgcn_s_waitcnt(0x0f70);
        barrier();
        products(st);
        barrier();
        if (st + 2 < whole) load(st + 2);
      }
      if (whole * SU::KC < ch.rows) {   // the rest, with zeros behind it; all loads are done
        char *const to = lds + (whole & 1) * kStage;
        SU::load_end(to, u, p.ldu, ch.rows, p.N - n0, whole * SU::KC);
        SX::load_end(to + SU::kBytes, x, p.ldx, ch.rows, p.K - k0, whole * SU::KC);
        __syncthreads();
        products(whole);
      }
      return;
    }
    uint4 vu[DMA ? 1 : SU::NL], vx[DMA ? 1 : SX::NL];
    if constexpr (!DMA) {
      SU::load(vu, u, p.ldu, ch.rows, p.N - n0, 0);
      SX::load(vx, x, p.ldx, ch.rows, p.K - k0, 0);
    }
    for (int r0 = 0; r0 < ch.rows; r0 += SU::KC) {
      if (r0) __syncthreads();
      if constexpr (DMA) {
        SU::load_either(lds, u, p.ldu, ch.rows, p.N - n0, r0);
        SX::load_either(lds + SU::kBytes, x, p.ldx, ch.rows, p.K - k0, r0);
        __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0): this wave's loads are in LDS
      } else {
        SU::store(lds, vu);
        SX::store(lds + SU::kBytes, vx);
        if (r0 + SU::KC < ch.rows) {
          SU::load(vu, u, p.ldu, ch.rows, p.N - n0, r0 + SU::KC);
          SX::load(vx, x, p.ldx, ch.rows, p.K - k0, r0 + SU::KC);
        }
      }
      __syncthreads();
  #pragma unroll
      for (int s = 0; s < 2; ++s) {
        typename Type<T>::frag fx[NI];
  #pragma unroll
        for (int n = 0; n < NI; ++n) fx[n] = SX::frag(lds + SU::kBytes, s, [&](int i) { return wc * TN + column_of<T>(n, i); }, threadIdx.x & 63);
  #pragma unroll
        for (int m = 0; m < MI; ++m) {
          const typename Type<T>::frag fu = SU::frag(lds, s, [&](int i) { return wr * TM + m * 16 + i; }, threadIdx.x & 63);
  #pragma unroll
          for (int n = 0; n < NI; ++n) acc[m][n] = Type<T>::mma(fx[n], fu, acc[m][n]);
          if (with_b) accb[m] = Type<T>::mma(Type<T>::ones(), fu, accb[m]);
        }
      }
    }
  };
  if constexpr (RUNS) {
    for (int item = 0; item < ch.items; ++item) {
      if (item) __syncthreads();
      add(ch.first + (int64_t)item * p.g.S);
    }
  } else {
    add(ch.first);
  }
  // lane (i, q) of acc[m][n]: row n0 + m * 16 + i of gw, columns k0 + column_of(n, 4 q) .. + 3
  constexpr int CH = 16 / (int)sizeof(T), NP = CH / 4;
  const bool direct = ch.chunks == 1;
  const int i = lane & 15, q = lane >> 4;
#pragma unroll
  for (int m = 0; m < MI; ++m) {
    const int row = n0 + wr * TM + m * 16 + i;
    if (row >= p.N) continue;
#pragma unroll
    for (int t = 0; t < NI / NP && p.gw; ++t) {
      const int col = k0 + wc * TN + t * NP * 16 + q * CH, left = p.K - col;
      if (left <= 0) continue;
      if (direct) {
        Chunk<T> out;
#pragma unroll
        for (int j = 0; j < CH; ++j) out.e[j] = (T)acc[m][t * NP + j / 4][j & 3];
        store_chunk<T>(static_cast<T *>(p.gw) + ((int64_t)ch.e * p.N + row) * p.K + col, out.raw, left);
      } else {
#pragma unroll
        for (int j = 0; j < NP; ++j)
          if (left > j * 4)
            store_chunk<float>(p.part + ((int64_t)slot * p.N + row) * p.K + col + j * 4,
                               __builtin_bit_cast(uint4, acc[m][t * NP + j]), left - j * 4);
      }
    }
    if (with_b && q == 0) {
      if (direct) static_cast<T *>(p.gb)[(int64_t)ch.e * p.N + row] = (T)accb[m][0];
      else p.part_b[(int64_t)slot * p.N + row] = accb[m][0];
    }
  }
}

// dz = grad_y * act_grad, where no input gradient's kernel forms it
template <typename T> __global__ __launch_bounds__(256) void scale_kernel(const T *u, int64_t ldu, const void *scale, T *dz, int64_t rows, int N) {
  constexpr int CH = 16 / (int)sizeof(T);
  typedef typename Deriv<T>::type D;
  const int per = (N + CH - 1) / CH;
  for (int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x; c < rows * per; c += (int64_t)gridDim.x * 256) {
    const int64_t row = c / per;
    const int col = (int)(c - row * per) * CH;
    const uint4 v = Deriv<T>::apply(fetch(u + row * ldu, 0, 0, col, 1, N),
                                    fetch(static_cast<const D *>(scale) + row * N, 0, 0, col, 1, N));
    store_chunk<T>(dz + row * N + col, v, N - col);
  }
}

// dst = src in rows of a group, 0 in the others, of all items: the gradient of a residual, which rows of no
// group do not take (73728 x 256 bf16, three groups: 14 us, 5.4 TB/s).  A row takes 2^log threads of a block.
template <typename T>
__global__ __launch_bounds__(256) void keep_rows_kernel(const T *src, int64_t ld, T *dst, int64_t rows, int N, int log, Groups g) {
  constexpr int CH = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63;
  int carry = 0, first = 0, end = 0;   // an item's rows in groups: from bound(0) to bound(E)
  for (int base = 0; base <= g.E; base += 64) {
    const Segment s = segment_at(g, base + lane, carry);
    if (base == 0) first = __builtin_amdgcn_readlane(s.upper, 0);
    end = __builtin_amdgcn_readlane(s.upper, min(g.E - base, 63));
  }
  const int64_t step = (int64_t)gridDim.x * (256 >> log);
  for (int64_t row = (int64_t)blockIdx.x * (256 >> log) + (threadIdx.x >> log); row < rows; row += step) {
    const int r = (int)((uint32_t)row % (uint32_t)g.S);   // rows of all items fit 31 bits
    const bool keep = r >= first && r < end;
    for (int col = (threadIdx.x & ((1 << log) - 1)) * CH; col < N; col += CH << log)
      store_chunk<T>(dst + row * N + col, keep ? fetch(src + row * ld, 0, 0, col, 1, N) : make_uint4(0, 0, 0, 0), N - col);
  }
}

// Sums the chunks' partial results in order.  Blocks of 64 elements,
// four threads an element, each a quarter of the slots.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(WeightArgs p) {
  __shared__ float red[4][64];
  const int e = blockIdx.y;
  RowChunk ch;
  find_chunk(p.g, e, p.chunk, p.items, true, ch);
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

// Row tiles of BM rows at most: every segment may end inside one, but an item has no more than its rows.
inline int64_t max_row_tiles(const Groups &g, int BM) {
  if (!g.start) return ceil_div(g.S, BM);
  const int64_t tiles = (int64_t)g.S / BM + g.E + 2;
  return (int64_t)g.B * (tiles < g.S ? tiles : g.S);
}

// A launch holds less than 2^32 threads; more go in several, each a multiple of the XCDs' 8 blocks.
template <typename K, typename A> inline hipError_t launch(K kernel, int64_t grid, int threads, hipStream_t st, A p) {
  if (grid <= 0 || grid > 0x7fffffff) return hipErrorInvalidConfiguration;
  const int64_t most = 0xffffffff / threads & ~(int64_t)7;
  for (int64_t at = 0; at < grid; at += most) {
    p.block0 = (unsigned)at;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(grid - at < most ? grid - at : most)), dim3(threads), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int BM, int BN, int WR, int WC, int U, bool DMA, int OCC, bool WSTR, bool SCALE, bool EPI, bool SPLIT = false>
inline hipError_t launch_rows(RowsArgs p, hipStream_t st) {
  const int64_t rt = max_row_tiles(p.g, BM);
  p.row_tiles = (int)rt;
  p.col_tiles = ceil_div(p.N, BN);
  p.spread = rt >= 64;
  const int64_t grid = (p.spread ? (rt + 7) / 8 * 8 : rt) * p.col_tiles * (SPLIT ? p.splits : 1);
  return launch(rows_kernel<T, BM, BN, WR, WC, U, DMA, OCC, WSTR, SCALE, EPI, SPLIT>, grid, 64 * WR * WC, st, p);
}

// How many parts a sum of K elements is cut into, by tiles of 64 x 64: none where the tiles make 256
// blocks or there are less than 16 stages (four rounds of loads in one part, which two launches do not
// beat); otherwise parts of 4 stages or more, up to 512 blocks.  One row of dz, 3301 -> 1856 in bf16:
// 11 us, about 100 in one part; 576 x 256 -> 256 in fp32 (8 stages): 13 us in two parts, 9 in one.
inline int split_count(int esize, int64_t rows, int E, int N, int K) {
  const int stages = ceil_div(K, 128 / esize);
  const int64_t tiles = (ceil_div(rows, 64) + (E > 1 ? E : 0)) * (int64_t)ceil_div(N, 64);
  if (tiles >= 256 || stages < 16) return 1;
  int64_t parts = 512 / tiles < stages / 4 ? 512 / tiles : stages / 4;
  return parts < 2 ? 1 : ceil_div(stages, ceil_div(stages, parts));
}

template <typename T, int KS, bool WSTR, bool EPI, int ACT> inline hipError_t launch_stream_of(RowsArgs p, hipStream_t st) {
  p.row_tiles = (int)max_row_tiles(p.g, 64);
  p.col_tiles = ceil_div(p.N, 256);
  const int per_xcd = p.col_tiles < 32 ? 32 / p.col_tiles : 1;   // groups of row tiles on each XCD's 32 CUs
  return launch(stream_kernel<T, KS, WSTR, EPI, ACT>, (int64_t)8 * p.col_tiles * per_xcd, 512, st, p);
}
template <typename T, int KS, bool WSTR, bool EPI> inline hipError_t launch_stream(const RowsArgs &p, hipStream_t st) {
  if constexpr (EPI) {
    switch (p.act) {
      case kRelu: return launch_stream_of<T, KS, WSTR, EPI, kRelu>(p, st);
      case kGelu: return launch_stream_of<T, KS, WSTR, EPI, kGelu>(p, st);
      case kGeluTanh: return launch_stream_of<T, KS, WSTR, EPI, kGeluTanh>(p, st);
      case kSilu: return launch_stream_of<T, KS, WSTR, EPI, kSilu>(p, st);
      default: break;
    }
  }
  return launch_stream_of<T, KS, WSTR, EPI, kNone>(p, st);
}

// What the streaming kernel takes: sums of 128 or 256, columns that fill their slices of 256 for the most
// part, and 8 tiles of 64 rows or more for each block and segment, which starts by loading the weight
// (73728 rows: 1024 columns 46 us, 61 in tiles, 256 columns 21 and 20).  Not smooth activations that keep
// act_grad: their arithmetic needs more waves than two a SIMD (73728 x 256 -> 1024 gelu 101 us, 93).
inline bool streams(const RowsArgs &p) {
  return (p.K == 128 || p.K == 256) && p.N >= 256 && p.N % 8 == 0 && p.N * 4 >= ceil_div(p.N, 256) * 768 &&
         p.rows * ceil_div(p.N, 256) >= (int64_t)131072 * p.g.E * p.g.B && (!p.act_grad || p.act == kRelu);
}

template <typename T, int RT, int NW> inline hipError_t launch_few(RowsArgs p, hipStream_t st) {
  const int64_t rt = max_row_tiles(p.g, 16 * RT);
  p.row_tiles = (int)rt;
  p.col_tiles = ceil_div(p.N, 16);
  return launch(few_rows_kernel<T, RT, NW>, rt * p.col_tiles, 64 * NW, st, p);
}

// Whether every row of a matrix starts at a 16-byte boundary, within the offsets of Stage::load_lds.
inline bool rows_aligned(const void *p, int64_t ld, int esize) {
  return ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * esize)) & 15u) == 0 && ld < (1 << 22);
}

template <typename T, bool DMA, bool WSTR, bool SCALE, bool EPI> inline hipError_t launch_tiles(const RowsArgs &p, hipStream_t st) {
  if constexpr (DMA && !SCALE && sizeof(T) == 2) {
    if (streams(p)) return p.K == 128 ? launch_stream<T, 2, WSTR, EPI>(p, st) : launch_stream<T, 4, WSTR, EPI>(p, st);
  }
  if constexpr (DMA && !SCALE) {
    // long sums: wider tiles read their operands less often (4096^3 bf16 136 us, 144 in tiles of 128; at
    // sums of 256 those are as fast or faster)
    if (p.K >= 1024 && p.N >= 256 && p.rows / p.g.E >= 512 && (p.rows + 127) / 128 * ceil_div(p.N, 256) >= 384)
      return launch_rows<T, 128, 256, 2, 4, 1, true, 4, WSTR, SCALE, EPI>(p, st);
  }
  if constexpr (!DMA && !SCALE && sizeof(T) == 2) {
    // through registers the widest tiles that fill the CUs (4096 x 4095 -> 4093 bf16 202 us, 252; its input
    // gradient 179, 229)
    if (p.K >= 512 && p.N >= 256 && p.rows / p.g.E >= 512 && (p.rows + 255) / 256 * ceil_div(p.N, 256) >= 192)
      return launch_rows<T, 256, 256, 2, 4, 1, false, 2, WSTR, SCALE, EPI>(p, st);
  }
  if ((p.rows + 127) / 128 * ceil_div(p.N, 128) >= 256 && p.N > 64) {
    // act_grad through registers takes a block a CU more off the unaligned 128 x 128 (73728 x 1024 -> 256:
    // 64 x 128 142 us, 157; aligned 128 x 128 121, 64 x 128 137)
    if constexpr (SCALE && !DMA) return launch_rows<T, 64, 128, 1, 4, 1, DMA, 4, WSTR, SCALE, EPI>(p, st);
    else return launch_rows<T, 128, 128, 2, 2, 1, DMA, DMA && !SCALE ? 4 : 3, WSTR, SCALE, EPI>(p, st);
  }
  // 64 x 64: from two tiles a CU on the blocks wait in turn, and a stage at a time leaves room for more of
  // them (10013 x 250 -> 333 fp32 34 us, 42 in fours); fewer tiles load four stages at once
  if ((p.rows + 63) / 64 * ceil_div(p.N, 64) >= 512)
    return launch_rows<T, 64, 64, 2, 2, 1, DMA, 4, WSTR, SCALE, EPI>(p, st);
  constexpr int U = SCALE ? 2 : 4, OCC = SCALE ? 4 : 2;
  if (p.splits > 1) {
    const hipError_t e = launch_rows<T, 64, 64, 2, 2, U, DMA, OCC, WSTR, SCALE, EPI, true>(p, st);
    if (e != hipSuccess) return e;
    RowsArgs j = p;
    j.col_tiles = ceil_div(p.N, 64);
    return launch(split_join_kernel<T, EPI>, max_row_tiles(p.g, 16) * j.col_tiles, kJoinThreads, st, j);
  }
  return launch_rows<T, 64, 64, 2, 2, U, DMA, OCC, WSTR, SCALE, EPI>(p, st);
}

template <typename T, bool WSTR, bool SCALE, bool EPI> inline hipError_t launch_rows_of(const RowsArgs &p, hipStream_t st) {
  const bool aligned = (SCALE || rows_aligned(p.a, p.lda, sizeof(T))) && rows_aligned(p.w, WSTR ? p.N : p.K, sizeof(T));
  return aligned ? launch_tiles<T, true, WSTR, SCALE, EPI>(p, st) : launch_tiles<T, false, WSTR, SCALE, EPI>(p, st);
}

// Rows a group up to which the forward takes the kernel for few rows.
constexpr int kFewRows = 64;

template <typename T> hipError_t forward(const RowsArgs &p, hipStream_t st) {
  const int64_t per_group = p.rows / p.g.E;
  if (per_group <= 16) return p.K >= 2048 ? launch_few<T, 1, 8>(p, st) : launch_few<T, 1, 4>(p, st);
  if (per_group <= 32) return p.K >= 2048 ? launch_few<T, 2, 8>(p, st) : launch_few<T, 2, 4>(p, st);
  if (per_group <= kFewRows) return p.K >= 2048 ? launch_few<T, 4, 8>(p, st) : launch_few<T, 4, 4>(p, st);
  return launch_rows_of<T, false, false, true>(p, st);
}

template <typename T> hipError_t grad_x(const RowsArgs &p, hipStream_t st) {
  return p.scale ? launch_rows_of<T, true, true, false>(p, st) : launch_rows_of<T, true, false, false>(p, st);
}

// Tile, rows per chunk and number of chunks of the weight kernel; the workspace follows from it.
// 512 blocks of 128 x 128 fill the 256 CUs once (two blocks each; groups take theirs off, since each may end
// inside a chunk: 524 blocks cost a second round, 425 -> 409 us a step for 598016 rows in three groups).
// Where the tiles times chunks of 256 rows do not make 256 blocks, or where one side has 64 columns at most,
// tiles of 64 x 64 and chunks of 64 rows do better, up to 1024 blocks.  From 64 tiles on chunks of 512 rows
// and more, up to 2048 blocks: a few long ones end one after another, and their partial sums are little
// beside the products (9642 rows in two groups, 849 x 2976 fp32: 672 blocks took two rounds on CUs that hold
// 512).
// Many items of many groups: a chunk takes the same rows of several items, so that items times groups do
// not make more partial sums than there are blocks to fill the CUs (64 items of 128 groups, 1024 x 4096:
// 139 GB of them otherwise).
struct ChunkPlan {
  int tile, chunk, items;
  int64_t slots;
  bool joined;   // a group may have several chunks
  ChunkPlan(int esize, bool grouped, int B, int64_t S, int E, int N, int K) {
    const int kc = 128 / esize;
    const int64_t rows = (int64_t)B * S, big = (int64_t)ceil_div(N, 128) * ceil_div(K, 128);
    tile = big * (rows / 256 > E ? rows / 256 : E) >= 256 && N > 64 && K > 64 ? 128 : 64;
    const int64_t tiles = (int64_t)ceil_div(N, tile) * ceil_div(K, tile);
    const bool many = tile == 128 && tiles >= 64;
    const int64_t least = many ? 512 : tile == 128 ? 256 : 64;
    int64_t want = (many ? 2048 : tile == 128 ? 512 : 1024) / tiles;
    const int64_t fill = want > E ? want : E;
    items = (int64_t)B * E > fill ? ceil_div((int64_t)B * E, fill) : 1;
    if (want > rows / least) want = rows / least;
    if (want <= E) want = 1;
    if (grouped && want > (int64_t)2 * B * E) want -= (int64_t)B * E;   // every segment may end inside a chunk
    chunk = (int)((S + kc - 1) / kc * kc);
    if (want > 1) chunk = (int)((rows / want / items + kc - 1) / kc * kc);
    if (chunk < kc) chunk = kc;
    const int64_t runs = ceil_div(B, items);
    slots = grouped ? runs * (S / chunk + E) : S > chunk ? ceil_div(S, chunk) : 1;
    joined = grouped ? runs > 1 || chunk < S : slots > 1;
  }
};

template <typename T>
hipError_t scale(const void *u, int64_t ldu, const void *act_grad, void *dz, int64_t rows, int N, hipStream_t st) {
  const int64_t chunks = rows * ceil_div(N, 16 / (int)sizeof(T)), blocks = (chunks + 255) / 256;
  hipLaunchKernelGGL((scale_kernel<T>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, st,
                     static_cast<const T *>(u), ldu, act_grad, static_cast<T *>(dz), rows, N);
  return hipGetLastError();
}

template <typename T>
hipError_t keep_rows(const void *src, int64_t ld, void *dst, int64_t rows, int N, const Groups &g, hipStream_t st) {
  int log = 0;
  while (log < 8 && (16 / (int)sizeof(T) << log) < N) ++log;
  const int64_t blocks = (rows + (256 >> log) - 1) / (256 >> log);
  hipLaunchKernelGGL((keep_rows_kernel<T>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, st,
                     static_cast<const T *>(src), ld, static_cast<T *>(dst), rows, N, log, g);
  return hipGetLastError();
}

template <typename T> hipError_t grad_weight(const WeightArgs &q, int tile, bool joined, hipStream_t st) {
  WeightArgs p = q;
  p.n_tiles = ceil_div(p.N, tile);
  p.k_tiles = p.gw ? ceil_div(p.K, tile) : 1;
  const int64_t grid = ((int64_t)p.slots + 7) / 8 * 8 * p.n_tiles * p.k_tiles;
  const bool aligned = rows_aligned(p.u, p.ldu, sizeof(T)) && rows_aligned(p.x, p.ldx, sizeof(T)) &&
                       p.N % (16 / sizeof(T)) == 0 && p.K % (16 / sizeof(T)) == 0;
  const auto start = [&](auto runs) {
    constexpr bool R = decltype(runs)::value;
    if (tile == 128 && aligned) return launch(weight_kernel<T, 128, 128, 2, 2, true, R, false, 2>, grid, 256, st, p);
    if (tile == 128) return launch(weight_kernel<T, 128, 128, 2, 2, false, R, false, 2>, grid, 256, st, p);
    if (aligned) return launch(weight_kernel<T, 64, 64, 2, 2, true, R, false, 4>, grid, 256, st, p);
    return launch(weight_kernel<T, 64, 64, 2, 2, false, R, false, 4>, grid, 256, st, p);
  };
  hipError_t e = hipSuccess;
  bool ring = false;
  if constexpr (sizeof(T) == 2) {
    ring = tile == 128 && aligned && p.items == 1 && (int64_t)p.g.B * p.g.S / p.slots >= 512;
    if (ring) e = launch(weight_kernel<T, 128, 128, 2, 2, true, false, true, 2>, grid, 256, st, p);
  }
  if (!ring) e = p.items > 1 ? start(std::true_type()) : start(std::false_type());
  if (e != hipSuccess) return e;
  if (joined) {
    const int64_t total = (p.gw ? (int64_t)p.N * p.K : 0) + (p.gb ? p.N : 0), want = (total + 63) / 64;
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(want < 2048 ? want : 2048), p.g.E), dim3(256), 0, st, p);
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
extern template hipError_t grad_weight<float>(const WeightArgs &, int, bool, hipStream_t);
extern template hipError_t scale<float>(const void *, int64_t, const void *, void *, int64_t, int, hipStream_t);
extern template hipError_t grad_weight<_Float16>(const WeightArgs &, int, bool, hipStream_t);
extern template hipError_t scale<_Float16>(const void *, int64_t, const void *, void *, int64_t, int, hipStream_t);
extern template hipError_t grad_weight<__bf16>(const WeightArgs &, int, bool, hipStream_t);
extern template hipError_t scale<__bf16>(const void *, int64_t, const void *, void *, int64_t, int, hipStream_t);

extern template hipError_t keep_rows<float>(const void *, int64_t, void *, int64_t, int, const Groups &, hipStream_t);
extern template hipError_t keep_rows<_Float16>(const void *, int64_t, void *, int64_t, int, const Groups &, hipStream_t);
extern template hipError_t keep_rows<__bf16>(const void *, int64_t, void *, int64_t, int, const Groups &, hipStream_t);

}  // namespace ops3d_linear
