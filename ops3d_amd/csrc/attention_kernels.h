// Attention over all tokens (gfx950), forward and backward (include/ops3d_attention.h).
//
// One scheme for its three kernels: a block owns some columns of the logits, whose operands stay in
// registers, and the other side's rows come by in stages through LDS:
//   forward   owns queries, keys and values come by      S^T = K Q^T,  O^T += V^T P^T
//   grad q    owns queries, keys and values come by      S^T, dP^T = V dO^T,  dQ^T += K^T dS^T
//   grad k v  owns keys, queries and grad_out come by    S = Q K^T, dP = dO V^T,  dV^T += dO^T P, dK^T += Q^T dS
// The products run on 16 x 16 MFMA results: lane (i, q) (i the lane mod 16, q its quarter of the wave) holds
// rows 4 q .. 4 q + 3 of column i.  Those are the operand elements that the next product wants from the lane
// if its sum runs over the rows in the order 4 q .. 4 q + 3 of one result, the same of the next: so P and
// dS go from result to operand in registers, rounded, and the other operand is read from LDS transposed in
// that order.
//
// Columns of queries are pairs of a query and a head of the key head's group, c = query G + head: the heads of
// a group share the keys that come by, in training and where one query is all there is.
//
// Softmax runs along: a column's reference m is raised, and its sums are rescaled, only when a logit passes
// it by 2^kSlack; P is at most that.  Statistics are kept in log2 units.
//
// What bounds them (one MI355X, bf16, 8 heads; a large library product reaches 1184 TFLOP/s): with 32 channels a logit
// is 128 operations on the matrix units and, beside them, an exponential, a multiply-add, a comparison and a rounding, and
// where all blocks are alike the vector units are the bound (79 % of the cycles).  Elsewhere nothing is full: with 128
// channels the registers leave two waves a SIMD, which wait for their own loads and products (matrix units 33 to 39 % of the
// cycles, vector units 26 to 39, LDS 38 at most).
//   forward  4096 x 4096     32 / 64 / 96 / 128 channels   47 / 58 / 86 / 88 us   367 / 594 / 597 / 782 TFLOP/s
//            32768 x 32768   32                            1700 us                647
//   backward 4096 x 4096     32 / 64 / 96 / 128            124 / 158 / 250 / 263  347 / 543 / 515 / 653 (10 D a logit; 14 D
//                                                          are done, as both kernels form S and dP)
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "elements.h"
#include "launch.h"
#include "reduce.h"
#include "segments.h"

namespace ops3d_attention {

using namespace ops3d_elements;

struct Tensor {
  void *p;
  int64_t item, token, head;
};

struct Args {
  Tensor q, k, v, o, g, gq, gk, gv;   // g: grad_out
  const int64_t *q_start, *k_start, *q_len, *k_len;
  int q_count, k_count, E;            // E: sequences (packed)
  int Sq, Sk;                         // rows of an item
  int Hk, G, D;                       // key heads, query heads of each, channels
  uint32_t magic;                     // c / G = 2 c magic >> 32 >> shift
  int shift;
  int causal;
  int dma;                            // rows go straight to LDS: bit 0 k and v, bit 1 q and grad_out
  float scale, c;                     // c = scale log2 e
  int tiles, tiles_item, splits;      // tiles of all items (a bound), of one, and parts of the other side
  unsigned block0;                    // blocks in launches before this one
  int heads;                          // items Hk
  int64_t cells;                      // heads Sq G: queries times heads
  const int4 *table;                  // two for each tile of packed sequences (see table_kernel), or nullptr
  void *rest;                         // what rounding took from o, [items, Sq, heads, D] contiguous, or nullptr
  float *lse, *delta;                 // [items, Hk, Sq G]; log2 of the sum of exponentials, and sum of o g
  float *part;                        // [splits, columns, DP]
  f32x4 *part_ml;                     // [splits, columns]: reference, sum of rounded P, sum of P, whether the column sees a key
};

// What a block works on.
struct Work {
  int item, q0, k0;      // first rows of the sequence
  int nq, nk;            // queries and keys that count
  int rows;              // rows of the owned side, all of which are written
  int first;             // first owned column
};

// Tile t in the order of the launch, which starts with those that have most to do: of a causal mask's queries the last
// ones, of its keys the first; of up to 62 packed sequences those that see most (16411 tokens in 7 sequences, 8 heads of
// 32, bf16: forward 165 -> 154 us, grad q 166 -> 155, grad k v 203 -> 191).
template <bool KEYS> __device__ __forceinline__ bool find_work(const Args &p, int t, int per, Work &w) {
  const int unit = KEYS ? 1 : p.G;
  const bool sorted = p.q_start && p.E + 2 <= 64;
  if (!KEYS && !sorted) t = p.tiles - 1 - t;
  if (!p.q_start) {
    const int e = t / p.tiles_item;
    w.item = e;
    w.q0 = w.k0 = 0;
    const auto held = [](const int64_t *len, int e, int rows) __attribute__((always_inline)) {
      if (!len) return rows;
      const int64_t v = len[e];
      return v < 0 ? 0 : (int)(v < rows ? v : rows);
    };
    w.nq = held(p.q_len, e, p.Sq);
    w.nk = held(p.k_len, e, p.Sk);
    w.rows = KEYS ? p.Sk : p.Sq;
    w.first = (t - e * p.tiles_item) * per;
    return true;
  }
  if (p.table) {
    const int4 a = p.table[2 * t], b = p.table[2 * t + 1];
    w = Work{0, a.x, a.y, a.z, a.w, b.x, b.y};
    return b.y >= 0;
  }
  using ops3d_segments::Segment;
  using ops3d_segments::segment_at;
  const int lane = threadIdx.x & 63;
  const int64_t *own = KEYS ? p.k_start : p.q_start, *other = KEYS ? p.q_start : p.k_start;
  const int own_count = KEYS ? p.k_count : p.q_count, other_count = KEYS ? p.q_count : p.k_count;
  const int own_rows = KEYS ? p.Sk : p.Sq, other_rows = KEYS ? p.Sq : p.Sk;
  int carry = 0, before = 0, j = -1, lower = 0, rows = 0, first = 0;
  if (sorted) {   // a lane a segment
    const Segment s = segment_at(own, own_count, own_rows, lane, carry);
    carry = 0;
    const Segment o = segment_at(other, other_count, other_rows, lane, carry);
    const int own_n = lane < p.E + 2 ? s.upper - s.lower : 0, other_n = lane >= 1 && lane <= p.E ? o.upper - o.lower : 0;
    const int tiles = (int)(((int64_t)own_n * unit + per - 1) / per);
    for (int l = 0; l < p.E + 2; ++l) {
      const int most = __builtin_amdgcn_readlane(other_n, l), n = __builtin_amdgcn_readlane(tiles, l);
      if (most > other_n || (most == other_n && l < lane)) before += n;
    }
    const uint64_t m = __ballot(t >= before && t < before + tiles);
    if (!m) return false;
    const int src = __builtin_ctzll(m), nth = t - __builtin_amdgcn_readlane(before, src), n = __builtin_amdgcn_readlane(tiles, src);
    lower = __builtin_amdgcn_readlane(s.lower, src);
    rows = __builtin_amdgcn_readlane(own_n, src);
    const int o_lower = __builtin_amdgcn_readlane(o.lower, src), o_rows = __builtin_amdgcn_readlane(other_n, src);
    const int counted = src >= 1 && src <= p.E ? rows : 0;   // rows of no sequence: none that count
    w = Work{0, KEYS ? o_lower : lower, KEYS ? lower : o_lower, KEYS ? o_rows : counted, KEYS ? counted : o_rows, rows,
             (p.causal && !KEYS ? n - 1 - nth : nth) * per};
    return true;
  }
  for (int base = 0; base < p.E + 2 && j < 0; base += 64) {
    const Segment s = segment_at(own, own_count, own_rows, base + lane, carry);
    const int tiles = base + lane < p.E + 2 ? (int)(((int64_t)(s.upper - s.lower) * unit + per - 1) / per) : 0;
    const int incl = before + ops3d_segments::scan_add(tiles);
    const uint64_t m = __ballot(incl > t);
    before = __builtin_amdgcn_readlane(incl, 63);
    if (m) {
      const int src = __builtin_ctzll(m);
      j = base + src;
      lower = __builtin_amdgcn_readlane(s.lower, src);
      rows = __builtin_amdgcn_readlane(s.upper, src) - lower;
      first = (t - (__builtin_amdgcn_readlane(incl, src) - __builtin_amdgcn_readlane(tiles, src))) * per;
    }
  }
  if (j < 0) return false;
  int o_lower = 0, o_rows = 0;
  if (j >= 1 && j <= p.E) {
    carry = 0;
    for (int base = 0; base <= j; base += 64) {
      const Segment s = segment_at(other, other_count, other_rows, base + lane, carry);
      if (j < base + 64) {
        o_lower = __builtin_amdgcn_readlane(s.lower, j - base);
        o_rows = __builtin_amdgcn_readlane(s.upper, j - base) - o_lower;
      }
    }
  }
  const bool in = j >= 1 && j <= p.E;   // rows of no sequence: none that count
  w.item = 0;
  w.q0 = KEYS ? o_lower : lower;
  w.k0 = KEYS ? lower : o_lower;
  w.nq = KEYS ? o_rows : (in ? rows : 0);
  w.nk = KEYS ? (in ? rows : 0) : o_rows;
  w.rows = rows;
  w.first = first;
  return true;
}

// The work of each of n tiles of many sequences (more than a wave looks over in a step or two), for a kernel's blocks
// to look up: {q0, k0, nq, nk}, {rows, first, 0, 0}, first -1 where there is none.  One block: each thread has a run of
// segments, whose bounds and tiles depend on the runs before, scanned in LDS.  Forward, bf16, 8 heads of 32: 4096
// sequences of 16 tokens 156 us (2487 where each block walks over them), 1000 of 50: 40 (135), 16384 of 4: 534 (22188).
constexpr int kWalk = 64;   // sequences that blocks find by themselves
template <bool KEYS> __global__ __launch_bounds__(1024) void table_kernel(Args p, int per, int4 *table, int n) {
  __shared__ int scan[3][1024];
  const int64_t *own = KEYS ? p.k_start : p.q_start, *other = KEYS ? p.q_start : p.k_start;
  const int own_count = KEYS ? p.k_count : p.q_count, other_count = KEYS ? p.q_count : p.k_count;
  const int own_rows = KEYS ? p.Sk : p.Sq, other_rows = KEYS ? p.Sq : p.Sk;
  const int unit = KEYS ? 1 : p.G, t = threadIdx.x, run = (p.E + 2 + 1023) / 1024;
  const int begin = min(p.E + 2, t * run), end = min(p.E + 2, begin + run);
  const auto entry = [](const int64_t *start, int count, int rows, int j) __attribute__((always_inline)) {
    const int64_t v = j < count ? start[j] : (int64_t)rows;
    return v < 0 ? 0 : (int)(v < rows ? v : rows);
  };
  int most[2] = {0, 0};   // of the run's entries
  for (int j = begin; j < end; ++j) {
    most[0] = max(most[0], entry(own, own_count, own_rows, j));
    most[1] = max(most[1], entry(other, other_count, other_rows, j));
  }
  scan[0][t] = most[0];
  scan[1][t] = most[1];
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    const int a = t >= o ? scan[0][t - o] : 0, b = t >= o ? scan[1][t - o] : 0;
    __syncthreads();
    scan[0][t] = max(scan[0][t], a);
    scan[1][t] = max(scan[1][t], b);
    __syncthreads();
  }
  const int lower = t ? scan[0][t - 1] : 0, o_lower = t ? scan[1][t - 1] : 0;   // where the run's first segment starts
  int tiles = 0, from = lower;
  for (int j = begin; j < end; ++j) {
    const int to = max(from, entry(own, own_count, own_rows, j));
    tiles += (int)(((int64_t)(to - from) * unit + per - 1) / per);
    from = to;
  }
  scan[2][t] = tiles;
  __syncthreads();
  for (int o = 1; o < 1024; o <<= 1) {
    const int a = t >= o ? scan[2][t - o] : 0;
    __syncthreads();
    scan[2][t] += a;
    __syncthreads();
  }
  int at = t ? scan[2][t - 1] : 0, o_from = o_lower;
  from = lower;
  for (int j = begin; j < end; ++j) {
    const int to = max(from, entry(own, own_count, own_rows, j)), o_to = max(o_from, entry(other, other_count, other_rows, j));
    const bool in = j >= 1 && j <= p.E;   // rows of no sequence: none that count
    const int rows = to - from, o_rows = in ? o_to - o_from : 0, o_at = in ? o_from : 0, counted = in ? rows : 0;
    const int4 a = KEYS ? make_int4(o_at, from, o_rows, counted) : make_int4(from, o_at, counted, o_rows);
    for (int64_t first = 0; first < (int64_t)rows * unit && at < n; first += per, ++at) {
      table[2 * at] = a;
      table[2 * at + 1] = make_int4(rows, (int)first, 0, 0);
    }
    from = to;
    o_from = o_to;
  }
  for (int i = scan[2][1023] + t; i < n; i += 1024) {
    table[2 * i] = make_int4(0, 0, 0, 0);
    table[2 * i + 1] = make_int4(0, -1, 0, 0);
  }
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Tile t of `per` columns, the same for the block.  KEYS: columns are keys, otherwise queries times heads.
template <bool KEYS> __device__ __forceinline__ bool locate(const Args &p, int t, int per, Work &w) {
  Work v{};
  if (!find_work<KEYS>(p, t, per, v)) return false;
  w = Work{uniform(v.item), uniform(v.q0), uniform(v.k0), uniform(v.nq), uniform(v.nk), uniform(v.rows), uniform(v.first)};
  return true;
}

__device__ __forceinline__ int divide(const Args &p, int c) { return (int)(__umulhi((uint32_t)c << 1, p.magic) >> p.shift); }

// A stage of R rows of DP elements in LDS, in 16-byte chunks, XOR-swizzled within the 16 chunks that the banks
// hold: 16 rows and a chunk of each, and 8 rows that follow each other and two neighbouring chunks of each, fall on
// different banks.
template <typename T, int DP, int R, int NT> struct Stage {
  static constexpr int CH = 16 / (int)sizeof(T), RC = DP / CH, NL = R * RC / NT;
  static constexpr int kBytes = R * DP * (int)sizeof(T);
  static_assert(R * RC % NT == 0 && RC >= 4, "chunks divide over the threads");
  static_assert((kBytes & (kBytes - 1)) == 0, "buffers are told apart by a bit of the address");

  // The place of a row among those that share banks (all, every second, every fourth), its upper bit folded
  // into the next one: two rows whose places differ in the lowest bit alone are read in one cycle, whichever way
  // the hardware groups lanes.
  static __device__ __forceinline__ int swizzle(int row) {
    constexpr int kBits = RC >= 16 ? 3 : RC == 8 ? 2 : 1;   // below the row's bit 3
    const int low = (row >> (3 - kBits)) & ((1 << kBits) - 1), top = (row >> 3) & 1;
    return (low ^ (top << (kBits - 1))) << 1 | top;
  }
  static __device__ __forceinline__ int address(int row, int chunk) { return (row * RC + (chunk ^ swizzle(row))) << 4; }
  static __device__ __forceinline__ int row_of(int i) { return (int)(threadIdx.x + i * NT) / RC; }
  static __device__ __forceinline__ int chunk_of(int i) { return (int)(threadIdx.x + i * NT) % RC; }

  // at(row): the row's first element; zeros from row n on and behind D.  n > 0.  Whole chunks are loaded without
  // branches, those outside from the last row's or the row's last place.
  template <typename F> static __device__ __forceinline__ void load(uint4 (&v)[NL], F at, int n, int D) {
    if (D % CH == 0) {
#pragma unroll
      for (int i = 0; i < NL; ++i) v[i] = load16(at(min(row_of(i), n - 1)) + min(chunk_of(i) * CH, D - CH));
      if (n < R || D < DP) {
#pragma unroll
        for (int i = 0; i < NL; ++i)
          if (row_of(i) >= n || chunk_of(i) * CH >= D) v[i] = make_uint4(0, 0, 0, 0);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = row_of(i), col = chunk_of(i) * CH;
      v[i] = make_uint4(0, 0, 0, 0);
      if (row < n && col < D) v[i] = fetch(at(row), 0, 0, col, 1, D);
    }
  }
  // The same without registers between (32768 x 32768 forward, 8 heads of 32, bf16: 1680 us for 2004; the registers let
  // four waves a SIMD run): an instruction of a wave fills 1024 bytes of LDS in lane order, so the
  // lane at a place loads the chunk that the swizzle puts there.  For whole chunks, and rows that start at 16-byte
  // boundaries.  off: the lanes' places, in bytes, of rows at at(row); rows from n on are the last one again.
  // Chunks behind D stay as they are: 0 from clear() on.
  template <typename F> static __device__ __forceinline__ void places(uint32_t (&off)[NL], F at, int n, int D) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int slot = (wave * NL + i) * 64 + lane, row = slot / RC, chunk = (address(row, slot % RC) >> 4) - row * RC;
      off[i] = chunk * CH < D ? at(min(row, n - 1)) + chunk * 16 : ~0u;
    }
  }
  static __device__ __forceinline__ void load_lds(char *lds, const char *base, const uint32_t (&off)[NL], int D) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < NL; ++i)
      if (D == DP || off[i] != ~0u) __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(base + off[i]),
                                       (__attribute__((address_space(3))) void *)(lds + (wave * NL + i) * 1024), 16, 0, 0);
  }
  // A barrier behind which what the block's waves have loaded is in LDS: the compiler waits for no such load.
  static __device__ __forceinline__ void arrived() {
    __builtin_amdgcn_s_waitcnt(0x0f70);   // vmcnt(0)
    __syncthreads();
  }
  static __device__ __forceinline__ void clear(char *lds, int bytes) {
    for (int i = threadIdx.x * 16; i < bytes; i += NT * 16) *reinterpret_cast<uint4 *>(lds + i) = make_uint4(0, 0, 0, 0);
    __syncthreads();
  }
  static __device__ __forceinline__ void store(char *lds, const uint4 (&v)[NL]) {
#pragma unroll
    for (int i = 0; i < NL; ++i) *reinterpret_cast<uint4 *>(lds + address(row_of(i), chunk_of(i))) = v[i];
  }

  // A lane's places in the first of two buffers of two stages, or, flipped, in the second: of its row in a
  // tile of 16 rows at each step of the channels, and of its piece of 4 rows of 16 channels at each 16 channels
  // (16 bits).
  struct Lane {
    int row[DP * (int)sizeof(T) / 64], col[DP / 16];
    __device__ __forceinline__ void flip() {
#pragma unroll
      for (int s = 0; s < DP * (int)sizeof(T) / 64; ++s) row[s] ^= 2 * kBytes;
#pragma unroll
      for (int d = 0; d < DP / 16; ++d) col[d] ^= 2 * kBytes;
    }
  };
  static __device__ __forceinline__ Lane lane_places(int lane) {
    const int i = lane & 15, q = lane >> 4;
    Lane l;
#pragma unroll
    for (int s = 0; s < DP * (int)sizeof(T) / 64; ++s) l.row[s] = address(i, s * 4 + q);
#pragma unroll
    for (int d = 0; d < DP / 16; ++d)
      l.col[d] = sizeof(T) == 2 ? address(q * 4 + (i >> 2), d * 2 + ((i & 3) >> 1)) + (i & 1) * 8 : 0;   // 32 bits: the buffer
    return l;
  }
  // MFMA operand: 16 rows from r0 (a multiple of 16) on, step s of the channels
  static __device__ __forceinline__ typename Type<T>::frag rows(const char *lds, int r0, int s, const Lane &l) {
    return __builtin_bit_cast(typename Type<T>::frag, *reinterpret_cast<const uint4 *>(lds + r0 * RC * 16 + l.row[s]));
  }
  // MFMA operand: 16 channels from 16 d on, summed over rows: in 16 bits rows r0 + 4 q .. + 3 and those 16
  // further, in 32 bits the former.  16 lanes read 4 rows of 16 channels, 4 channels a lane, and get them
  // transposed.
  static __device__ __forceinline__ typename Type<T>::frag columns(const char *lds, int r0, int d, const Lane &l, int lane) {
    if constexpr (sizeof(T) == 2) {
      s16x4 h[2];
#pragma unroll
      for (int p = 0; p < 2; ++p)
        h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4 *)(const_cast<char *>(lds + (r0 + p * 16) * RC * 16 + l.col[d])));
      return __builtin_bit_cast(typename Type<T>::frag, __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
      const int i = lane & 15, q = lane >> 4;
      f32x4 f;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        f[j] = *reinterpret_cast<const float *>(lds + l.col[d] + address(r0 + q * 4 + j, d * 4 + (i >> 2)) + (i & 3) * 4);
      return __builtin_bit_cast(typename Type<T>::frag, f);
    }
  }
};

// Results of one (fp32) or two (16 bits) tiles of 16 rows as the operand of a product summed over them.
template <typename T> __device__ __forceinline__ typename Type<T>::frag operand(const f32x4 *s) {
  if constexpr (sizeof(T) == 4) {
    return s[0];
  } else {
    typename Type<T>::frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)s[j >> 2][j & 3];
    return f;
  }
}

// The operand of a column's row of channels, from memory; zeros behind D, and everywhere without a row.
template <typename T, int STEPS>
__device__ __forceinline__ void load_column(typename Type<T>::frag (&f)[STEPS], const T *row, int D, int q) {
  constexpr int CH = 16 / (int)sizeof(T);
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
    f[s] = __builtin_bit_cast(typename Type<T>::frag, row ? fetch(row, 0, 0, (s * 4 + q) * CH, 1, D) : make_uint4(0, 0, 0, 0));
}

// The output's rounding: what is left of v in T; nothing of an infinity, which would be NaN.
template <typename T> __device__ __forceinline__ f32x4 rest_of(f32x4 v) {
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = fabsf(v[j]) == INFINITY ? 0.f : v[j] - (float)(T)v[j];
  return v;
}

// 4 consecutive channels of a row; those behind D are left out.
template <typename T> __device__ __forceinline__ void store4(T *row, int d, const f32x4 &v, int D) {
  if (d + 4 <= D) {
    struct __attribute__((packed, aligned(sizeof(T)))) Four { T e[4]; } f;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.e[j] = (T)v[j];
    *reinterpret_cast<Four *>(row + d) = f;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (d + j < D) row[d + j] = (T)v[j];
  }
}

__device__ __forceinline__ f32x4 splat(float x) { return f32x4{x, x, x, x}; }

// A mask's 0 times an infinity or NaN of a hidden row (or of the last row, which stands in for those behind it) would be
// NaN.  Stages with hidden rows are looked over: by
// their results, where each row has some, or else by the operand times 0, which is NaN where one of its rows is not
// finite.
template <int N> __device__ __forceinline__ bool finite_results(const f32x4 *s) {
  float z = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) z = fmaf(s[i][j], 0.f, z);
  return !__ballot(z != z);
}
template <typename T, int DP, int ROWS, typename ST>
__device__ __forceinline__ bool all_finite(const char *lds, int r0, const typename ST::Lane &at, int lane) {
  f32x4 z = splat(0.f);
#pragma unroll
  for (int r = 0; r < ROWS; r += sizeof(T) == 2 ? 32 : 16)
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) z = Type<T>::mma(ST::columns(lds, r0 + r, d, at, lane), typename Type<T>::frag{}, z);
  return !__ballot(z[0] != z[0] || z[1] != z[1] || z[2] != z[2] || z[3] != z[3]);
}
// acc += a b row by row of the sum, for the columns that see the row: seen(row).
template <typename T, typename F>
__device__ __forceinline__ void add_seen(f32x4 &acc, const typename Type<T>::frag &a, const typename Type<T>::frag &b, int q, F seen) {
  constexpr int N = 16 / (int)sizeof(T);
#pragma unroll 1
  for (int e = 0; e < 4 * N; ++e) {
    const int owner = e / N, j = e % N;
    typename Type<T>::frag one_a, one_b;   // this row's alone: another's infinity times 0 would be NaN
#pragma unroll
    for (int k = 0; k < N; ++k) {
      one_a[k] = k == j && q == owner ? a[k] : (T)0.f;
      one_b[k] = k == j && q == owner ? b[k] : (T)0.f;
    }
    const f32x4 x = Type<T>::mma(one_a, one_b, splat(0.f));
    if (seen((j >> 2) * 16 + owner * 4 + (j & 3))) acc += x;
  }
}

// 16-bit fractions as fp16 numbers lose precision below 2^-14, so that of P is kept 2^kShift up; with the
// slack below, P stays under 2^15.
template <typename T> struct Range {
  static constexpr float kShift = 0.f, kSlack = 8.f;
  static constexpr bool kScaled = false;
};
template <> struct Range<_Float16> {
  static constexpr float kShift = 10.f, kSlack = 4.f;
  static constexpr bool kScaled = true;   // see Scale
};

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// fp16: dS has no bounds of its own (grad_out may be scaled, and P is small where keys are many), so a column's is held
// times a power of two, chosen like the softmax's reference: the first that are not 0 come to 2^9 at most, and so do, with
// the sums so far, those of which one would pass 2^15.  The maxima and the branch cost 2 to 18 % of the backward (16411 tokens
// in 7 sequences, 8 heads of 32: 309 -> 342 us; 8192 causal tokens in 5, 16/4 heads of 128: 355 -> 361).
struct Scale {
  float top = 0.f;   // what raises it: 2^15 over the power, or 0 where there is none yet
  __device__ __forceinline__ float power() const { return __uint_as_float(0x86800000u - __float_as_uint(top)); }   // finite for 0 too
  __device__ __forceinline__ float inverse() const { return top * 0x1p-15f; }
  // most: the largest size of the lane's new ones
  template <int N> __device__ __forceinline__ void raise(float most, f32x4 (&sums)[N]) {
    most = ops3d_reduce::across32<ops3d_reduce::Max>(ops3d_reduce::across16<ops3d_reduce::Max>(most));
    if (!(most > top)) return;
    const int e = 9 - __builtin_amdgcn_frexp_expf(fminf(most, 0x1p127f));   // the power's exponent
    const float now = __uint_as_float((uint32_t)(127 + 15 - max(-111, min(100, e))) << 23), change = top * __uint_as_float(0x7f000000u - __float_as_uint(now));   // powers of two, 1 over now not 0
#pragma unroll
    for (int i = 0; i < N; ++i) sums[i] *= change;
    top = now;
  }
};

// dS as operands of products that are summed to sums, NC columns of PR tiles.
template <typename F, int NC, int PR, int N>
__device__ __forceinline__ void scaled(F (&f)[NC], f32x4 (&ds)[NC][PR], Scale (&scale)[NC], f32x4 (&sums)[NC][N]) {
  float most[NC];
  bool raise = false;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    most[n] = 0.f;
#pragma unroll
    for (int u = 0; u < PR; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) most[n] = fmaxf(most[n], fabsf(ds[n][u][j]));
    raise |= most[n] > scale[n].top;
  }
  if (__ballot(raise)) {
#pragma unroll
    for (int n = 0; n < NC; ++n) scale[n].raise(most[n], sums[n]);
  }
#pragma unroll
  for (int n = 0; n < NC; ++n) {
#pragma unroll
    for (int u = 0; u < PR; ++u) ds[n][u] *= scale[n].power();
    f[n] = operand<_Float16>(ds[n]);
  }
}

// The block's place: key head, part and tile.  Blocks go to XCD block % 8, so with 8 key heads one has a head, whose rows its L2 then keeps.
__device__ __forceinline__ void place(const Args &p, int &h, int &part, int &tile) {
  const int block = blockIdx.x + p.block0, r = block / p.Hk;
  h = block - r * p.Hk;
  part = r % p.splits;
  tile = r / p.splits;
}

// Adds the waves' results of a block whose WK waves had each a share of the rows: lane by lane through LDS,
// wave 0 has the sum.  f(i): the i-th of n results.
template <int WK, int N, typename F> __device__ __forceinline__ void add_waves(char *lds, int wk, int lane, F f) {
  f32x4 *x = reinterpret_cast<f32x4 *>(lds);
  __syncthreads();
  if (wk) {
#pragma unroll
    for (int i = 0; i < N; ++i) x[((wk - 1) * N + i) * 64 + lane] = f(i);
  }
  __syncthreads();
  if (wk == 0) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int k = 0; k < WK - 1; ++k) f(i) += x[(k * N + i) * 64 + lane];
  }
}

// ---------------------------------------------------------------------------------------------
// Forward: WC waves of NC x 16 columns side by side, and WK of them that share out each stage's KT keys.
// Vector instructions issue in 79 % of the cycles and the matrix units are busy in 37 % at 32 channels (32768 x
// 32768, 8 heads, bf16: 1700 us); where sequences differ, blocks that end early leave fewer waves: 64 and 23 % (16411
// tokens in 7 sequences: 154 us), at 128 channels 36 and 31 % (8192 causal tokens in 5 sequences, 16/4 heads: 143 us).  LDS
// is read without bank conflicts, two buffers of KT keys and values hide the loads.  One query of 32/8 heads over 8
// caches of 8192 tokens, 128 channels: 41 us of which 33 are its bytes.
// Tried: 4 x 16 columns a wave 1700 us beside 1745 then (and less to share out among the CUs), 128 keys a stage 1990,
// the sums of P by fp32 additions alone 1835, the scale multiplied into Q beforehand (as two 16-bit terms, to be exact)
// 1820 beside 1720.
template <typename T, int DP, int NC, int WC, int WK, int KT, int OCC, bool DMA>
__global__ __launch_bounds__(64 * WC *WK) __attribute__((amdgpu_waves_per_eu(OCC))) void forward_kernel(Args p) {
  constexpr int NT = 64 * WC * WK, BM = WC * NC * 16, KW = KT / WK, KN = KW / 16;
  constexpr int STEPS = DP * (int)sizeof(T) / 64, DT = DP / 16, PR = sizeof(T) == 2 ? 2 : 1;   // tiles an operand holds
  typedef Stage<T, DP, KT, NT> ST;
  static_assert(KN % PR == 0, "whole operands");
  constexpr int kMerge = (WK - 1) * NC * (DT + 1) * 1024;
  constexpr int kLds = 4 * ST::kBytes > kMerge ? 4 * ST::kBytes : kMerge;
  __shared__ __attribute__((aligned(16))) char lds[kLds];

  int h, part, tile;
  place(p, h, part, tile);
  Work w;
  if (!locate<false>(p, tile, BM, w)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const int wc = wave % WC, wk = wave / WC;
  const int active = w.nq * p.G, off = w.nk - w.nq, c0 = w.first + wc * NC * 16;
  const T *qb = static_cast<const T *>(p.q.p) + w.item * p.q.item + w.q0 * p.q.token + (int64_t)h * p.G * p.q.head;
  const T *kb = static_cast<const T *>(p.k.p) + w.item * p.k.item + w.k0 * p.k.token + h * p.k.head;
  const T *vb = static_cast<const T *>(p.v.p) + w.item * p.v.item + w.k0 * p.v.token + h * p.v.head;

  typename Type<T>::frag qf[NC][STEPS];
  int limit[NC];   // keys that the column sees; those of columns that do not count are not held back
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int c = c0 + n * 16 + i, t = divide(p, c);
    load_column<T, STEPS>(qf[n], c < active ? qb + t * p.q.token + (c - t * p.G) * p.q.head : nullptr, p.D, q);
    limit[n] = p.causal && c < active ? min(w.nk, t + off + 1) : w.nk;
  }
  // what every column of the block sees: its first column's keys
  const int least = uniform(p.causal ? min(w.nk, max(0, divide(p, w.first) + off + 1)) : w.nk);
  // keys that any column of the block sees, and this part of them
  int keys = w.first < active ? w.nk : 0;
  if (p.causal && keys) keys = uniform(max(0, min(keys, divide(p, min(active, w.first + BM) - 1) + off + 1)));
  int k_begin = 0, k_end = keys;
  if (p.splits > 1) {
    const int per = ((keys + KT - 1) / KT + p.splits - 1) / p.splits * KT;
    k_begin = min(keys, part * per);
    k_end = min(keys, k_begin + per);
  }

  // sums of P V and of P; in 16 bits the latter by the matrix units, from the rounded P, and where the backward is to
  // have its logarithm, of P as it is too: the rounded sum's would put the same error into all of a row's gradients
  f32x4 o[NC][DT], sum[NC];
  float m[NC], mc[NC], l[NC], top[NC];     // reference, the same times c, sum of P (this lane's rows), what raises it
  constexpr bool SUMS = sizeof(T) == 2;
  const bool exact = !SUMS || p.lse;
  constexpr float kShift = Range<T>::kShift;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    m[n] = top[n] = -INFINITY;
    mc[n] = -kShift;
    l[n] = 0.f;
    sum[n] = splat(0.f);
#pragma unroll
    for (int d = 0; d < DT; ++d) o[n][d] = splat(0.f);
  }
  const float slack = Range<T>::kSlack / p.c;

  uint4 kv[DMA ? 1 : ST::NL], vv[DMA ? 1 : ST::NL];
  uint32_t k_off[DMA ? ST::NL : 1], v_off[DMA ? ST::NL : 1];
  if constexpr (DMA) {
    ST::places(k_off, [&](int r) { return r * (uint32_t)(p.k.token * sizeof(T)); }, KT, p.D);
    ST::places(v_off, [&](int r) { return r * (uint32_t)(p.v.token * sizeof(T)); }, KT, p.D);
  }
  const auto load = [&](int k0, int buf) __attribute__((always_inline)) {
    const int left = k_end - k0;
    if constexpr (DMA) {
      char *const lk = lds + buf * 2 * ST::kBytes;
      if (left < KT) {
        ST::places(k_off, [&](int r) { return r * (uint32_t)(p.k.token * sizeof(T)); }, left, p.D);
        ST::places(v_off, [&](int r) { return r * (uint32_t)(p.v.token * sizeof(T)); }, left, p.D);
      }
      ST::load_lds(lk, reinterpret_cast<const char *>(kb + k0 * p.k.token), k_off, p.D);
      ST::load_lds(lk + ST::kBytes, reinterpret_cast<const char *>(vb + k0 * p.v.token), v_off, p.D);
    } else {
      ST::load(kv, [&](int r) { return kb + (k0 + r) * p.k.token; }, left, p.D);
      ST::load(vv, [&](int r) { return vb + (k0 + r) * p.v.token; }, left, p.D);
    }
  };
  const int r0 = wk * KW;
  typename ST::Lane at = ST::lane_places(lane);
  const char *const lk = lds, *const lv = lds + ST::kBytes;
  int k0 = k_begin, buf = 0;
  const auto stage = [&](auto masked) __attribute__((always_inline)) {
    if constexpr (!DMA) {
      ST::store(lds + buf * 2 * ST::kBytes, kv);
      ST::store(lds + buf * 2 * ST::kBytes + ST::kBytes, vv);
      if (k0 + KT < k_end) load(k0 + KT, 0);
      __syncthreads();   // the other buffer's readers are past the barrier before
    } else {
      ST::arrived();     // this stage, everywhere; and the other buffer's readers are done
      if (k0 + KT < k_end) load(k0 + KT, buf ^ 1);
    }

    f32x4 s[NC][KN];
#pragma unroll
    for (int kt = 0; kt < KN; ++kt) {
#pragma unroll
      for (int n = 0; n < NC; ++n) s[n][kt] = splat(0.f);
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        const auto kf = ST::rows(lk, r0 + kt * 16, st, at);
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][kt] = Type<T>::mma(kf, qf[n][st], s[n][kt]);
      }
    }
    if constexpr (decltype(masked)::value) {   // also keys behind the last
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int kt = 0; kt < KN; ++kt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (k0 + r0 + kt * 16 + q * 4 + j >= limit[n]) s[n][kt][j] = -INFINITY;
    }
    const bool finite = !decltype(masked)::value || all_finite<T, DP, KW, ST>(lv, r0, at, lane);
    bool raise = false;
    float mx[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      mx[n] = s[n][0][0];
#pragma unroll
      for (int kt = 0; kt < KN; ++kt)
#pragma unroll
        for (int j = 0; j < 4; ++j) mx[n] = fmaxf(mx[n], s[n][kt][j]);
      raise |= mx[n] > top[n];
    }
    if (__ballot(raise)) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const float now = fmaxf(m[n], ops3d_reduce::across32<ops3d_reduce::Max>(ops3d_reduce::across16<ops3d_reduce::Max>(mx[n])));
        if (now != m[n]) {
          const float by = m[n] == -INFINITY ? 0.f : exp2_((m[n] - now) * p.c);
          l[n] *= by;
          sum[n] *= by;
#pragma unroll
          for (int d = 0; d < DT; ++d) o[n][d] *= by;
          m[n] = now;
          mc[n] = now * p.c - kShift;
          top[n] = now + slack;
        }
      }
    }
#pragma unroll
    for (int kt = 0; kt < KN; kt += PR) {
      typename Type<T>::frag pf[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
#pragma unroll
        for (int u = 0; u < PR; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][kt + u][j] = exp2_(fmaf(s[n][kt + u][j], p.c, -mc[n]));
        if (exact) {
#pragma unroll
          for (int u = 0; u < PR; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j) l[n] += s[n][kt + u][j];
        }
        pf[n] = operand<T>(&s[n][kt]);
        if (SUMS) sum[n] = Type<T>::mma(Type<T>::ones(), pf[n], sum[n]);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const auto vf = ST::columns(lv, r0 + kt * 16, d, at, lane);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          if (!decltype(masked)::value || finite) o[n][d] = Type<T>::mma(vf, pf[n], o[n][d]);
          else add_seen<T>(o[n][d], vf, pf[n], q, [&](int r) { return k0 + r0 + kt * 16 + r < limit[n]; });
        }
      }
    }
    k0 += KT;
    buf ^= 1;
    at.flip();
  };
  if (DMA && p.D < DP) ST::clear(lds, 4 * ST::kBytes);
  if (k_begin < k_end) load(k_begin, 0);
  while (k0 < k_end && k0 + KT <= least) stage(std::false_type());
  while (k0 < k_end) stage(std::true_type());
  float whole[NC];   // what the output is divided by
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] = ops3d_reduce::across32<ops3d_reduce::Add>(ops3d_reduce::across16<ops3d_reduce::Add>(l[n]));
    whole[n] = SUMS ? sum[n][0] : l[n];
    m[n] *= p.c;   // from here on log2
  }

  if constexpr (WK > 1) {   // the waves' shares, each with its own reference
    f32x4 *x = reinterpret_cast<f32x4 *>(lds);
    __syncthreads();
    if (wk) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        f32x4 *y = x + (((wk - 1) * WC + wc) * NC + n) * (DT + 1) * 64 + lane;
#pragma unroll
        for (int d = 0; d < DT; ++d) y[d * 64] = o[n][d];
        y[DT * 64] = f32x4{m[n], whole[n], l[n], 0.f};
      }
    }
    __syncthreads();
    if (wk) return;
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int k = 0; k < WK - 1; ++k) {
        const f32x4 *y = x + ((k * WC + wc) * NC + n) * (DT + 1) * 64 + lane;
        const float mk = y[DT * 64][0], now = fmaxf(m[n], mk);
        const float a = m[n] == -INFINITY ? 0.f : exp2_(m[n] - now), b = mk == -INFINITY ? 0.f : exp2_(mk - now);
        whole[n] = whole[n] * a + y[DT * 64][1] * b;
        l[n] = l[n] * a + y[DT * 64][2] * b;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[n][d] = o[n][d] * a + y[d * 64] * b;
        m[n] = now;
      }
  }

  const int64_t cell0 = ((int64_t)(w.item * p.Hk + h) * p.Sq + w.q0) * p.G;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int c = c0 + n * 16 + i;
    if (c >= w.rows * p.G) continue;
    // 0 for columns that do not count or see no key.  By what they see: a sum of 0 is also that of logits of minus
    // infinity, whose softmax is NaN.
    const bool none = c >= active || limit[n] <= 0;
    if (p.splits > 1) {
      const int64_t to = part * p.cells + cell0 + c;
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(p.part + to * DP + d * 16 + q * 4) = o[n][d];
      if (q == 0) p.part_ml[to] = none ? f32x4{-INFINITY, 0.f, 0.f, 0.f} : f32x4{m[n], whole[n], l[n], 1.f};
      continue;
    }
    const float inv = none ? 0.f : 1.f / whole[n];
    const int t = divide(p, c);
    const int head = h * p.G + c - t * p.G;
    T *const to = static_cast<T *>(p.o.p) + w.item * p.o.item + (w.q0 + t) * p.o.token + head * p.o.head;
    T *const rest = static_cast<T *>(p.rest) + (((int64_t)w.item * p.Sq + w.q0 + t) * (p.Hk * p.G) + head) * p.D;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 v = none ? splat(0.f) : o[n][d] * inv;
      store4(to, d * 16 + q * 4, v, p.D);
      if (p.rest) store4(rest, d * 16 + q * 4, rest_of<T>(v), p.D);
    }
    if (p.lse && q == 0) p.lse[cell0 + c] = none ? INFINITY : m[n] + __builtin_amdgcn_logf(l[n]) - kShift;
  }
}

// The parts of a query and head joined: a wave each, 4 channels a lane, as many parts at a time as that leaves
// lanes for.
template <typename T, int DP> __global__ __launch_bounds__(256) void join_forward_kernel(Args p) {
  constexpr int PER = DP / 4, AT = 64 / PER;   // lanes of a row, parts at a time
  const int64_t cell = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (cell >= p.cells) return;
  const int lane = threadIdx.x & 63, d = lane % PER * 4;
  float m = -INFINITY;
  for (int z = lane; z < p.splits; z += 64) m = fmaxf(m, p.part_ml[z * p.cells + cell][0]);
  m = ops3d_reduce::all<64, ops3d_reduce::Max>(m);
  float whole = 0.f, l = 0.f;
  f32x4 o = splat(0.f);
#pragma unroll 2
  for (int z = lane / PER; z < p.splits; z += AT) {
    const int64_t at = z * p.cells + cell;
    const f32x4 ml = p.part_ml[at], v = *reinterpret_cast<const f32x4 *>(p.part + at * DP + d);
    // without a reference the sums are 0, or NaN where the part's logits are: both count
    const float by = ml[0] == -INFINITY ? 1.f : exp2_(ml[0] - m);
    whole = fmaf(by, ml[1], whole);
    l = fmaf(by, ml[2], l);
    o += v * by;
  }
#pragma unroll
  for (int s = PER; s < 64; s <<= 1) {
    whole += __shfl_xor(whole, s);
    l += __shfl_xor(l, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], s);
  }
  const int per = p.Sq * p.G, ih = (int)(cell / per), c = (int)(cell - (int64_t)ih * per);
  const int item = ih / p.Hk, h = ih - item * p.Hk, t = divide(p, c), head = h * p.G + c - t * p.G;
  const bool none = p.part_ml[cell][3] == 0.f;   // the same in all parts
  const f32x4 v = none ? splat(0.f) : o * (1.f / whole);
  if (lane < PER) {
    store4(static_cast<T *>(p.o.p) + item * p.o.item + t * p.o.token + head * p.o.head, d, v, p.D);
    if (p.rest) store4(static_cast<T *>(p.rest) + (((int64_t)item * p.Sq + t) * (p.Hk * p.G) + head) * p.D, d, rest_of<T>(v), p.D);
  }
  if (p.lse && lane == 0) p.lse[cell] = none ? INFINITY : m + __builtin_amdgcn_logf(l) - Range<T>::kShift;
}

// ---------------------------------------------------------------------------------------------
// Gradient of the queries, and delta = sum of o grad_out, which the keys' needs (gq NULL: that alone).
// The keys' gradient is a kernel of its own, which forms S and dP again: one kernel for both would have to add up
// grad q over the blocks of keys, by atomics in an order that changes results, or in a workspace of one grad q a block.
// 16411 tokens in 7 sequences, 8 heads of 32: 155 us (three products of 30 GF: 583 TFLOP/s; vector units 57 %, matrix units
// 28 % of the cycles); 8192 causal tokens in 5 sequences, 16/4 heads of 128: 165 us (35 and 38 %).  At 128 channels stages are 32 keys
// long: Q, dO and dQ of 128 columns leave registers for no more.
template <typename T, int DP, int NC, int WC, int WK, int KT, int OCC, bool DMA>
__global__ __launch_bounds__(64 * WC *WK) __attribute__((amdgpu_waves_per_eu(OCC))) void grad_q_kernel(Args p) {
  constexpr int NT = 64 * WC * WK, BM = WC * NC * 16, KW = KT / WK, KN = KW / 16;
  constexpr int STEPS = DP * (int)sizeof(T) / 64, DT = DP / 16, PR = sizeof(T) == 2 ? 2 : 1, CH = 16 / (int)sizeof(T);
  typedef Stage<T, DP, KT, NT> ST;
  static_assert(KN % PR == 0, "whole operands");
  constexpr int kMerge = (WK - 1) * NC * DT * 1024;
  constexpr int kLds = 4 * ST::kBytes > kMerge ? 4 * ST::kBytes : kMerge;
  __shared__ __attribute__((aligned(16))) char lds[kLds];

  int h, part, tile;
  place(p, h, part, tile);
  Work w;
  if (!locate<false>(p, tile, BM, w)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const int wc = wave % WC, wk = wave / WC;
  const int active = w.nq * p.G, off = w.nk - w.nq, c0 = w.first + wc * NC * 16;
  const T *kb = static_cast<const T *>(p.k.p) + w.item * p.k.item + w.k0 * p.k.token + h * p.k.head;
  const T *vb = static_cast<const T *>(p.v.p) + w.item * p.v.item + w.k0 * p.v.token + h * p.v.head;
  const int64_t cell0 = ((int64_t)(w.item * p.Hk + h) * p.Sq + w.q0) * p.G;

  typename Type<T>::frag qf[NC][STEPS], gf[NC][STEPS];
  int limit[NC];
  float lse[NC], delta[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int c = c0 + n * 16 + i, t = divide(p, c), head = h * p.G + c - t * p.G;
    const bool in = c < active;
    const auto row = [&](const Tensor &x) __attribute__((always_inline)) {
      return in ? static_cast<const T *>(x.p) + w.item * x.item + (w.q0 + t) * x.token + head * x.head : nullptr;
    };
    load_column<T, STEPS>(qf[n], row(p.q), p.D, q);
    load_column<T, STEPS>(gf[n], row(p.g), p.D, q);
    typename Type<T>::frag of[STEPS], rf[STEPS];
    load_column<T, STEPS>(of, row(p.o), p.D, q);
    load_column<T, STEPS>(rf, in && p.rest ? static_cast<const T *>(p.rest) + (((int64_t)w.item * p.Sq + w.q0 + t) * (p.Hk * p.G) + head) * p.D : nullptr, p.D, q);
    float d = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < CH; ++j) d = fmaf((float)of[s][j] + (float)rf[s][j], (float)gf[n][s][j], d);
    delta[n] = ops3d_reduce::across32<ops3d_reduce::Add>(ops3d_reduce::across16<ops3d_reduce::Add>(d));
    lse[n] = in ? p.lse[cell0 + c] : INFINITY;
    if (c < w.rows * p.G && q == 0 && wk == 0 && part == 0) p.delta[cell0 + c] = delta[n];
    limit[n] = p.causal && in ? min(w.nk, t + off + 1) : w.nk;
  }
  if (!p.gq.p) return;
  const int least = uniform(p.causal ? min(w.nk, max(0, divide(p, w.first) + off + 1)) : w.nk);
  int keys = w.first < active ? w.nk : 0;
  if (p.causal && keys) keys = uniform(max(0, min(keys, divide(p, min(active, w.first + BM) - 1) + off + 1)));
  int k_begin = 0, k_end = keys;
  if (p.splits > 1) {
    const int per = ((keys + KT - 1) / KT + p.splits - 1) / p.splits * KT;
    k_begin = min(keys, part * per);
    k_end = min(keys, k_begin + per);
  }

  f32x4 a[NC][DT];
  Scale scale[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int d = 0; d < DT; ++d) a[n][d] = splat(0.f);
  uint4 kv[DMA ? 1 : ST::NL], vv[DMA ? 1 : ST::NL];
  uint32_t k_off[DMA ? ST::NL : 1], v_off[DMA ? ST::NL : 1];
  if constexpr (DMA) {
    ST::places(k_off, [&](int r) { return r * (uint32_t)(p.k.token * sizeof(T)); }, KT, p.D);
    ST::places(v_off, [&](int r) { return r * (uint32_t)(p.v.token * sizeof(T)); }, KT, p.D);
  }
  const auto load = [&](int k0, int buf) __attribute__((always_inline)) {
    const int left = k_end - k0;
    if constexpr (DMA) {
      char *const lk = lds + buf * 2 * ST::kBytes;
      if (left < KT) {
        ST::places(k_off, [&](int r) { return r * (uint32_t)(p.k.token * sizeof(T)); }, left, p.D);
        ST::places(v_off, [&](int r) { return r * (uint32_t)(p.v.token * sizeof(T)); }, left, p.D);
      }
      ST::load_lds(lk, reinterpret_cast<const char *>(kb + k0 * p.k.token), k_off, p.D);
      ST::load_lds(lk + ST::kBytes, reinterpret_cast<const char *>(vb + k0 * p.v.token), v_off, p.D);
    } else {
      ST::load(kv, [&](int r) { return kb + (k0 + r) * p.k.token; }, left, p.D);
      ST::load(vv, [&](int r) { return vb + (k0 + r) * p.v.token; }, left, p.D);
    }
  };
  const int r0 = wk * KW;
  typename ST::Lane at = ST::lane_places(lane);
  const char *const lk = lds, *const lv = lds + ST::kBytes;
  int k0 = k_begin, buf = 0;
  const auto stage = [&](auto masked) __attribute__((always_inline)) {
    if constexpr (!DMA) {
      ST::store(lds + buf * 2 * ST::kBytes, kv);
      ST::store(lds + buf * 2 * ST::kBytes + ST::kBytes, vv);
      if (k0 + KT < k_end) load(k0 + KT, 0);
      __syncthreads();
    } else {
      ST::arrived();
      if (k0 + KT < k_end) load(k0 + KT, buf ^ 1);
    }
#pragma unroll
    for (int kt = 0; kt < KN; kt += PR) {
      f32x4 s[NC][PR], dp[NC][PR];
#pragma unroll
      for (int u = 0; u < PR; ++u) {
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][u] = splat(0.f), dp[n][u] = splat(-delta[n]);
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          const auto kf = ST::rows(lk, r0 + (kt + u) * 16, st, at), vf = ST::rows(lv, r0 + (kt + u) * 16, st, at);
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            s[n][u] = Type<T>::mma(kf, qf[n][st], s[n][u]);
            dp[n][u] = Type<T>::mma(vf, gf[n][st], dp[n][u]);
          }
        }
      }
      // a key that is not finite has no finite logit
      const bool finite = !decltype(masked)::value || !p.causal || finite_results<NC * PR>(s[0]);
      typename Type<T>::frag ds[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
#pragma unroll
        for (int u = 0; u < PR; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x = exp2_(fmaf(s[n][u][j], p.c, -lse[n])) * dp[n][u][j];
            if (decltype(masked)::value && k0 + r0 + (kt + u) * 16 + q * 4 + j >= limit[n]) x = 0.f;
            s[n][u][j] = x;
          }
        if (!Range<T>::kScaled) ds[n] = operand<T>(s[n]);
      }
      if constexpr (Range<T>::kScaled) scaled(ds, s, scale, a);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const auto kf = ST::columns(lk, r0 + kt * 16, d, at, lane);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          if (!decltype(masked)::value || finite) a[n][d] = Type<T>::mma(kf, ds[n], a[n][d]);
          else add_seen<T>(a[n][d], kf, ds[n], q, [&](int r) { return k0 + r0 + kt * 16 + r < limit[n]; });
        }
      }
    }
    k0 += KT;
    buf ^= 1;
    at.flip();
  };
  if (DMA && p.D < DP) ST::clear(lds, 4 * ST::kBytes);
  if (k_begin < k_end) load(k_begin, 0);
  while (k0 < k_end && k0 + KT <= least) stage(std::false_type());
  while (k0 < k_end) stage(std::true_type());
  if constexpr (Range<T>::kScaled) {
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int d = 0; d < DT; ++d) a[n][d] *= scale[n].inverse();
  }
  if constexpr (WK > 1) {
    static_assert(WC == 1, "the waves' results lie one behind another");
    add_waves<WK, NC * DT>(lds, wk, lane, [&](int k) -> f32x4 & { return a[k / DT][k % DT]; });
    if (wk) return;
  }
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int c = c0 + n * 16 + i, t = divide(p, c);
    if (c >= w.rows * p.G) continue;
    if (p.splits > 1) {
      const int64_t to = part * p.cells + cell0 + c;
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4 *>(p.part + to * DP + d * 16 + q * 4) = c < active ? a[n][d] : splat(0.f);
      continue;
    }
    T *to = static_cast<T *>(p.gq.p) + w.item * p.gq.item + (w.q0 + t) * p.gq.token + ((int64_t)h * p.G + c - t * p.G) * p.gq.head;
#pragma unroll
    for (int d = 0; d < DT; ++d)
      store4(to, d * 16 + q * 4, c < active ? a[n][d] * p.scale : splat(0.f), p.D);
  }
}

// ---------------------------------------------------------------------------------------------
// Gradients of keys and values.  A block owns keys, and queries, output gradients and their two statistics come by: the
// heads of a group are rows like any other, so their sum is part of the product's.
// 16411 tokens in 7 sequences, 8 heads of 32: 185 us (four products of 30 GF: 650 TFLOP/s; vector units 55 %, matrix units
// 32 % of the cycles); 8192 causal tokens in 5 sequences, 16/4 heads of 128: 257 us and 16 for the join (26 and 33 %, LDS
// 38 %: the operands of four products pass through it for 16 columns a wave, since K, V, dK and dV of 32 columns need
// more registers than two waves a SIMD have; with them 374 us where these tiles took 273 in one part).
template <typename T, int DP, int NC, int WC, int WK, int QT, int OCC, bool DMA>
__global__ __launch_bounds__(64 * WC *WK) __attribute__((amdgpu_waves_per_eu(OCC))) void grad_kv_kernel(Args p) {
  constexpr int NT = 64 * WC * WK, BN = WC * NC * 16, QW = QT / WK, QN = QW / 16;
  constexpr int STEPS = DP * (int)sizeof(T) / 64, DT = DP / 16, PR = sizeof(T) == 2 ? 2 : 1;
  typedef Stage<T, DP, QT, NT> ST;
  static_assert(QN % PR == 0 && QT <= NT, "whole operands, a thread a row");
  constexpr int kMerge = (WK - 1) * NC * DT * 1024;
  constexpr int kStages = 4 * ST::kBytes + 4 * QT * 4;   // and the rows' lse and delta
  constexpr int kLds = kStages > kMerge ? kStages : kMerge;
  __shared__ __attribute__((aligned(16))) char lds[kLds];

  int h, part, tile;
  place(p, h, part, tile);
  Work w;
  if (!locate<true>(p, tile, BN, w)) return;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, i = lane & 15, q = lane >> 4;
  const int wc = wave % WC, wk = wave / WC;
  const int active = w.nq * p.G, off = w.nk - w.nq, j0 = w.first + wc * NC * 16;
  const auto rows_of = [&](const Tensor &x) __attribute__((always_inline)) { return static_cast<const T *>(x.p) + w.item * x.item + w.q0 * x.token + (int64_t)h * p.G * x.head; };
  const T *qb = rows_of(p.q), *gb = rows_of(p.g);
  const int64_t cell0 = ((int64_t)(w.item * p.Hk + h) * p.Sq + w.q0) * p.G;

  typename Type<T>::frag kf[NC][STEPS], vf[NC][STEPS];
  int since[NC];   // the first column of queries that sees the key
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int j = j0 + n * 16 + i;
    const auto row = [&](const Tensor &x) __attribute__((always_inline)) {
      return j < w.nk ? static_cast<const T *>(x.p) + w.item * x.item + (w.k0 + j) * x.token + h * x.head : nullptr;
    };
    load_column<T, STEPS>(kf[n], row(p.k), p.D, q);
    load_column<T, STEPS>(vf[n], row(p.v), p.D, q);
    since[n] = p.causal ? (int)min((int64_t)active, max((int64_t)0, (int64_t)(j - off) * p.G)) : 0;
  }
  const int last = w.first + BN - 1;   // of this block
  const int all_see = !p.causal ? 0 : uniform( (int)min((int64_t)active, max((int64_t)0, (int64_t)(last - off) * p.G)));
  int begin = w.first < w.nk ? 0 : active;
  if (p.causal) begin = max(begin, (int)min((int64_t)active, max((int64_t)0, (int64_t)(w.first - off) * p.G)) / QT * QT);
  begin = uniform(begin);
  int c_begin = begin, c_end = active;
  if (p.splits > 1) {
    const int per = ((active - begin + QT - 1) / QT + p.splits - 1) / p.splits * QT;
    c_begin = min(active, begin + part * per);
    c_end = min(active, c_begin + per);
  }

  f32x4 ak[NC][DT], av[NC][DT];
  Scale scale[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int d = 0; d < DT; ++d) ak[n][d] = av[n][d] = splat(0.f);
  uint4 qv[DMA ? 1 : ST::NL], gv[DMA ? 1 : ST::NL];
  uint32_t q_off[ST::NL], g_off[ST::NL];
  float row_lse = INFINITY, row_delta = 0.f;
  const bool fixed = QT % p.G == 0;   // each stage starts at a query, and its rows lie as those of the one before
  const auto place_rows = [&](int c0, int n) __attribute__((always_inline)) {
    const int t0 = fixed ? 0 : uniform(divide(p, c0)), c = fixed ? 0 : c0 - t0 * p.G;
    const auto at = [&](const Tensor &x, int r) __attribute__((always_inline)) {
      const int t = divide(p, c + r);
      return (uint32_t)((t * (uint32_t)x.token + (c + r - t * p.G) * (uint32_t)x.head) * sizeof(T));
    };
    ST::places(q_off, [&](int r) { return at(p.q, r); }, n, p.D);
    ST::places(g_off, [&](int r) { return at(p.g, r); }, n, p.D);
  };
  const auto load = [&](int c0, int buf) __attribute__((always_inline)) {
    const int left = c_end - c0;
    if constexpr (DMA) {
      char *const lq = lds + buf * 2 * ST::kBytes;
      const int t0 = uniform(divide(p, c0));
      if (!fixed || left < QT) place_rows(c0, min(left, QT));
      ST::load_lds(lq, reinterpret_cast<const char *>(qb + t0 * p.q.token), q_off, p.D);
      ST::load_lds(lq + ST::kBytes, reinterpret_cast<const char *>(gb + t0 * p.g.token), g_off, p.D);
    } else {
      const auto at = [&](const T *base, const Tensor &x, int r) __attribute__((always_inline)) {
        const int t = divide(p, c0 + r);
        return base + t * x.token + (c0 + r - t * p.G) * x.head;
      };
      ST::load(qv, [&](int r) { return at(qb, p.q, r); }, left, p.D);
      ST::load(gv, [&](int r) { return at(gb, p.g, r); }, left, p.D);
    }
    if (threadIdx.x < QT) {
      const bool in = (int)threadIdx.x < left;   // P = 0 in the others
      row_lse = in ? p.lse[cell0 + c0 + threadIdx.x] : INFINITY;
      row_delta = in ? p.delta[cell0 + c0 + threadIdx.x] : 0.f;
    }
  };
  if constexpr (DMA) place_rows(0, QT);
  constexpr float kDown = sizeof(T) == 2 ? 1.f / (float)(1 << (int)Range<T>::kShift) : 1.f;
  const int r0 = wk * QW;
  typename ST::Lane at = ST::lane_places(lane);
  const char *const lq = lds, *const lg = lds + ST::kBytes;
  int c0 = c_begin, buf = 0;
  const auto stage = [&](auto masked) __attribute__((always_inline)) {
    float *const ll = reinterpret_cast<float *>(lds + 4 * ST::kBytes) + buf * 2 * QT, *const ld = ll + QT;
    if constexpr (!DMA) {
      ST::store(lds + buf * 2 * ST::kBytes, qv);
      ST::store(lds + buf * 2 * ST::kBytes + ST::kBytes, gv);
    }
    if (threadIdx.x < QT) {
      ll[threadIdx.x] = Range<T>::kShift - row_lse;
      ld[threadIdx.x] = -row_delta;
    }
    if (!DMA && c0 + QT < c_end) load(c0 + QT, 0);
    if (DMA) ST::arrived();
    else __syncthreads();
    if (DMA && c0 + QT < c_end) load(c0 + QT, buf ^ 1);
#pragma unroll
    for (int qt = 0; qt < QN; qt += PR) {
      f32x4 s[NC][PR], dp[NC][PR], lse[PR];
#pragma unroll
      for (int u = 0; u < PR; ++u) {
        const int r = r0 + (qt + u) * 16 + q * 4;
        lse[u] = *reinterpret_cast<const f32x4 *>(ll + r);
        const f32x4 delta = *reinterpret_cast<const f32x4 *>(ld + r);
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][u] = splat(0.f), dp[n][u] = delta;
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          const auto qf = ST::rows(lq, r0 + (qt + u) * 16, st, at), gf = ST::rows(lg, r0 + (qt + u) * 16, st, at);
#pragma unroll
          for (int n = 0; n < NC; ++n) {
            s[n][u] = Type<T>::mma(qf, kf[n][st], s[n][u]);
            dp[n][u] = Type<T>::mma(gf, vf[n][st], dp[n][u]);
          }
        }
      }
      // a query or an output gradient that is not finite has no finite logit or no finite product with a value
      const bool finite = !decltype(masked)::value || (finite_results<NC * PR>(s[0]) && finite_results<NC * PR>(dp[0]));
      typename Type<T>::frag pf[NC], ds[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) {
#pragma unroll
        for (int u = 0; u < PR; ++u) {
          const int r = c0 + r0 + (qt + u) * 16 + q * 4;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float x = exp2_(fmaf(s[n][u][j], p.c, lse[u][j])), y = x * dp[n][u][j];
            if (decltype(masked)::value && (r + j < since[n] || r + j >= c_end)) x = y = 0.f;
            s[n][u][j] = x;
            dp[n][u][j] = y;
          }
        }
        pf[n] = operand<T>(s[n]);
        if (!Range<T>::kScaled) ds[n] = operand<T>(dp[n]);
      }
      if constexpr (Range<T>::kScaled) scaled(ds, dp, scale, ak);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const auto gf = ST::columns(lg, r0 + qt * 16, d, at, lane), qf = ST::columns(lq, r0 + qt * 16, d, at, lane);
#pragma unroll
        for (int n = 0; n < NC; ++n) {
          if (!decltype(masked)::value || finite) {
            av[n][d] = Type<T>::mma(gf, pf[n], av[n][d]);
            ak[n][d] = Type<T>::mma(qf, ds[n], ak[n][d]);
          } else {
            const auto seen = [&](int r) { return c0 + r0 + qt * 16 + r >= since[n] && c0 + r0 + qt * 16 + r < c_end; };
            add_seen<T>(av[n][d], gf, pf[n], q, seen);
            add_seen<T>(ak[n][d], qf, ds[n], q, seen);
          }
        }
      }
    }
    c0 += QT;
    buf ^= 1;
    at.flip();
  };
  if (DMA && p.D < DP) ST::clear(lds, 4 * ST::kBytes);
  if (c_begin < c_end) load(c_begin, 0);
  while (c0 < c_end) {   // rows behind the last are hidden too: an infinite key times their zeros is NaN
    while (c0 < c_end && (c0 < all_see || c_end - c0 < QT)) stage(std::true_type());
    while (c0 >= all_see && c0 + QT <= c_end) stage(std::false_type());
  }
  if constexpr (Range<T>::kScaled) {
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int d = 0; d < DT; ++d) ak[n][d] *= scale[n].inverse() * kDown;
  }
  if constexpr (WK > 1) {
    static_assert(WC == 1, "the waves' results lie one behind another");
    add_waves<WK, NC * DT>(lds, wk, lane, [&](int k) -> f32x4 & { return ak[k / DT][k % DT]; });
    add_waves<WK, NC * DT>(lds, wk, lane, [&](int k) -> f32x4 & { return av[k / DT][k % DT]; });
    if (wk) return;
  }
  const int64_t keys = (int64_t)p.heads * p.Sk;
  const int64_t key0 = (int64_t)(w.item * p.Hk + h) * p.Sk + w.k0;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const int j = j0 + n * 16 + i;
    if (j >= w.rows) continue;
    const bool in = j < w.nk;   // keys that do not count, whose operands are 0, have gathered exp(0) all the same
    if (p.splits > 1) {
      const int64_t to = (part * keys + key0 + j) * 2;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        *reinterpret_cast<f32x4 *>(p.part + to * DP + d * 16 + q * 4) = in ? ak[n][d] : splat(0.f);
        *reinterpret_cast<f32x4 *>(p.part + (to + 1) * DP + d * 16 + q * 4) = in ? av[n][d] * kDown : splat(0.f);
      }
      continue;
    }
    const auto row = [&](const Tensor &x) __attribute__((always_inline)) { return static_cast<T *>(x.p) + w.item * x.item + (w.k0 + j) * x.token + h * x.head; };
    T *const gk = row(p.gk), *const gv = row(p.gv);
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      store4(gk, d * 16 + q * 4, in ? ak[n][d] * p.scale : splat(0.f), p.D);
      store4(gv, d * 16 + q * 4, in ? av[n][d] * kDown : splat(0.f), p.D);
    }
  }
}

// Sums of parts: of grad q (KEYS false), a row a cell; of grad k and grad v, two rows a key.  4 channels a
// thread, the parts in order.
template <typename T, int DP, bool KEYS> __global__ __launch_bounds__(256) void join_sum_kernel(Args p) {
  constexpr int PER = DP / 4;
  const int per = KEYS ? p.Sk : p.Sq * p.G;
  const int64_t n = (int64_t)p.heads * per * (KEYS ? 2 : 1);
  const int64_t at = (int64_t)blockIdx.x * (256 / PER) + threadIdx.x / PER;
  const int d = threadIdx.x % PER * 4;
  if (at >= n || d >= p.D) return;
  const int64_t row = KEYS ? at >> 1 : at;
  const int ih = (int)(row / per), c = (int)(row - (int64_t)ih * per), item = ih / p.Hk, h = ih - item * p.Hk;
  const bool value = KEYS && (at & 1);
  const Tensor &x = KEYS ? (value ? p.gv : p.gk) : p.gq;
  const int t = KEYS ? c : divide(p, c), head = KEYS ? h : h * p.G + c - t * p.G;
  f32x4 s = splat(0.f);
#pragma unroll 4
  for (int z = 0; z < p.splits; ++z) s += *reinterpret_cast<const f32x4 *>(p.part + (z * n + at) * DP + d);
  store4(static_cast<T *>(x.p) + item * x.item + t * x.token + head * x.head, d, value ? s : s * p.scale, p.D);
}

// ---------------------------------------------------------------------------------------------
// Launches (attention_f32.hip and its like).  dp: the padded number of channels, 32, 64 or 128.
// Waves a SIMD that a kernel's registers are to leave room for: two of 256 at least, whose results then stay in
// registers that vector instructions read, where they fit.
enum Kernel { kforward, kgrad_q, kgrad_kv };
template <typename T> constexpr int occupancy(bool direct, int dp, int wk) {
  if (dp <= 32) return direct ? 4 : 3;
  if (dp <= 64) return 2;
  return wk > 1 || sizeof(T) == 4 || !direct ? 1 : 2;
}

// Columns of a block: 128, 64, or 16, of which each of 4 waves takes a quarter of a stage's rows.
enum Shape { kMany = 0, kSome = 1, kFew = 2 };
template <typename T, int DP, Kernel kKernel, typename F> hipError_t with_shape(int shape, F f) {
  typedef std::integral_constant<int, 1> one;
  constexpr int E = (int)sizeof(T) / 2;   // stages of as many bytes in each type
  typedef std::integral_constant<int, 64 / E> rows;
  typedef std::integral_constant<int, 4> four;
  if constexpr (kKernel != kgrad_kv || DP < 128)
    if (shape == kMany)
      return f(std::integral_constant<int, 2>(), four(), one(), std::integral_constant<int, kKernel == kgrad_q && DP == 128 ? 32 : 64 / E>());
  if (shape == kSome) return f(one(), four(), one(), rows());
  return f(one(), one(), four(), std::integral_constant<int, 128 / E>());
}
// The table of a kernel's tiles, where the sequences are many.
template <bool KEYS> Args with_table(Args p, int shape, hipStream_t st) {
  if (p.table) table_kernel<KEYS><<<1, 1024, 0, st>>>(p, shape == kMany ? 128 : shape == kSome ? 64 : 16, const_cast<int4 *>(p.table), p.tiles);
  return p;
}
template <typename F> hipError_t with_dim(int dp, F f) {
  if (dp == 32) return f(std::integral_constant<int, 32>());
  if (dp == 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}
// The launch itself, and its errors.  Those of joins are small: what is cut into parts has few columns.
template <typename K> hipError_t start(K kernel, const Args &p, int threads, hipStream_t st) {
  return ops3d_launch::launch(kernel, (int64_t)p.tiles * p.splits * p.Hk, threads, st, p);
}

template <typename T> hipError_t forward(const Args &args, int dp, int shape, hipStream_t st) {
  const Args p = with_table<false>(args, shape, st);
  return with_dim(dp, [&](auto d) {
    constexpr int DP = decltype(d)::value;
    return with_shape<T, DP, kforward>(shape, [&](auto nc, auto wc, auto wk, auto kt) {
      constexpr int NC = decltype(nc)::value, WC = decltype(wc)::value, WK = decltype(wk)::value, KT = decltype(kt)::value;
      const hipError_t e = p.dma & 1 ? start(forward_kernel<T, DP, NC, WC, WK, KT, occupancy<T>(true, DP, WK), true>, p, 64 * WC * WK, st)
                                     : start(forward_kernel<T, DP, NC, WC, WK, KT, occupancy<T>(false, DP, WK), false>, p, 64 * WC * WK, st);
      if (e != hipSuccess) return e;
      if (p.splits > 1) join_forward_kernel<T, DP><<<(unsigned)((p.cells + 3) / 4), 256, 0, st>>>(p);
      return hipGetLastError();
    });
  });
}
template <typename T> hipError_t grad_q(const Args &args, int dp, int shape, hipStream_t st) {
  const Args p = with_table<false>(args, shape, st);
  return with_dim(dp, [&](auto d) {
    constexpr int DP = decltype(d)::value;
    return with_shape<T, DP, kgrad_q>(shape, [&](auto nc, auto wc, auto wk, auto kt) {
      constexpr int NC = decltype(nc)::value, WC = decltype(wc)::value, WK = decltype(wk)::value, KT = decltype(kt)::value;
      const hipError_t e = p.dma & 1 ? start(grad_q_kernel<T, DP, NC, WC, WK, KT, occupancy<T>(true, DP, WK), true>, p, 64 * WC * WK, st)
                                     : start(grad_q_kernel<T, DP, NC, WC, WK, KT, occupancy<T>(false, DP, WK), false>, p, 64 * WC * WK, st);
      if (e != hipSuccess) return e;
      if (p.splits > 1) join_sum_kernel<T, DP, false><<<(unsigned)((p.cells * (DP / 4) + 255) / 256), 256, 0, st>>>(p);
      return hipGetLastError();
    });
  });
}
template <typename T> hipError_t grad_kv(const Args &args, int dp, int shape, hipStream_t st) {
  const Args p = with_table<true>(args, shape, st);
  return with_dim(dp, [&](auto d) {
    constexpr int DP = decltype(d)::value;
    return with_shape<T, DP, kgrad_kv>(shape, [&](auto nc, auto wc, auto wk, auto kt) {
      constexpr int NC = decltype(nc)::value, WC = decltype(wc)::value, WK = decltype(wk)::value, KT = decltype(kt)::value;
      const hipError_t e = p.dma & 2 ? start(grad_kv_kernel<T, DP, NC, WC, WK, KT, occupancy<T>(true, DP, WK), true>, p, 64 * WC * WK, st)
                                     : start(grad_kv_kernel<T, DP, NC, WC, WK, KT, occupancy<T>(false, DP, WK), false>, p, 64 * WC * WK, st);
      if (e != hipSuccess) return e;
      const int64_t rows = (int64_t)p.heads * p.Sk * 2;
      if (p.splits > 1) join_sum_kernel<T, DP, true><<<(unsigned)((rows * (DP / 4) + 255) / 256), 256, 0, st>>>(p);
      return hipGetLastError();
    });
  });
}

// instantiated in attention_f32.hip, attention_f16.hip and attention_bf16.hip
#define OPS3D_ATTENTION_TYPE(EXTERN, T)                                   \
  EXTERN template hipError_t forward<T>(const Args &, int, int, hipStream_t); \
  EXTERN template hipError_t grad_q<T>(const Args &, int, int, hipStream_t);  \
  EXTERN template hipError_t grad_kv<T>(const Args &, int, int, hipStream_t);
OPS3D_ATTENTION_TYPE(extern, float)
OPS3D_ATTENTION_TYPE(extern, _Float16)
OPS3D_ATTENTION_TYPE(extern, __bf16)

}  // namespace ops3d_attention
