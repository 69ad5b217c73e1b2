// Element types, MFMA operands and 16-byte chunks of rows, for the kernels whose tensors may start
// anywhere and whose rows may end anywhere.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ops3d_elements {

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

}  // namespace ops3d_elements
