// mx4.cuh — the MXFP4 matrix format of the library: layout, element types and
// the block quantiser.
//
// MXFP4 (the Open Compute Project's Microscaling Formats 1.0): 32 values along
// the summed axis share one power-of-two scale 2^e (E8M0: the byte e + 127,
// 255 = NaN) and are held as E2M1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
// sign).  e = max(floor(log2(max |v|)) - 2, -127), so the largest value lands
// in [4, 8) and saturates at 6; codes round to nearest, ties to even.  A block
// that holds an infinity or a NaN gets the NaN scale.
//
// Layout in memory.  A matrix of `rows` x `cols` is a sequence of row tiles of
// 128 rows; a tile is a sequence of K chunks of 8 blocks (256 values; the last
// chunk may be shorter, blocks rounded up to an even number because one
// tensor-core instruction sums two).  A chunk of n blocks holds
//   scales: ceil(n / 4) groups of 512 bytes, block b of row r at
//           (b / 4) * 512 + (r % 32) * 16 + (r / 32) * 4 + b % 4
//           — what one 32x128b tcgen05.cp spreads over four TMEM columns;
//   codes:  row group r / 8, then block, then row r % 8: 16 bytes each —
//           a block of 8 rows is one 128-byte core matrix of the canonical
//           K-major operand layout without swizzle.
// So a K chunk of a whole tile, or of its first 8n rows, is one contiguous
// run that a single bulk copy brings to shared memory, ready for the tensor
// cores.  Rows and values past the matrix's edge inside a tile are zero.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace mrml {

constexpr int kF32 = 0, kF16 = 1, kBF16 = 30;  // GGML type ids

constexpr int kMxRows = 128;    // rows per tile
constexpr int kMxChunk = 8;     // blocks per K chunk
constexpr int kMxChunkBytes = kMxChunk * kMxRows * 16 + 2 * 512;

__host__ __device__ inline int mx_blocks(int cols) { return (((cols + 31) >> 5) + 1) & ~1; }
__host__ __device__ inline int mx_scale_bytes(int n) { return ((n + 3) >> 2) * 512; }
__host__ __device__ inline int mx_chunk_bytes(int n) { return n * (kMxRows * 16) + mx_scale_bytes(n); }
__host__ __device__ inline size_t mx_tile_bytes(int nb) {
  return (size_t)(nb / kMxChunk) * kMxChunkBytes + (nb % kMxChunk ? mx_chunk_bytes(nb % kMxChunk) : 0);
}
__host__ __device__ inline size_t mx_matrix_bytes(long long rows, int cols) {
  return (size_t)((rows + kMxRows - 1) / kMxRows) * mx_tile_bytes(mx_blocks(cols));
}
// Offsets inside a tile of row r's block b (nb blocks per row).
__host__ __device__ inline size_t mx_code_offset(int nb, int r, int b) {
  const int c = b / kMxChunk, bl = b % kMxChunk, n = nb - c * kMxChunk < kMxChunk ? nb - c * kMxChunk : kMxChunk;
  return (size_t)c * kMxChunkBytes + mx_scale_bytes(n) + (size_t)(r >> 3) * (n * 128) + bl * 128 + (r & 7) * 16;
}
__host__ __device__ inline size_t mx_scale_offset(int r, int b) {
  const int c = b / kMxChunk, bl = b % kMxChunk;
  return (size_t)c * kMxChunkBytes + (bl >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (bl & 3);
}
// Row of a gated matrix ([0, I) gate, [I, 2I) up, 2I = rows): a tile holds 64
// gate rows, then the 64 up rows of the same outputs, so that one product
// tile has both factors of its GeGLU.
__host__ __device__ inline void mx_gated_row(int rows, int row, int& tile, int& r) {
  const int I = rows >> 1, up = row >= I, i = row - (up ? I : 0);
  tile = i >> 6;
  r = (i & 63) + (up << 6);
}

// Eight E2M1 codes, the first in the lowest nibble.  The conversion rounds to
// nearest even and saturates at 6.
__device__ __forceinline__ uint32_t mx_codes8(float v0, float v1, float v2, float v3, float v4, float v5, float v6,
                                              float v7) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v0), "f"(v1), "f"(v2), "f"(v3), "f"(v4), "f"(v5), "f"(v6), "f"(v7));
  return r;
}
// ... of v * inv, inv a power of two.
__device__ __forceinline__ uint32_t mx_pack8(const float* v, float inv) {
  return mx_codes8(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv, v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
}

// Scale byte of a block whose largest |v| has the bits `amax` (as an unsigned
// integer, which orders like the value; NaN above infinity), and the factor
// its values are multiplied by.  2^-e is exact: e <= 125, so 2^-e is normal.
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax, float& inv) {
  const int ex = (int)(amax >> 23);  // biased exponent; 0 for zero and subnormals, 255 for inf and NaN
  if (ex == 255) {
    inv = 0.f;
    return 255u;
  }
  const int e = ex - 2 > 0 ? ex - 2 : 0;  // e + 127
  inv = __uint_as_float((uint32_t)(254 - e) << 23);
  return (uint32_t)e;
}

// Element types: 16-byte vectors to and from f32.
template <int TYPE>
struct Elem;
template <>
struct Elem<kF32> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float get(T x) { return x; }
  static __device__ __forceinline__ T put(float x) { return x; }
  static __device__ __forceinline__ void unpack(uint4 u, float* v) {
    v[0] = __uint_as_float(u.x), v[1] = __uint_as_float(u.y), v[2] = __uint_as_float(u.z), v[3] = __uint_as_float(u.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <>
struct Elem<kF16> {
  using T = __half;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(T x) { return __half2float(x); }
  static __device__ __forceinline__ T put(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ void unpack(uint4 u, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Elem<kBF16> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float get(T x) { return __bfloat162float(x); }
  static __device__ __forceinline__ T put(float x) { return __float2bfloat16_rn(x); }
  static __device__ __forceinline__ void unpack(uint4 u, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// N values of a block held as they came: f32, or pairs of 16-bit floats, whose
// magnitudes are compared two at a time as integers (they order alike, NaN
// above infinity).
template <int TYPE, int N>
struct MxPart {
  static constexpr int kWords = TYPE == kF32 ? N : N / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  // Bits of the largest magnitude, as f32.
  __device__ __forceinline__ uint32_t amax() const {
    uint32_t m = 0;
    if constexpr (TYPE == kF32) {
#pragma unroll
      for (int i = 0; i < N; ++i) m = max(m, w[i] & 0x7fffffffu);
      return m;
    } else {
      // one instruction per pair: the larger magnitude, NaN if either is
#pragma unroll
      for (int i = 0; i < kWords; ++i) {
        if constexpr (TYPE == kBF16) asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
        else asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
      }
      m &= 0x7fff7fffu;
      m = max(m & 0xffffu, m >> 16);
      if constexpr (TYPE == kBF16) return m << 16;
      else return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m))) & 0x7fffffffu;
    }
  }
  // Codes of the values times inv, eight to a word.
  __device__ __forceinline__ void codes(float inv, uint32_t* q) const {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      float v[8];
      if constexpr (TYPE == kF32) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[8 * i + j]);
        q[i] = mx_pack8(v, inv);
      } else if constexpr (TYPE == kBF16) {
        // scaled in pairs: exact, but for values so small that their code is 0
        const uint32_t inv2 = __byte_perm(__float_as_uint(inv), 0, 0x3232);
        uint32_t t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(t[j]) : "r"(w[4 * i + j]), "r"(inv2));
        Elem<TYPE>::unpack(make_uint4(t[0], t[1], t[2], t[3]), v);
        q[i] = mx_codes8(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
      } else {
        Elem<TYPE>::unpack(make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]), v);
        q[i] = mx_pack8(v, inv);
      }
    }
  }
};

// The 32 values of block b of a row that starts at `row`; zero past `cols`.
template <int TYPE>
__device__ __forceinline__ void load_block(const typename Elem<TYPE>::T* row, int b, int cols, bool vec,
                                           MxPart<TYPE, 32>& v) {
  const int c0 = b * 32;
  if (vec && c0 + 32 <= cols) {
    const uint4* p = reinterpret_cast<const uint4*>(row + c0);
#pragma unroll
    for (int i = 0; i < MxPart<TYPE, 32>::kWords / 4; ++i) {
      const uint4 u = __ldg(p + i);
      v.w[4 * i] = u.x, v.w[4 * i + 1] = u.y, v.w[4 * i + 2] = u.z, v.w[4 * i + 3] = u.w;
    }
  } else {
    typename Elem<TYPE>::T t[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) t[i] = c0 + i < cols ? row[c0 + i] : Elem<TYPE>::put(0.f);
    memcpy(v.w, t, sizeof(v.w));
  }
}

// Codes and scale byte of a whole block.
template <int TYPE>
__device__ __forceinline__ uint32_t quantize_block(const MxPart<TYPE, 32>& v, uint4& q) {
  float inv;
  const uint32_t s = mx_scale(v.amax(), inv);
  uint32_t w[4];
  v.codes(inv, w);
  q = make_uint4(w[0], w[1], w[2], w[3]);
  return s;
}

__host__ inline size_t elem_bytes(int type) { return type == kF32 ? 4 : 2; }

}  // namespace mrml
