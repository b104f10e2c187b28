// mx4.cu — quantisation to and from the MXFP4 matrix format (mx4.cuh).
//
// All of these kernels are bound by memory: they read each value once and
// write 17/32 byte for it (dequantisation: the other way round).
#include "../../include/mrml_moe.h"
#include "mx4.cuh"
#include "kernels.h"

namespace mrml {

namespace {

// The 32 values of block b of a row that starts at `row`; zero past `cols`.
template <int TYPE>
__device__ __forceinline__ void load_block(const typename Elem<TYPE>::T* row, int b, int cols, bool vec, float (&v)[32]) {
  using E = Elem<TYPE>;
  const int c0 = b * 32;
  if (vec && c0 + 32 <= cols) {
    const uint4* p = reinterpret_cast<const uint4*>(row + c0);
    uint4 u[32 / E::kVec];
#pragma unroll
    for (int i = 0; i < 32 / E::kVec; ++i) u[i] = __ldg(p + i);
#pragma unroll
    for (int i = 0; i < 32 / E::kVec; ++i) E::unpack(u[i], v + i * E::kVec);
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = c0 + i < cols ? E::get(row[c0 + i]) : 0.f;
  }
}

// GGUF blocks of 32 values as source (quant.rs:135-190): Q4_0 holds elements
// 0..15 in the low nibbles and 16..31 in the high ones, offset by 8.
__device__ __forceinline__ void load_gguf_block(const uint8_t* blk, bool q4, float (&v)[32]) {
  const uint16_t* h = reinterpret_cast<const uint16_t*>(blk);  // blocks are 2-byte aligned
  const float d = f16_bits_to_f32(h[0]);
  if (q4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = h[1 + i];
      v[2 * i] = (float)((int)(w & 15) - 8) * d;
      v[2 * i + 1] = (float)((int)((w >> 8) & 15) - 8) * d;
      v[16 + 2 * i] = (float)((int)((w >> 4) & 15) - 8) * d;
      v[16 + 2 * i + 1] = (float)((int)(w >> 12) - 8) * d;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t w = h[1 + i];
      v[2 * i] = (float)(int8_t)(w & 0xff) * d;
      v[2 * i + 1] = (float)(int8_t)(w >> 8) * d;
    }
  }
}

// Writes a block; the four lanes of blocks 4g .. 4g+3 of a row (adjacent
// lanes) store their scale bytes as one word.
__device__ __forceinline__ void store_block(uint8_t* tile, int nb, int r, int b, uint4 q, uint32_t s, bool live) {
  uint32_t w = s << (8 * (b & 3));
  w |= __shfl_xor_sync(0xffffffffu, w, 1);
  w |= __shfl_xor_sync(0xffffffffu, w, 2);
  if (!live) return;
  *reinterpret_cast<uint4*>(tile + mx_code_offset(nb, r, b)) = q;
  if ((b & 3) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, b)) = w;
}

// A warp takes 8 rows x 4 blocks of a tile: each lane one block, so that a
// row is read in 128 contiguous values and every 128-byte line of codes is
// written whole.  TYPE < 0: GGUF blocks.
template <int TYPE>
__global__ void __launch_bounds__(256) mx4_quantize_kernel(const void* __restrict__ src, long long ldx,
                                                           long long mstride, uint8_t* __restrict__ dst, int rows,
                                                           int cols, int gated, int q4, int vec) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nb = mx_blocks(cols), m = blockIdx.y;
  const int tiles = (rows + kMxRows - 1) / kMxRows;
  const int nx = (nb + 31) >> 5, by = blockIdx.x / nx, bx = blockIdx.x % nx;
  const int tile = by >> 4, r = (by & 15) * 8 + (lane >> 2);
  const int b = (bx * 8 + warp) * 4 + (lane & 3);
  int row;
  if (gated) {
    const int I = rows >> 1, i = tile * 64 + (r & 63);
    row = i < I ? (r < 64 ? i : I + i) : rows;
  } else {
    row = tile * kMxRows + r;
  }
  float v[32];
  if (row < rows && b * 32 < cols) {
    if constexpr (TYPE >= 0) {
      using T = typename Elem<TYPE>::T;
      load_block<TYPE>(static_cast<const T*>(src) + m * mstride + row * ldx, b, cols, vec != 0, v);
    } else {
      load_gguf_block(static_cast<const uint8_t*>(src) + (((size_t)m * rows + row) * (cols / 32) + b) * (q4 ? 18 : 34),
                      q4 != 0, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0.f;
  }
  uint4 q;
  const uint32_t s = mx_quantize32(v, q);
  store_block(dst + ((size_t)m * tiles + tile) * mx_tile_bytes(nb), nb, r, b, q, s, b < nb);
}

// Both directions in one read: a CTA stages 64 rows x 128 columns in shared
// memory; each thread then quantises one block along a row and one along a
// column (a block of the transposed matrix).  `dst` [rows][cols] and `dst_t`
// [cols][rows] are written with whole 128-byte lines.
constexpr int kBothRows = 64, kBothCols = 128;
template <int TYPE>
__global__ void __launch_bounds__(256) mx4_quantize_both_kernel(const typename Elem<TYPE>::T* __restrict__ src,
                                                                long long ldx, uint8_t* __restrict__ dst,
                                                                uint8_t* __restrict__ dst_t, int rows, int cols,
                                                                int vec) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int kPitch = kBothCols + 16 / sizeof(T);  // 16-byte aligned rows, shifted by four banks each
  __shared__ __align__(16) T sm[kBothRows * kPitch];
  pdl_wait();
  pdl_trigger();
  const int nx = (cols + kMxRows - 1) / kMxRows * (kMxRows / kBothCols);  // every row of dst_t's tiles
  const int r0 = blockIdx.x / nx * kBothRows, c0 = blockIdx.x % nx * kBothCols;
  for (int i = threadIdx.x; i < kBothRows * (kBothCols / E::kVec); i += 256) {
    const int r = i / (kBothCols / E::kVec), c = (i % (kBothCols / E::kVec)) * E::kVec;
    const T* p = src + (r0 + r) * ldx + c0 + c;
    uint4 u = make_uint4(0, 0, 0, 0);
    if (r0 + r < rows) {
      if (vec && c0 + c + E::kVec <= cols) {
        u = __ldg(reinterpret_cast<const uint4*>(p));
      } else {
        T t[E::kVec];
#pragma unroll
        for (int j = 0; j < E::kVec; ++j) t[j] = c0 + c + j < cols ? p[j] : E::put(0.f);
        memcpy(&u, t, 16);
      }
    }
    *reinterpret_cast<uint4*>(&sm[r * kPitch + c]) = u;
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float v[32];
  uint4 q;
  {
    const int r = warp * 8 + (lane >> 2), b = lane & 3, nb = mx_blocks(cols);
    const uint4* p = reinterpret_cast<const uint4*>(&sm[r * kPitch + b * 32]);
#pragma unroll
    for (int i = 0; i < 32 / E::kVec; ++i) E::unpack(p[i], v + i * E::kVec);
    const uint32_t s = mx_quantize32(v, q);
    const int row = r0 + r, bg = (c0 >> 5) + b;
    store_block(dst + (size_t)(row / kMxRows) * mx_tile_bytes(nb), nb, row % kMxRows, bg, q, s, bg < nb);
  }
  {
    // 16 columns x 2 blocks per warp: a block of 8 columns is one line
    const int c = warp * 16 + (lane & 15), b = lane >> 4, nb = mx_blocks(rows);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = E::get(sm[(b * 32 + i) * kPitch + c]);
    const uint32_t s = mx_quantize32(v, q);
    const int row = c0 + c, bg = (r0 >> 5) + b;
    if (bg < nb) {
      uint8_t* tile = dst_t + (size_t)(row / kMxRows) * mx_tile_bytes(nb);
      *reinterpret_cast<uint4*>(tile + mx_code_offset(nb, row % kMxRows, bg)) = q;
      tile[mx_scale_offset(row % kMxRows, bg)] = (uint8_t)s;
    }
  }
}

__device__ __forceinline__ float e2m1_value(uint32_t code) {
  // magnitude codes 0..7 -> 0, .5, 1, 1.5, 2, 3, 4, 6
  const uint32_t m = code & 7u, ex = m >> 1, f = m & 1u;
  const float a = ex ? __uint_as_float(((ex + 126u) << 23) | (f << 22)) : 0.5f * f;
  return code & 8u ? -a : a;
}

// A lane takes 8 values (4 code bytes); 16 lanes write 128 contiguous values
// of a row.
template <int TYPE>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const uint8_t* __restrict__ src,
                                                             typename Elem<TYPE>::T* __restrict__ dst, long long ldo,
                                                             long long mstride, int rows, int cols, int gated,
                                                             int vec) {
  using E = Elem<TYPE>;
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nx = (cols + 127) / 128, m = blockIdx.y;
  const int row = blockIdx.x / nx * 16 + warp * 2 + (lane >> 4);
  const int c0 = blockIdx.x % nx * 128 + (lane & 15) * 8, b = c0 >> 5;
  if (row >= rows || c0 >= cols) return;
  const int nb = mx_blocks(cols), tiles = (rows + kMxRows - 1) / kMxRows;
  int tile = row / kMxRows, r = row % kMxRows;
  if (gated) mx_gated_row(rows, row, tile, r);
  const uint8_t* t = src + ((size_t)m * tiles + tile) * mx_tile_bytes(nb);
  const uint32_t q = *reinterpret_cast<const uint32_t*>(t + mx_code_offset(nb, r, b) + (lane & 3) * 4);
  const uint32_t s = t[mx_scale_offset(r, b)];
  // 2^(s - 127); s = 0 is the subnormal 2^-127, s = 255 NaN
  const float scale = s == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(s ? s << 23 : 0x00400000u);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = e2m1_value(q >> (4 * i)) * scale;
  typename E::T* o = dst + m * mstride + row * ldo + c0;
  if (vec && c0 + 8 <= cols) {
#pragma unroll
    for (int i = 0; i < 8 / E::kVec; ++i) reinterpret_cast<uint4*>(o)[i] = E::pack(v + i * E::kVec);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c0 + i < cols) o[i] = E::put(v[i]);
  }
}

// Tokens gathered in expert order and quantised on the way: a lane quantises
// one block of a token once and stores it at each of the token's positions.
template <int TYPE>
__global__ void __launch_bounds__(256) mx4_gather_kernel(const typename Elem<TYPE>::T* __restrict__ x, long long ldx,
                                                         const int32_t* __restrict__ pos, uint8_t* __restrict__ dst,
                                                         int T, int H, int K, int vec) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nb = mx_blocks(H), spans = (nb + 31) >> 5;
  const long long i = (long long)blockIdx.x * 8 + warp;
  const int t = (int)(i / spans), b = (int)(i % spans) * 32 + lane;
  if (t >= T) return;
  float v[32];
  if (b * 32 < H) {
    load_block<TYPE>(x + t * ldx, b, H, vec != 0, v);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] = 0.f;
  }
  uint4 q;
  uint32_t s = mx_quantize32(v, q);
  uint32_t w = s << (8 * (b & 3));
  w |= __shfl_xor_sync(0xffffffffu, w, 1);
  w |= __shfl_xor_sync(0xffffffffu, w, 2);
  if (b >= nb) return;
  const size_t tb = mx_tile_bytes(nb);
  const int32_t* p = pos + (size_t)t * K;
  for (int k = 0; k < K; ++k) {
    const int at = p[k];
    if (at < 0) continue;
    uint8_t* tile = dst + (size_t)(at / kMxRows) * tb;
    *reinterpret_cast<uint4*>(tile + mx_code_offset(nb, at % kMxRows, b)) = q;
    if ((b & 3) == 0) *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(at % kMxRows, b)) = w;
  }
}

bool vec_ok(const void* p, long long ld, long long mstride, size_t s) {
  return ((uintptr_t)p & 15) == 0 && (size_t)ld * s % 16 == 0 && (size_t)mstride * s % 16 == 0;
}

}  // namespace

cudaError_t launch_mx4_quantize(int type, const void* x, long long ldx, long long mstride, uint8_t* dst, int rows,
                                int cols, int matrices, bool gated, cudaStream_t s) {
  const int nb = mx_blocks(cols), tiles = (rows + kMxRows - 1) / kMxRows;
  const dim3 grid((unsigned)((nb + 31) / 32 * (long long)tiles * 16), matrices);
  const int vec = type == kF32 || type == kF16 || type == kBF16 ? vec_ok(x, ldx, mstride, elem_bytes(type)) : 0;
  switch (type) {
    case kF32: return launch_pdl(mx4_quantize_kernel<kF32>, grid, 256, 0, s, x, ldx, mstride, dst, rows, cols, (int)gated, 0, vec);
    case kF16: return launch_pdl(mx4_quantize_kernel<kF16>, grid, 256, 0, s, x, ldx, mstride, dst, rows, cols, (int)gated, 0, vec);
    case kBF16: return launch_pdl(mx4_quantize_kernel<kBF16>, grid, 256, 0, s, x, ldx, mstride, dst, rows, cols, (int)gated, 0, vec);
    default: return launch_pdl(mx4_quantize_kernel<-1>, grid, 256, 0, s, x, ldx, mstride, dst, rows, cols, (int)gated, (int)(type == kQ4_0), 0);
  }
}

cudaError_t launch_mx4_quantize_both(int type, const void* x, long long ldx, uint8_t* dst, uint8_t* dst_t, int rows,
                                     int cols, cudaStream_t s) {
  // every row of both matrices' tiles, so that the padding is written too
  const int pr = (rows + kMxRows - 1) / kMxRows * kMxRows, pc = (cols + kMxRows - 1) / kMxRows * kMxRows;
  const dim3 grid((unsigned)((long long)(pc / kBothCols) * (pr / kBothRows)));
  const int vec = vec_ok(x, ldx, 0, elem_bytes(type));
  switch (type) {
    case kF32: return launch_pdl(mx4_quantize_both_kernel<kF32>, grid, 256, 0, s, (const float*)x, ldx, dst, dst_t, rows, cols, vec);
    case kF16: return launch_pdl(mx4_quantize_both_kernel<kF16>, grid, 256, 0, s, (const __half*)x, ldx, dst, dst_t, rows, cols, vec);
    default: return launch_pdl(mx4_quantize_both_kernel<kBF16>, grid, 256, 0, s, (const __nv_bfloat16*)x, ldx, dst, dst_t, rows, cols, vec);
  }
}

cudaError_t launch_mx4_dequantize(int type, const uint8_t* src, void* out, long long ldo, long long mstride, int rows,
                                  int cols, int matrices, bool gated, cudaStream_t s) {
  const dim3 grid((unsigned)((cols + 127) / 128 * (long long)((rows + 15) / 16)), matrices);
  const int vec = vec_ok(out, ldo, mstride, elem_bytes(type)), g = gated;
  switch (type) {
    case kF32: return launch_pdl(mx4_dequantize_kernel<kF32>, grid, 256, 0, s, src, (float*)out, ldo, mstride, rows, cols, g, vec);
    case kF16: return launch_pdl(mx4_dequantize_kernel<kF16>, grid, 256, 0, s, src, (__half*)out, ldo, mstride, rows, cols, g, vec);
    default: return launch_pdl(mx4_dequantize_kernel<kBF16>, grid, 256, 0, s, src, (__nv_bfloat16*)out, ldo, mstride, rows, cols, g, vec);
  }
}

cudaError_t launch_mx4_gather(int type, const void* x, long long ldx, const int32_t* pos, uint8_t* dst, int T, int H,
                              int K, cudaStream_t s) {
  const int spans = (mx_blocks(H) + 31) / 32;
  const dim3 grid((unsigned)(((long long)T * spans + 7) / 8));
  const int vec = vec_ok(x, ldx, 0, elem_bytes(type));
  switch (type) {
    case kF32: return launch_pdl(mx4_gather_kernel<kF32>, grid, 256, 0, s, (const float*)x, ldx, pos, dst, T, H, K, vec);
    case kF16: return launch_pdl(mx4_gather_kernel<kF16>, grid, 256, 0, s, (const __half*)x, ldx, pos, dst, T, H, K, vec);
    default: return launch_pdl(mx4_gather_kernel<kBF16>, grid, 256, 0, s, (const __nv_bfloat16*)x, ldx, pos, dst, T, H, K, vec);
  }
}

}  // namespace mrml
