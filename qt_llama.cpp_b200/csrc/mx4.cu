// mx4.cu — quantisation to and from the MXFP4 matrix format (mx4.cuh).
//
// All of these kernels are bound by memory: they read each value once and
// write 17/32 byte for it (dequantisation: the other way round).
#include "../../include/mrml_moe.h"
#include "mx4.cuh"
#include "kernels.h"

namespace mrml {

namespace {

// GGUF blocks of 32 values as source (quant.rs:135-190): Q4_0 holds elements
// 0..15 in the low nibbles and 16..31 in the high ones, offset by 8.
__device__ __forceinline__ void load_gguf_block(const uint8_t* blk, bool q4, MxPart<kF32, 32>& part) {
  float v[32];
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
  memcpy(part.w, v, sizeof(v));
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
// written whole.  128 bf16 matrices of 1408 x 2816 (1285 MB) take 187 us, 6.9
// TB/s.  TYPE < 0: GGUF blocks, read in their two-byte units (18 and 34 bytes,
// so no wider load is aligned): Q4_0 (555 MB) 259 us, 2.1 TB/s, Q8_0 (809 MB) 265
// us, 3.1 TB/s, once per model.
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
  constexpr int kPart = TYPE < 0 ? kF32 : TYPE;
  MxPart<kPart, 32> v;
  if (row < rows && b * 32 < cols) {
    if constexpr (TYPE >= 0) {
      using T = typename Elem<TYPE>::T;
      load_block<TYPE>(static_cast<const T*>(src) + m * mstride + row * ldx, b, cols, vec != 0, v);
    } else {
      load_gguf_block(static_cast<const uint8_t*>(src) + (((size_t)m * rows + row) * (cols / 32) + b) * (q4 ? 18 : 34),
                      q4 != 0, v);
    }
  } else {
    v.zero();
  }
  uint4 q;
  const uint32_t s = quantize_block(v, q);
  store_block(dst + ((size_t)m * tiles + tile) * mx_tile_bytes(nb), nb, r, b, q, s, b < nb);
}

// Both directions in one read: a CTA stages 64 (f32) or 128 rows x 128 columns
// in shared memory; a thread then quantises blocks along a row, and blocks along a
// column (a block of the transposed matrix) together with a partner: each of
// the two reads half the rows of two adjacent columns, so that 16-bit values
// come in whole words, they share the columns' maxima, and half a block of
// codes changes hands.  Both outputs are written in whole 128-byte lines.
// 22528 x 2816 bf16 (194 MB) 43 us, 4.5 TB/s, no unit at its limit: instruction
// issue at 58 %, the load/store data pipe at 60 (33 of them shared memory), DRAM
// at 44, with 46 % of the warps that an SM could hold.
constexpr int kBothCols = 128;
template <int TYPE>
constexpr int kBothRows = TYPE == kF32 ? 64 : 128;  // of 48 KB of shared memory
template <int TYPE>
__global__ void __launch_bounds__(256) mx4_quantize_both_kernel(const typename Elem<TYPE>::T* __restrict__ src,
                                                                long long ldx, uint8_t* __restrict__ dst,
                                                                uint8_t* __restrict__ dst_t, int rows, int cols,
                                                                int vec) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  constexpr int kRows = kBothRows<TYPE>, kIter = kRows / 64;
  // Rows are shifted by eight banks each.  Along a row, lanes of the upper two
  // blocks read their 16-byte pieces with neighbours exchanged; along the
  // columns the two lanes of a pair take rows 4j, 4j + 1 and 4j + 2, 4j + 3:
  // both without bank conflicts for 16-bit values.
  constexpr int kPitch = kBothCols + 32 / sizeof(T);
  __shared__ __align__(16) T sm[kRows * kPitch];
  pdl_wait();
  pdl_trigger();
  const int nx = (cols + kMxRows - 1) / kMxRows * (kMxRows / kBothCols);  // every row of dst_t's tiles
  const int r0 = blockIdx.x / nx * kRows, c0 = blockIdx.x % nx * kBothCols;
  constexpr int kVecs = kBothCols / E::kVec, kLoads = kRows * kVecs / 256;
  const int lr = threadIdx.x / kVecs, lc = (threadIdx.x % kVecs) * E::kVec;
  {
    const T* p = src + (r0 + lr) * ldx + c0 + lc;
    uint4 u[kLoads];
    if (vec && r0 + kRows <= rows && c0 + kBothCols <= cols) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) u[i] = __ldg(reinterpret_cast<const uint4*>(p + i * (256 / kVecs) * ldx));
    } else {
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const T* q = p + i * (256 / kVecs) * ldx;
        T t[E::kVec];
#pragma unroll
        for (int j = 0; j < E::kVec; ++j)
          t[j] = r0 + lr + i * (256 / kVecs) < rows && c0 + lc + j < cols ? q[j] : E::put(0.f);
        memcpy(&u[i], t, 16);
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      *reinterpret_cast<uint4*>(&sm[(lr + i * (256 / kVecs)) * kPitch + lc]) = u[i];
  }
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  {
    const int r = warp * 8 + (lane >> 2), b = lane & 3, nb = mx_blocks(cols), bg = (c0 >> 5) + b;
    uint8_t* tile = dst + (size_t)(r0 / kMxRows) * mx_tile_bytes(nb);
    const int rt = r0 % kMxRows + r, n = min(kMxChunk, nb - bg / kMxChunk * kMxChunk);
    uint8_t* qp = tile + mx_code_offset(nb, rt, bg);
    uint8_t* sp = tile + mx_scale_offset(rt, bg);
#pragma unroll
    for (int i = 0; i < kIter; ++i) {  // 64 rows further: 8 row groups, two words of scales
      MxPart<TYPE, 32> v;
      const int swap = (b >> 1) * E::kVec;
#pragma unroll
      for (int k = 0; k < 32 / E::kVec; ++k)
        memcpy(v.w + 4 * k, __builtin_assume_aligned(&sm[(r + 64 * i) * kPitch + b * 32 + (k * E::kVec ^ swap)], 16), 16);
      uint4 q;
      uint32_t w = quantize_block(v, q) << (8 * b);
      if (swap) {  // 8 codes per 16-byte piece of 16-bit values, 4 of f32
        if constexpr (TYPE == kF32) {
          q = make_uint4(__byte_perm(q.x, 0, 0x1032), __byte_perm(q.y, 0, 0x1032), __byte_perm(q.z, 0, 0x1032),
                         __byte_perm(q.w, 0, 0x1032));
        } else {
          q = make_uint4(q.y, q.x, q.w, q.z);
        }
      }
      w |= __shfl_xor_sync(0xffffffffu, w, 1);
      w |= __shfl_xor_sync(0xffffffffu, w, 2);
      if (bg < nb) {
        *reinterpret_cast<uint4*>(qp + i * 8 * (n * 128)) = q;
        if (b == 0) *reinterpret_cast<uint32_t*>(sp + 8 * i) = w;
      }
    }
  }
  {
    // 32 columns x 1 block per warp: lanes l and l + 16 each take 16 of the
    // block's rows in columns 2l and 2l + 1
    const int half = lane >> 4, c = (warp & 3) * 32 + (lane & 15) * 2, nb = mx_blocks(rows);
    const int row = c0 + c + half, bg = (r0 >> 5) + (warp >> 2);
    const T* p = &sm[((warp >> 2) * 32 + half * 2) * kPitch + c];
    uint8_t* tile = dst_t + (size_t)(row / kMxRows) * mx_tile_bytes(nb);
    uint8_t* qp = tile + mx_code_offset(nb, row % kMxRows, bg);
    uint8_t* sp = tile + mx_scale_offset(row % kMxRows, bg);
#pragma unroll
    for (int i = 0; i < kIter; ++i) {  // two blocks further, in the same chunk (r0 is a multiple of 128 then)
      MxPart<TYPE, 16> x, y;
      if constexpr (TYPE == kF32) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          uint2 t;
          memcpy(&t, __builtin_assume_aligned(p + (64 * i + j / 2 * 4 + j % 2) * kPitch, 8), 8);
          x.w[j] = t.x, y.w[j] = t.y;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t t0, t1;
          memcpy(&t0, __builtin_assume_aligned(p + (64 * i + 4 * j) * kPitch, 4), 4);
          memcpy(&t1, __builtin_assume_aligned(p + (64 * i + 4 * j + 1) * kPitch, 4), 4);
          x.w[j] = __byte_perm(t0, t1, 0x5410);
          y.w[j] = __byte_perm(t0, t1, 0x7632);
        }
      }
      uint32_t mx = x.amax(), my = y.amax();
      mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      my = max(my, __shfl_xor_sync(0xffffffffu, my, 16));
      float ix, iy;
      const uint32_t sx = mx_scale(mx, ix), sy = mx_scale(my, iy);
      uint32_t qx[2], qy[2];
      x.codes(ix, qx);
      y.codes(iy, qy);
      // the lower lane ends with all of column 2l, the upper with 2l + 1; a
      // byte holds two rows, so the lanes' bytes alternate
      const uint32_t g0 = __shfl_xor_sync(0xffffffffu, half ? qx[0] : qy[0], 16);
      const uint32_t g1 = __shfl_xor_sync(0xffffffffu, half ? qx[1] : qy[1], 16);
      const uint32_t l0 = half ? g0 : qx[0], l1 = half ? g1 : qx[1], u0 = half ? qy[0] : g0, u1 = half ? qy[1] : g1;
      if (bg + 2 * i < nb) {
        *reinterpret_cast<uint4*>(qp + 256 * i) = make_uint4(__byte_perm(l0, u0, 0x5140), __byte_perm(l0, u0, 0x7362),
                                                             __byte_perm(l1, u1, 0x5140), __byte_perm(l1, u1, 0x7362));
        sp[2 * i] = (uint8_t)(half ? sy : sx);
      }
    }
  }
}

// Two E2M1 codes (a byte) as f32.
__device__ __forceinline__ float2 e2m1_pair(uint32_t byte) {
  uint32_t h;
  asm("{\n\t.reg .b8 a;\n\tcvt.u8.u32 a, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}" : "=r"(h) : "r"(byte));
  __half2 v;
  memcpy(&v, &h, 4);
  return __half22float2(v);
}

// A warp takes 8 rows x 128 columns of a tile: lanes side by side write one
// 16-byte vector each of a row, and the addresses of the first rows serve all
// eight.  (The codes of the 8 rows are four lines, read once and then from
// L1.)  22528 x 2816 to bf16 (161 MB): 26 us, 6.1 TB/s.
template <int TYPE>
__global__ void __launch_bounds__(256) mx4_dequantize_kernel(const uint8_t* __restrict__ src,
                                                             typename Elem<TYPE>::T* __restrict__ dst, long long ldo,
                                                             long long mstride, int rows, int cols, int gated,
                                                             int vec) {
  using E = Elem<TYPE>;
  constexpr int V = E::kVec, kLanes = 128 / V, kStep = 32 / kLanes;  // lanes per row, rows at a time
  pdl_wait();  // no early start for the next launch, which may read dst without waiting (kernels.h)
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int nx = (cols + 127) / 128, m = blockIdx.y;
  const int tiles = (rows + kMxRows - 1) / kMxRows, tile = (int)(blockIdx.x / nx) >> 1;
  const int g = ((int)(blockIdx.x / nx) & 1) * 8 + warp;  // row group of the tile
  const int c = (int)(blockIdx.x % nx) * 128 + (lane % kLanes) * V, b = c >> 5;
  if (c >= cols) return;
  const int nb = mx_blocks(cols), r0 = g * 8 + lane / kLanes;
  const uint8_t* t = src + ((size_t)m * tiles + tile) * mx_tile_bytes(nb);
  const uint8_t* qp = t + mx_code_offset(nb, r0, b) + (c & 31) / 2;
  const uint8_t* sp = t + mx_scale_offset(r0, b);
  int row, limit;  // of the first row, and where the rows end
  if (gated) {
    const int I = rows >> 1;
    row = tile * 64 + (r0 & 63) + (r0 < 64 ? 0 : I);
    limit = r0 < 64 ? I : rows;
  } else {
    row = tile * kMxRows + r0;
    limit = rows;
  }
  typename E::T* o = dst + m * mstride + row * ldo + c;
#pragma unroll
  for (int i = 0; i < 8; i += kStep) {
    if (row + i >= limit) break;
    uint32_t q;
    if constexpr (V == 8) q = __ldg(reinterpret_cast<const uint32_t*>(qp + 16 * i));
    else q = __ldg(reinterpret_cast<const uint16_t*>(qp + 16 * i));
    const uint32_t s = __ldg(sp + 16 * i);
    // 2^(s - 127); s = 0 is the subnormal 2^-127, s = 255 NaN
    const float scale = s == 255u ? __uint_as_float(0x7fffffffu) : __uint_as_float(s ? s << 23 : 0x00400000u);
    float v[V];
#pragma unroll
    for (int j = 0; j < V / 2; ++j) {
      const float2 f = e2m1_pair((q >> (8 * j)) & 0xffu);
      v[2 * j] = f.x * scale, v[2 * j + 1] = f.y * scale;
    }
    if (vec && c + V <= cols) {
      *reinterpret_cast<uint4*>(o) = E::pack(v);
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (c + j < cols) o[j] = E::put(v[j]);
    }
    o += kStep * ldo;
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
  MxPart<TYPE, 32> v;
  if (b * 32 < H) load_block<TYPE>(x + t * ldx, b, H, vec != 0, v);
  else v.zero();
  uint4 q;
  const uint32_t s = quantize_block(v, q);
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

// The same in two steps for large batches, where the 16-byte stores above,
// each half a 32-byte sector in a line of eight different tokens, are what
// bounds: the tokens quantised once, row by row (codes [T][nb][16], scales
// [T][nb rounded up to 4]), then whole lines gathered.  65536 pairs of 2816: 78
// us in one step, 10 + 30 in two; 512 pairs: 5.4 us in one.
__host__ __device__ inline int flat_scales(int nb) { return (nb + 3) & ~3; }

template <int TYPE>
__global__ void __launch_bounds__(256) mx4_quantize_flat_kernel(const typename Elem<TYPE>::T* __restrict__ x,
                                                                long long ldx, uint4* __restrict__ codes,
                                                                uint8_t* __restrict__ scales, int T, int H, int vec) {
  pdl_wait();
  pdl_trigger();
  const int nb = mx_blocks(H), np = flat_scales(nb);
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int t = (int)(i / np), b = (int)(i % np);
  if (t >= T) return;
  MxPart<TYPE, 32> v;
  if (b * 32 < H) load_block<TYPE>(x + t * ldx, b, H, vec != 0, v);
  else v.zero();
  uint4 q;
  scales[i] = (uint8_t)quantize_block(v, q);
  if (b < nb) codes[(size_t)t * nb + b] = q;
}

// A warp takes 8 positions (a row group): lane = (row, block of four).
__global__ void __launch_bounds__(256) mx4_gather_flat_kernel(const uint4* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales,
                                                              const int32_t* __restrict__ pair,
                                                              const int32_t* __restrict__ end,
                                                              uint8_t* __restrict__ dst, int H, int K, int n_rows) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31, j = lane & 3;
  const int row = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 8 + (lane >> 2);
  if (row >= min(n_rows, __ldg(end))) return;
  const int p = __ldg(pair + row);
  if (p < 0) return;
  const int nb = mx_blocks(H), r = row % kMxRows;
  const uint4* q = codes + (size_t)(p / K) * nb;
  const uint32_t* s = reinterpret_cast<const uint32_t*>(scales + (size_t)(p / K) * flat_scales(nb));
  uint8_t* tile = dst + (size_t)(row / kMxRows) * mx_tile_bytes(nb);
#pragma unroll 4
  for (int b = j; b < nb; b += 4) *reinterpret_cast<uint4*>(tile + mx_code_offset(nb, r, b)) = __ldg(q + b);
  for (int g = j; g < (nb + 3) / 4; g += 4)
    *reinterpret_cast<uint32_t*>(tile + mx_scale_offset(r, 4 * g)) = __ldg(s + g);
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
  const dim3 grid((unsigned)((long long)(pc / kBothCols) * (pr / (type == kF32 ? kBothRows<kF32> : kBothRows<kBF16>))));
  const int vec = vec_ok(x, ldx, 0, elem_bytes(type));
  switch (type) {
    case kF32: return launch_pdl(mx4_quantize_both_kernel<kF32>, grid, 256, 0, s, (const float*)x, ldx, dst, dst_t, rows, cols, vec);
    case kF16: return launch_pdl(mx4_quantize_both_kernel<kF16>, grid, 256, 0, s, (const __half*)x, ldx, dst, dst_t, rows, cols, vec);
    default: return launch_pdl(mx4_quantize_both_kernel<kBF16>, grid, 256, 0, s, (const __nv_bfloat16*)x, ldx, dst, dst_t, rows, cols, vec);
  }
}

cudaError_t launch_mx4_dequantize(int type, const uint8_t* src, void* out, long long ldo, long long mstride, int rows,
                                  int cols, int matrices, bool gated, cudaStream_t s) {
  const dim3 grid((unsigned)((cols + 127) / 128 * (long long)((rows + kMxRows - 1) / kMxRows * 2)), matrices);
  const int vec = vec_ok(out, ldo, mstride, elem_bytes(type)), g = gated;
  switch (type) {
    case kF32: return launch_pdl(mx4_dequantize_kernel<kF32>, grid, 256, 0, s, src, (float*)out, ldo, mstride, rows, cols, g, vec);
    case kF16: return launch_pdl(mx4_dequantize_kernel<kF16>, grid, 256, 0, s, src, (__half*)out, ldo, mstride, rows, cols, g, vec);
    default: return launch_pdl(mx4_dequantize_kernel<kBF16>, grid, 256, 0, s, src, (__nv_bfloat16*)out, ldo, mstride, rows, cols, g, vec);
  }
}

// The gather runs in two steps where a token goes to several experts and the
// rows are many: from 80 million gathered values.  The expert layer (us) in one
// and in two steps, by pairs:
//   H 2816, 128 experts top-8: 24576 pairs (69 M) 240 / 242, 32768 (92 M) 298 / 290, 65536 506 / 466
//   H 8192, 64 top-8:          8192 (67 M) 211 / 220, 16384 (134 M) 368 / 349, 65536 1231 / 1060
//   H 4096, 32 top-4:          16384 (67 M) 178 / 179, 24576 (101 M) 241 / 234
//   H 1024, 16 top-2:          65536 (67 M) 261 / 264, 131072 (134 M) 512 / 505
//   H 256, 128 top-8:          131072 (34 M) 145 / 145
//   H 2816, 16 top-1:          65536 (185 M) 761 / 774, 131072 1503 / 1531
constexpr long long kGatherFlatValues = 80'000'000;

bool gather_flat(int H, int K, int T) { return K > 1 && (long long)T * K * H >= kGatherFlatValues; }

size_t mx4_flat_bytes(int H, int K, int T) {
  const int nb = mx_blocks(H);
  return gather_flat(H, K, T) ? (size_t)T * (nb * 16 + flat_scales(nb)) : 0;
}

namespace {
template <int TYPE>
cudaError_t gather_as(const void* x, long long ldx, const int32_t* pos, const int32_t* pair, const int32_t* end,
                      uint8_t* dst, uint8_t* flat, int T, int H, int K, int n_rows, cudaStream_t s) {
  using E = typename Elem<TYPE>::T;
  const int vec = vec_ok(x, ldx, 0, sizeof(E)), nb = mx_blocks(H);
  if (!gather_flat(H, K, T)) {
    const dim3 grid((unsigned)(((long long)T * ((nb + 31) / 32) + 7) / 8));
    return launch_pdl(mx4_gather_kernel<TYPE>, grid, 256, 0, s, (const E*)x, ldx, pos, dst, T, H, K, vec);
  }
  uint4* codes = reinterpret_cast<uint4*>(flat);
  uint8_t* scales = flat + (size_t)T * nb * 16;
  const dim3 grid((unsigned)(((long long)T * flat_scales(nb) + 255) / 256));
  const cudaError_t st = launch_pdl(mx4_quantize_flat_kernel<TYPE>, grid, 256, 0, s, (const E*)x, ldx, codes, scales, T, H, vec);
  if (st != cudaSuccess) return st;
  return launch_pdl(mx4_gather_flat_kernel, dim3((n_rows + 63) / 64), 256, 0, s, (const uint4*)codes, (const uint8_t*)scales, pair, end, dst, H, K, n_rows);
}
}  // namespace

cudaError_t launch_mx4_gather(int type, const void* x, long long ldx, const int32_t* pos, const int32_t* pair,
                              const int32_t* end, uint8_t* dst, uint8_t* flat, int T, int H, int K, int n_rows,
                              cudaStream_t s) {
  switch (type) {
    case kF32: return gather_as<kF32>(x, ldx, pos, pair, end, dst, flat, T, H, K, n_rows, s);
    case kF16: return gather_as<kF16>(x, ldx, pos, pair, end, dst, flat, T, H, K, n_rows, s);
    default: return gather_as<kBF16>(x, ldx, pos, pair, end, dst, flat, T, H, K, n_rows, s);
  }
}

}  // namespace mrml
