// permute.cu — (token, slot) pairs sorted by expert, the tokens' rows gathered
// in that order and brought back with weights, and the gradients of both.
//
//   sort       pos[p] = offsets[e] + #{q < p : ids[q] = e} for e = ids[p]
//   permute    rows[r] = x[pair[r] / K]
//   its gradient and unpermute
//              out[t] = sum_k w[t,k] rows[pos[t,k]]   (w = 1 for the gradient)
//   unpermute's gradients
//              drows[pos[t,k]] = w[t,k] dout[t],  dw[t,k] = <dout[t], rows[pos[t,k]]>
// Sums run in f32 in slot order and are rounded once.
//
// The kernels that write rows or tokens do not let the next launch start early:
// a caller may use any of them as a matrix that a later kernel reads without
// waiting (kernels.h).
#include "../../include/mrml_moe.h"
#include "kernels.h"
#include "mx4.cuh"

namespace mrml {

namespace {

// -------------------------------------------------------------------- sort
// Counting sort, stable by construction: a warp owns consecutive pairs, ranks
// those of one expert with a warp match, and starts from the counts of the
// warps (and chunks) before it.  No atomic decides an order.  Bound by latency:
// 64 pairs 2.8 us, 512 pairs 4.1 us in one CTA; 65536 pairs in two launches 7.1
// us, whose chunks each sum all chunks' counts instead of waiting for a scan in
// between.
struct SortArgs {
  const int32_t* ids;
  int32_t *offsets, *counts, *pos, *pair;
  int32_t* chunk_cnt;  // [chunks][E], more than one chunk only
  int* err;
  int n_pairs, E, align, n_rows, chunk;
};

// Every row starts without a pair.
__device__ __forceinline__ void clear_pairs(const SortArgs& a) {
  if (!a.pair) return;
  const int stride = gridDim.x * blockDim.x;
  int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (((uintptr_t)a.pair & 15) == 0) {
    for (; r < a.n_rows / 4; r += stride) reinterpret_cast<int4*>(a.pair)[r] = make_int4(-1, -1, -1, -1);
    r = (a.n_rows & ~3) + blockIdx.x * blockDim.x + threadIdx.x;
  }
  for (; r < a.n_rows; r += stride) a.pair[r] = -1;
}

__global__ void __launch_bounds__(1024) sort_count_kernel(SortArgs a) {
  __shared__ int cnt[kMaxExperts];
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) cnt[e] = 0;
  pdl_wait();
  pdl_trigger();
  clear_pairs(a);
  __syncthreads();
  const int p0 = blockIdx.x * a.chunk, p1 = min(a.n_pairs, p0 + a.chunk);
  for (int p = p0 + threadIdx.x; p < p1; p += blockDim.x) {
    const int e = a.ids[p];
    if ((unsigned)e < (unsigned)a.E) atomicAdd(&cnt[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) a.chunk_cnt[(size_t)blockIdx.x * a.E + e] = cnt[e];
}

template <int ITEMS>
__global__ void __launch_bounds__(1024) sort_place_kernel(SortArgs a) {
  extern __shared__ int sm[];
  const int nw = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, E = a.E;
  int* wcnt = sm;              // [nw][E] pairs of this chunk's earlier warps
  int* tot = wcnt + nw * E;    // [E] pairs of all chunks
  int* before = tot + E;       // [E] pairs of earlier chunks
  int* off = before + E;       // [E + 1]
  for (int i = threadIdx.x; i < nw * E + 2 * E; i += blockDim.x) sm[i] = 0;
  pdl_wait();
  pdl_trigger();
  if (gridDim.x == 1) clear_pairs(a);
  __syncthreads();
  int e[ITEMS], rank[ITEMS];
  const int p0 = blockIdx.x * a.chunk + warp * 32 * ITEMS;
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int p = p0 + i * 32 + lane;
    e[i] = p < a.n_pairs ? a.ids[p] : -1;
    if (e[i] >= E) {
      set_error(a.err, kDevBadExpert);
      e[i] = -1;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned same = __match_any_sync(0xffffffffu, e[i]);
    const int at = __popc(same & ((1u << lane) - 1));
    if (e[i] >= 0) rank[i] = wcnt[warp * E + e[i]] + at;
    __syncwarp();
    if (e[i] >= 0 && at == 0) wcnt[warp * E + e[i]] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int x = threadIdx.x; x < E; x += blockDim.x) {
    int s = 0;
    for (int w = 0; w < nw; ++w) {
      const int c = wcnt[w * E + x];
      wcnt[w * E + x] = s;
      s += c;
    }
    if (gridDim.x == 1) tot[x] = s;
  }
  if (gridDim.x > 1) {
    // this chunk's start and the totals, from every chunk's counts: a thread
    // sums one expert over every (threads / E)-th chunk
    const int x = threadIdx.x % E, step = blockDim.x / E, chunks = gridDim.x;
    if ((int)threadIdx.x < step * E) {
      int all = 0, mine = 0;
#pragma unroll 8
      for (int c = threadIdx.x / E; c < chunks; c += step) {
        const int n = a.chunk_cnt[(size_t)c * E + x];
        all += n;
        if (c < (int)blockIdx.x) mine += n;
      }
      atomicAdd(&tot[x], all);
      atomicAdd(&before[x], mine);
    }
  }
  __syncthreads();
  for (int x = threadIdx.x; x < E; x += blockDim.x) off[x] = (tot[x] + a.align - 1) / a.align * a.align;
  __syncthreads();
  if (warp == 0) {  // starts: each lane scans the rows of E / 32 experts
    constexpr int kPer = kMaxExperts / 32;
    int c[kPer], s = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int x = lane * kPer + i;
      c[i] = s;
      if (x < E) s += off[x];
    }
    int up = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += y;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane * kPer + i < E) off[lane * kPer + i] = up - s + c[i];
    if (lane == 31) off[E] = up;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int p = p0 + i * 32 + lane;
    if (p < a.n_pairs) {
      int at = -1;
      if (e[i] >= 0) {
        at = off[e[i]] + before[e[i]] + wcnt[warp * E + e[i]] + rank[i];
        if (a.pair) a.pair[at] = p;
      }
      a.pos[p] = at;
    }
  }
  if (blockIdx.x == 0) {
    for (int x = threadIdx.x; x < E; x += blockDim.x) a.counts[x] = tot[x];
    for (int x = threadIdx.x; x <= E; x += blockDim.x) a.offsets[x] = off[x];
  }
}

// ----------------------------------------------------------------- permute
// A warp per row, the row's sorted place being where it writes: whole lines in
// order, while the tokens are read from L2 after their first use.  VEC: 16-byte
// vectors (rows and strides aligned).  Bound by memory, seven eighths of it
// writes: 65536 rows of 2816 bf16 (415 MB) 77 us, 5.4 TB/s; the streaming hint
// on the stores is worth 7 % (85 us without), one on the loads nothing.  Rows that
// are not aligned go element by element: of 2815 bf16 172 us, f32 297 (194).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) permute_kernel(const T* __restrict__ x, long long ldx,
                                                      const int32_t* __restrict__ pair, T* __restrict__ rows, int H,
                                                      int K, int n_rows) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (r >= n_rows) return;
  const int p = pair[r];
  const T* src = x + (p >= 0 ? (long long)(p / K) : 0) * ldx;
  T* dst = rows + (size_t)r * H;
  if constexpr (VEC) {
    const int nv = H * (int)sizeof(T) / 16;
    const uint4* s = reinterpret_cast<const uint4*>(src);
    uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll 4
    for (int i = lane; i < nv; i += 32) __stcs(d + i, p >= 0 ? __ldg(s + i) : make_uint4(0, 0, 0, 0));
  } else {
#pragma unroll 4
    for (int i = lane; i < H; i += 32) {
      T v;
      if (p >= 0) v = src[i];
      else memset(&v, 0, sizeof(T));
      dst[i] = v;
    }
  }
}

// --------------------------------------------------------------- unpermute
// A CTA takes a token, or one of several column ranges of it (gridDim.y); a
// thread sums the K rows in two vectors of columns at a time, all of whose
// loads (16 for 8 slots) it issues before it needs one.  The rows' places and
// weights are read once for all columns.  Bound by memory: 65536 f32 rows of
// 2816 into 8192 bf16 tokens (785 MB) 120 us, 6.5 TB/s; bf16 rows (415 MB) 70 us,
// 5.9 TB/s (one vector per thread and CTA: 129 and 75 us); unaligned rows of
// 2815, element by element, bf16 315 us, f32 138 (122).  The weight of slot k is probs[t,k]
// (1 without probs) times scale[ids[t,k]] (with scale).
template <int TYPE_IN, int TYPE, bool VEC>
__global__ void __launch_bounds__(128) unpermute_kernel(const typename Elem<TYPE_IN>::T* __restrict__ rows,
                                                        const int32_t* __restrict__ pos,
                                                        const float* __restrict__ probs,
                                                        const int32_t* __restrict__ ids,
                                                        const float* __restrict__ scale,
                                                        typename Elem<TYPE>::T* __restrict__ out, long long ldo,
                                                        int H, int K) {
  using EI = Elem<TYPE_IN>;
  using E = Elem<TYPE>;
  constexpr int V = VEC ? EI::kVec : 1;  // values per vector: one 16-byte load of a row
  constexpr int S = 8;                   // slots at a time
  pdl_wait();
  const long long t = blockIdx.x;
  int at[S];
  float w[S];
  auto slots = [&](int k0) {
#pragma unroll
    for (int j = 0; j < S; ++j) {
      at[j] = -1;
      if (k0 + j < K) at[j] = __ldg(pos + t * K + k0 + j);
      w[j] = k0 + j < K && probs ? __ldg(probs + t * K + k0 + j) : 1.f;
      if (scale && at[j] >= 0) w[j] *= __ldg(scale + __ldg(ids + t * K + k0 + j));
    }
  };
  slots(0);
  const int step = gridDim.y * 128 * V;
  for (int c = (blockIdx.y * 128 + threadIdx.x) * V; c < H; c += 2 * step) {
    const bool second = c + step < H;
    float acc[2][V];
#pragma unroll
    for (int i = 0; i < V; ++i) acc[0][i] = acc[1][i] = 0.f;
    for (int k0 = 0; k0 < K; k0 += S) {
      if (k0 > 0 || K > S) slots(k0);
      uint4 u[2][S];
#pragma unroll
      for (int j = 0; j < S; ++j) {
        if (at[j] < 0) continue;
        const typename EI::T* p = rows + (size_t)at[j] * H + c;
        if constexpr (VEC) {
          u[0][j] = __ldg(reinterpret_cast<const uint4*>(p));
          if (second) u[1][j] = __ldg(reinterpret_cast<const uint4*>(p + step));
        } else {
          u[0][j].x = __float_as_uint(EI::get(p[0]));
          if (second) u[1][j].x = __float_as_uint(EI::get(p[step]));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && !second) break;
#pragma unroll
        for (int j = 0; j < S; ++j) {
          if (at[j] < 0) continue;
          float v[V];
          if constexpr (VEC) EI::unpack(u[h][j], v);
          else v[0] = __uint_as_float(u[h][j].x);
#pragma unroll
          for (int i = 0; i < V; ++i) acc[h][i] = fmaf(w[j], v[i], acc[h][i]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && !second) break;
      typename E::T* o = out + t * ldo + c + h * step;
      typename E::T r[V];
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = E::put(acc[h][i]);
      memcpy(__builtin_assume_aligned(o, V * sizeof(r[0])), r, sizeof(r));
    }
  }
}

// ------------------------------------------------------- unpermute gradient
// A warp per pair: reads the pair's row and the token's gradient once, writes
// the row's gradient and the weight's.  The K warps of a token share its
// gradient row through L1.  Bound by memory: 65536 bf16 rows of 2816 (784 MB)
// 126 us, 6.2 TB/s; unaligned rows of 2815 218 us, f32 340 (247).  The warp also clears the row of its own index
// when no pair takes it (there are at least as many rows as pairs).
template <int TYPE, bool VEC>
__global__ void __launch_bounds__(256) unpermute_grad_kernel(const typename Elem<TYPE>::T* __restrict__ dout,
                                                             long long ldd,
                                                             const typename Elem<TYPE>::T* __restrict__ rows,
                                                             const int32_t* __restrict__ pos,
                                                             const int32_t* __restrict__ pair,
                                                             const float* __restrict__ probs,
                                                             typename Elem<TYPE>::T* __restrict__ drows,
                                                             float* __restrict__ dprobs, int H, int K, int n_pairs,
                                                             int n_rows) {
  using E = Elem<TYPE>;
  using T = typename E::T;
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int i0 = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int nv = H / E::kVec;
  if (i0 < n_pairs) {
    const int at = pos[i0];
    const float w = probs ? probs[i0] : 1.f;
    const T* g = dout + (long long)(i0 / K) * ldd;
    float dot = 0.f;
    if (at >= 0) {
      const T* y = rows + (size_t)at * H;
      T* d = drows ? drows + (size_t)at * H : nullptr;
      if constexpr (VEC) {
#pragma unroll 4
        for (int i = lane; i < nv; i += 32) {
          float a[E::kVec], b[E::kVec];
          E::unpack(__ldg(reinterpret_cast<const uint4*>(g) + i), a);
          if (dprobs) {
            E::unpack(__ldg(reinterpret_cast<const uint4*>(y) + i), b);
#pragma unroll
            for (int j = 0; j < E::kVec; ++j) dot = fmaf(a[j], b[j], dot);
          }
          if (d) {
#pragma unroll
            for (int j = 0; j < E::kVec; ++j) a[j] *= w;
            reinterpret_cast<uint4*>(d)[i] = E::pack(a);
          }
        }
      } else {
#pragma unroll 4
        for (int i = lane; i < H; i += 32) {
          const float a = E::get(g[i]);
          if (dprobs) dot = fmaf(a, E::get(y[i]), dot);
          if (d) d[i] = E::put(a * w);
        }
      }
    }
    if (dprobs) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (lane == 0) dprobs[i0] = dot;
    }
  }
  if (drows && i0 < n_rows && pair[i0] < 0) {
    T* d = drows + (size_t)i0 * H;
    if constexpr (VEC) {
      for (int i = lane; i < nv; i += 32) reinterpret_cast<uint4*>(d)[i] = make_uint4(0, 0, 0, 0);
    } else {
      for (int i = lane; i < H; i += 32) d[i] = E::put(0.f);
    }
  }
}

bool rows_aligned(const void* p, long long ld, size_t s) { return ((uintptr_t)p & 15) == 0 && (size_t)ld * s % 16 == 0; }

}  // namespace

// Pairs up to which one CTA sorts, and the chunk of the larger sorts, whose two
// launches read the ids twice: 4096 pairs take 11.3 us in one CTA and 6.1 in
// chunks, 1024 pairs 5.4 in one.  Every chunk reads all chunks' counts, so many
// pairs take larger ones: chunks of 1024 and of 8192 pairs take 12.4 and 21.5 us
// for 262144 pairs, 31 and 22 for 524288, 78 and 25 for 2^20.
constexpr int kSortOne = 1024;

constexpr long long kSortSmallChunks = 3 << 17;

int sort_chunk(long long n_pairs) { return n_pairs <= kSortSmallChunks ? 1024 : 8192; }

// Never less than fewer pairs take, so that a workspace serves them too.
size_t sort_chunk_ints(long long n_pairs, int E) {
  if (n_pairs <= kSortOne) return 0;
  const int c = sort_chunk(n_pairs);
  const long long chunks = (n_pairs + c - 1) / c;
  return (size_t)(n_pairs > kSortSmallChunks ? std::max(chunks, kSortSmallChunks / 1024) : chunks) * E;
}

cudaError_t launch_sort(const int32_t* ids, int32_t* offsets, int32_t* counts, int32_t* pos, int32_t* pair, int E,
                        int n_pairs, int align, int n_rows, int32_t* chunk_cnt, int* err, cudaStream_t s) {
  SortArgs a{ids, offsets, counts, pos, pair, chunk_cnt, err, n_pairs, E, align, n_rows, 0};
  const bool one = n_pairs <= kSortOne;
  // one CTA: no more warps than pairs for them, as their counts are scanned one
  // after another (512 pairs: 4.1 us in 512 threads, 5.3 in 256 with four each)
  const int items = one ? 1 : sort_chunk(n_pairs) / 1024;
  const int threads = one ? std::max(256, (n_pairs + 255) / 256 * 256) : 1024;
  a.chunk = items * threads;
  const int grid = std::max(1, (n_pairs + a.chunk - 1) / a.chunk);
  const size_t smem = (size_t)(threads / 32 * E + 3 * E + 1) * 4;
  if (!one) {
    const cudaError_t st = launch_pdl(sort_count_kernel, dim3(grid), dim3(1024), 0, s, a);
    if (st != cudaSuccess) return st;
  }
  switch (items) {
    case 1: return launch_pdl(sort_place_kernel<1>, dim3(grid), dim3(threads), smem, s, a);
    default: return launch_pdl(sort_place_kernel<8>, dim3(grid), dim3(threads), smem, s, a);
  }
}

cudaError_t launch_permute(int type, const void* x, long long ldx, const int32_t* pair, void* rows, int H, int K,
                           int n_rows, cudaStream_t s) {
  const size_t sz = elem_bytes(type);
  const bool vec = rows_aligned(x, ldx, sz) && rows_aligned(rows, H, sz);
  const dim3 grid((n_rows + 7) / 8), block(256);
  if (sz == 4)
    return vec ? launch_pdl(permute_kernel<uint32_t, true>, grid, block, 0, s, (const uint32_t*)x, ldx, pair, (uint32_t*)rows, H, K, n_rows)
               : launch_pdl(permute_kernel<uint32_t, false>, grid, block, 0, s, (const uint32_t*)x, ldx, pair, (uint32_t*)rows, H, K, n_rows);
  return vec ? launch_pdl(permute_kernel<uint16_t, true>, grid, block, 0, s, (const uint16_t*)x, ldx, pair, (uint16_t*)rows, H, K, n_rows)
             : launch_pdl(permute_kernel<uint16_t, false>, grid, block, 0, s, (const uint16_t*)x, ldx, pair, (uint16_t*)rows, H, K, n_rows);
}

namespace {
template <int TI, int TO>
cudaError_t unpermute_as(const void* rows, const int32_t* pos, const float* probs, const int32_t* ids,
                         const float* scale, void* out, long long ldo, int H, int K, int T, cudaStream_t s) {
  using I = typename Elem<TI>::T;
  using O = typename Elem<TO>::T;
  const bool vec = rows_aligned(rows, H, sizeof(I)) && rows_aligned(out, ldo, sizeof(O));
  // Column ranges per token: enough CTAs to fill the GPU from few tokens.
  const int v = vec ? Elem<TI>::kVec : 1, most = (H + 128 * v - 1) / (128 * v);
  const int parts = std::max(1, std::min(most, 4 * tc_num_sms() / std::max(1, T)));
  const dim3 grid(T, parts), block(128);
  return vec ? launch_pdl(unpermute_kernel<TI, TO, true>, grid, block, 0, s, (const I*)rows, pos, probs, ids, scale, (O*)out, ldo, H, K)
             : launch_pdl(unpermute_kernel<TI, TO, false>, grid, block, 0, s, (const I*)rows, pos, probs, ids, scale, (O*)out, ldo, H, K);
}

template <int TYPE>
cudaError_t unpermute_grad_as(const void* dout, long long ldd, const void* rows, const int32_t* pos,
                              const int32_t* pair, const float* probs, void* drows, float* dprobs, int H, int K,
                              int n_pairs, int n_rows, cudaStream_t s) {
  using T = typename Elem<TYPE>::T;
  const bool vec = rows_aligned(dout, ldd, sizeof(T)) && (!rows || rows_aligned(rows, H, sizeof(T))) &&
                   (!drows || rows_aligned(drows, H, sizeof(T))) && (size_t)H * sizeof(T) % 16 == 0;
  const dim3 grid((std::max(n_pairs, drows ? n_rows : 0) + 7) / 8), block(256);
  return vec ? launch_pdl(unpermute_grad_kernel<TYPE, true>, grid, block, 0, s, (const T*)dout, ldd, (const T*)rows, pos, pair, probs, (T*)drows, dprobs, H, K, n_pairs, n_rows)
             : launch_pdl(unpermute_grad_kernel<TYPE, false>, grid, block, 0, s, (const T*)dout, ldd, (const T*)rows, pos, pair, probs, (T*)drows, dprobs, H, K, n_pairs, n_rows);
}
}  // namespace

cudaError_t launch_unpermute(int type, const void* rows, const int32_t* pos, const float* probs, void* out,
                             long long ldo, int H, int K, int T, cudaStream_t s) {
  switch (type) {
    case kF32: return unpermute_as<kF32, kF32>(rows, pos, probs, nullptr, nullptr, out, ldo, H, K, T, s);
    case kF16: return unpermute_as<kF16, kF16>(rows, pos, probs, nullptr, nullptr, out, ldo, H, K, T, s);
    default: return unpermute_as<kBF16, kBF16>(rows, pos, probs, nullptr, nullptr, out, ldo, H, K, T, s);
  }
}

cudaError_t launch_combine_rows(int type, const float* rows, const int32_t* pos, const float* probs,
                                const int32_t* ids, const float* scale, void* out, long long ldo, int H, int K, int T,
                                cudaStream_t s) {
  switch (type) {
    case kF32: return unpermute_as<kF32, kF32>(rows, pos, probs, ids, scale, out, ldo, H, K, T, s);
    case kF16: return unpermute_as<kF32, kF16>(rows, pos, probs, ids, scale, out, ldo, H, K, T, s);
    default: return unpermute_as<kF32, kBF16>(rows, pos, probs, ids, scale, out, ldo, H, K, T, s);
  }
}

cudaError_t launch_unpermute_grad(int type, const void* dout, long long ldd, const void* rows, const int32_t* pos,
                                  const int32_t* pair, const float* probs, void* drows, float* dprobs, int H, int K,
                                  int T, int n_rows, cudaStream_t s) {
  switch (type) {
    case kF32: return unpermute_grad_as<kF32>(dout, ldd, rows, pos, pair, probs, drows, dprobs, H, K, T * K, n_rows, s);
    case kF16: return unpermute_grad_as<kF16>(dout, ldd, rows, pos, pair, probs, drows, dprobs, H, K, T * K, n_rows, s);
    default: return unpermute_grad_as<kBF16>(dout, ldd, rows, pos, pair, probs, drows, dprobs, H, K, T * K, n_rows, s);
  }
}

}  // namespace mrml
