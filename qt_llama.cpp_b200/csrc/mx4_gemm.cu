// mx4_gemm.cu — products of MXFP4 matrices on the 5th-generation tensor cores.
//
//   out[t][n] = sum_b 2^(ea[t,b] + eb[n,b]) sum_i a[t,32b+i] w[n,32b+i]
//
// tcgen05.mma kind::mxf4 multiplies E2M1 codes, applies both blocks' scales
// and accumulates in f32 in tensor memory: a product of two codes is exact,
// and so is its scaling, so the only roundings are the f32 additions.
//
// The weights are the instruction's A operand (128 rows, the only M of one
// CTA for this kind) and the tokens its B operand (N = the tokens of the tile
// rounded up to 16), so a decode step with a handful of tokens per expert
// wastes tensor time (which it has) instead of memory traffic (which bounds
// it), and the same kernel serves prompts with N = 128.
//
// A work unit is (expert, 128 weight rows, 128 token rows).  One persistent
// CTA per SM takes units in turn:
//   warp 0     producer: one bulk copy per operand and K chunk (the matrix
//              format is the shared-memory operand layout, mx4.cuh)
//   warp 1     TMEM allocation; lane 0 copies the chunk's scales to tensor
//              memory and issues the MMAs
//   warps 4-11 epilogue, on the other of two accumulators
// Scales live in tensor memory per shared-memory stage, so a stage's scales
// are overwritten only after the MMAs that read them have completed.
// Every wait is bounded; on a timeout the CTA records the error, drains its
// copies and MMAs (bounded again), frees its TMEM and returns.
#include "../../include/mrml_moe.h"
#include "kernels.h"
#include "mx4.cuh"
#include "pipe.cuh"

namespace mrml {
namespace mx {

using tc::fence_after;
using tc::fence_before;
using tc::mbar_arrive;
using tc::mma_commit;
using tc::tmem_wait_ld;
using tc::wait_bar;

constexpr int kStages = 5;
constexpr int kStageBytes = 2 * kMxChunkBytes;
constexpr int kThreads = 384;
constexpr int kExPitch = 33;                          // f32 per row of the GeGLU exchange
constexpr int kExBytes = 2 * kMxRows * kExPitch * 4;  // two groups' 128 rows x 32 tokens
constexpr uint32_t kAcc0 = 0, kAccCols = 128;       // two accumulators of 128 columns
constexpr uint32_t kSf0 = 256, kSfCols = 16;        // scales: 8 + 8 columns per stage

struct Params {
  const uint8_t* w;        // weight tiles [E][w_tiles]
  const uint8_t* x;        // token tiles
  const int32_t* offsets;  // [E + 1] first token row per expert, multiples of 128; null: one matrix of n_tokens rows
  const int32_t* counts;   // [E] tokens per expert
  int E, n_tokens, w_tiles, nb;
  int n_out;               // outputs per token: weight rows, or I for the gated product
  void* out;               // [token row][ldo]
  long long ldo;
  uint8_t* act;            // gated: MXFP4 [token row][n_out]
  int* err;
};

struct __align__(8) Bars {
  uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], drain;
  uint32_t tmem_base;
  int abort;
  int first[kMaxExperts + 1];  // token tiles of earlier experts
  int row0[kMaxExperts], count[kMaxExperts];  // each expert's first row and rows
};
constexpr int kBarBytes = 4096;
static_assert(sizeof(Bars) <= kBarBytes, "the barrier block must fit its part of shared memory");

// Shared-memory operand descriptor, K-major without swizzle: core matrices of
// 8 rows x 16 bytes, 128 bytes apart along K and `sbo` along the rows.  The
// low word holds the address (in 16-byte units: adding to it moves the
// operand) and the K distance, the high word the row distance.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr) { return (addr >> 4) | (128 >> 4) << 16; }
__device__ __forceinline__ uint64_t desc(uint32_t lo, uint32_t sbo) {
  return (uint64_t)((sbo >> 4) | 1u << 14) << 32 | lo;
}

// Instruction descriptor of kind::mxf4: E2M1 operands (1), both K-major, E8M0
// scales (bit 23), M = 128; N in bits 17-22 (N / 8), the scales' pair within
// their 32-bit column in bits 4-5 (B) and 29-30 (A).
__device__ __forceinline__ uint32_t idesc(int N, int sf) {
  return (uint32_t)sf << 4 | 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | 1u << 23 | (uint32_t)(kMxRows >> 4) << 24 |
         (uint32_t)sf << 29;
}

__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb,
                                         bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"((uint32_t)add));
}

// 32 lanes x 16 bytes of shared memory to four TMEM columns, the same in each
// of the four lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t lo) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc(lo, 128)) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// Barrier of the 128 threads of an epilogue group, and whether `ok` holds in
// all of them.
__device__ __forceinline__ void group_barrier(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool all_of_group(bool ok, int id) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok), "r"(id)
      : "memory");
  return r != 0;
}

// mbarrier operations and bulk copies on shared-memory addresses.
__device__ __forceinline__ bool try_at(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, Bars* B, int* err) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (try_at(bar, parity)) return true;
    if ((i & 255) == 255 && tc::aborted(B)) return false;
    if (i > 128) __nanosleep(64);
  }
  set_error(err, kDevTimeout);
  *(volatile int*)&B->abort = 1;
  return false;
}
__device__ __forceinline__ bool wait_at(uint32_t bar, uint32_t parity, Bars* B, int* err) {
  return try_at(bar, parity) || wait_slow(bar, parity, B, err);
}
__device__ __forceinline__ void expect_at(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_at(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// One lane of a converged warp.  The compiler knows such a branch to have a
// single thread and keeps the operands of the tensor-core instructions in
// uniform registers; under `lane == 0` it serialises every one of them over
// the warp, about 90 cycles each (a K chunk of 128 tokens took 1500 cycles
// instead of 800).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

// The units of a CTA in turn (each role walks them by itself): weight tile,
// first token row, tokens.  Within an expert, units that follow one another
// share the weight tile.  The expert only moves forward, by steps through
// shared memory; searching for it in the offsets in global memory cost each
// role 1000 to 1700 cycles per unit.
struct Units {
  int u, e, first, next;  // unit; expert, its first unit and the next expert's
  int wt, row0, n;
  size_t w_tile;

  __device__ __forceinline__ void start(const Params& P, const Bars* B) {
    u = (int)blockIdx.x;
    e = 0;
    first = 0;
    next = P.offsets ? B->first[1] * P.w_tiles : 0x7fffffff;
  }
  __device__ __forceinline__ void locate(const Params& P, const Bars* B) {
    if (P.offsets) {
      while (u >= next) {  // u is below the last expert's end
        ++e;
        first = next;
        next = B->first[e + 1] * P.w_tiles;
      }
      const unsigned tt = (unsigned)(B->first[e + 1] - B->first[e]), r = (unsigned)(u - first);
      wt = (int)(r / tt);
      const int t = (int)(r - wt * tt);
      row0 = B->row0[e] + t * kMxRows;
      n = min(kMxRows, B->count[e] - t * kMxRows);
    } else {
      const unsigned tt = (unsigned)(P.n_tokens + kMxRows - 1) / kMxRows;
      wt = (int)((unsigned)u / tt);
      row0 = (int)(u - wt * tt) * kMxRows;
      n = min(kMxRows, P.n_tokens - row0);
    }
    w_tile = (size_t)e * P.w_tiles + wt;
  }
};

// gelu_tanh(g) * u; 0.5 g (1 + tanh(z)) = g / (1 + exp(-2z)), which keeps its
// relative precision for large negative g.  The exponent saturates harmlessly:
// exp -> inf gives 0, exp -> 0 gives g.
__device__ __forceinline__ float geglu(float g, float u) {
  const float z2 = 1.5957691216057308f * fmaf(0.044715f * g * g, g, g);
  return __fdividef(g, 1.f + __expf(-z2)) * u;
}

// A chunk of n blocks (even): its scales to tensor memory, then n / 2 MMAs.
// wa, xa: descriptor low words of the weights' and the tokens' chunk.
template <int n>
__device__ __forceinline__ void chunk_mma(uint32_t acc, uint32_t wa, uint32_t xa, uint32_t sf, uint32_t id0,
                                          uint32_t id2, bool add) {
  constexpr int kGroups = (n + 3) / 4;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    copy_scales(sf + 4 * g, wa + 32 * g);
    copy_scales(sf + 8 + 4 * g, xa + 32 * g);
  }
#pragma unroll
  for (int j = 0; j < n / 2; ++j)
    mma_mxf4(acc, desc(wa + 32 * kGroups + j * 16, n * 128), desc(xa + 32 * kGroups + j * 16, n * 128),
             j & 1 ? id2 : id0, sf + (j >> 1) * 4, sf + 8 + (j >> 1) * 4, add || j > 0);
}

enum : int { kModeF32 = 0, kModeF16 = 1, kModeBF16 = 2, kModeGated = 3 };

template <int MODE>
__global__ void __launch_bounds__(kThreads, 1) mx4_gemm_kernel(const Params P) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Bars* B = reinterpret_cast<Bars*>(smem_raw);
  uint8_t* ring = smem_raw + kBarBytes;
  float* ex = reinterpret_cast<float*>(ring + kStages * kStageBytes);  // GeGLU exchange
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&B->full[i], 1);
      mbar_init(&B->empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->acc_full[i], 1);
      mbar_init(&B->acc_empty[i], 8);
    }
    mbar_init(&B->drain, 1);
    B->abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&B->tmem_base)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  pdl_wait();
  pdl_trigger();
  if (P.offsets && warp == 2) {  // token tiles before each expert
    constexpr int kPer = kMaxExperts / 32;
    int c[kPer], s = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int x = lane * kPer + i;
      c[i] = s;
      if (x < P.E) {
        const int n = P.counts[x];
        B->count[x] = n;
        B->row0[x] = P.offsets[x];
        s += (n + kMxRows - 1) / kMxRows;
      }
    }
    int up = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += y;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane * kPer + i < P.E) B->first[lane * kPer + i] = up - s + c[i];
    if (lane == 31) B->first[P.E] = up;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = B->tmem_base;
  const int n_units = (P.offsets ? B->first[P.E] : (P.n_tokens + kMxRows - 1) / kMxRows) * P.w_tiles;
  const size_t tile_bytes = mx_tile_bytes(P.nb);

  // The producer's and the issuer's loops run in one thread each, where every
  // instruction costs its latency: addresses advance instead of being
  // computed, and whole chunks have constant sizes.
  const int n_full = P.nb / kMxChunk, n_tail = P.nb % kMxChunk;
  const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(&B->full[0]), empty0 = smem_u32(&B->empty[0]);
  if (warp == 0) {
    if (elect_one()) {
      int s = 0, issued = 0;
      uint32_t ph = 0;
      auto load = [&](const uint8_t* w, const uint8_t* x, uint32_t wb, uint32_t xb) {
        if (!wait_at(empty0 + 8 * s, ph ^ 1, B, P.err)) return false;
        const uint32_t bar = full0 + 8 * s, dst = ring0 + s * kStageBytes;
        expect_at(bar, wb + xb);
        copy_at(dst, w, wb, bar);
        copy_at(dst + kMxChunkBytes, x, xb, bar);
        ++issued;
        if (++s == kStages) {
          s = 0;
          ph ^= 1;
        }
        return true;
      };
      bool ok = true;
      Units U;
      for (U.start(P, B); U.u < n_units && ok; U.u += gridDim.x) {
        U.locate(P, B);
        const uint8_t* w = P.w + U.w_tile * tile_bytes;
        const uint8_t* x = P.x + (size_t)(U.row0 / kMxRows) * tile_bytes;
        const uint32_t groups = ((U.n + 15) & ~15) >> 3, xb = 1024 + groups * (kMxChunk * 128);
        for (int c = 0; c < n_full && ok; ++c) {
          ok = load(w, x, kMxChunkBytes, xb);
          w += kMxChunkBytes;
          x += kMxChunkBytes;
        }
        if (n_tail && ok) ok = load(w, x, mx_chunk_bytes(n_tail), mx_scale_bytes(n_tail) + groups * (n_tail * 128));
      }
      // Whatever happened, every copy lands before the block gives up its
      // shared memory.
      for (int i = 0; i < min(issued, kStages); ++i) {
        if (--s < 0) {
          s = kStages - 1;
          ph ^= 1;
        }
        mbar_wait_bounded(&B->full[s], ph, nullptr);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      int s = 0, a = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      Units U;
      for (U.start(P, B); U.u < n_units && ok; U.u += gridDim.x) {
        U.locate(P, B);
        const int N = (U.n + 15) & ~15;
        const uint32_t id0 = idesc(N, 0), id2 = idesc(N, 2);
        if (!(ok = wait_bar(&B->acc_empty[a], aph ^ 1, B, P.err))) break;
        fence_after();
        const uint32_t acc = tmem + kAcc0 + a * kAccCols;
        auto chunk = [&](auto issue, bool add) {
          if (!wait_at(full0 + 8 * s, ph, B, P.err)) return false;
          fence_after();
          const uint32_t wa = desc_lo(ring0 + s * kStageBytes);
          issue(acc, wa, wa + (kMxChunkBytes >> 4), tmem + kSf0 + s * kSfCols, id0, id2, add);
          mma_commit(&B->empty[s]);
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
          return true;
        };
        for (int c = 0; c < n_full && ok; ++c) ok = chunk(chunk_mma<kMxChunk>, c > 0);
        if (ok && n_tail == 2) ok = chunk(chunk_mma<2>, n_full > 0);
        if (ok && n_tail == 4) ok = chunk(chunk_mma<4>, n_full > 0);
        if (ok && n_tail == 6) ok = chunk(chunk_mma<6>, n_full > 0);
        if (!ok) break;
        mma_commit(&B->acc_full[a]);
        if (a ^= 1; a == 0) aph ^= 1;
      }
      mma_commit(&B->drain);  // and every MMA ends before the TMEM goes
      mbar_wait_bounded(&B->drain, 0, nullptr);
    }
  } else if (warp >= 4) {
    // Two groups of four warps; a group's warp q reads the lanes 32q..32q+31
    // of tensor memory (weight rows), the groups take 32 columns (tokens) in
    // turn.
    const int q = warp & 3, grp = (warp - 4) >> 2;
    int a = 0;
    uint32_t aph = 0;
    Units U;
    for (U.start(P, B); U.u < n_units; U.u += gridDim.x) {
      U.locate(P, B);
      bool ok = wait_bar(&B->acc_full[a], aph, B, P.err);
      // All lanes leave together; the four warps of a group where they meet
      // at barriers.
      if constexpr (MODE == kModeGated) ok = all_of_group(ok, 1 + grp);
      else ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16) + kAcc0 + a * kAccCols;
      uint32_t r[32];
      if constexpr (MODE == kModeGated) {
        // 32 tokens at a time: all rows to shared memory (rows 0..63 gate,
        // 64..127 up), then two threads per (token, block of 32 outputs).
        const int nba = mx_blocks(P.n_out);
        float* x = ex + grp * (kMxRows * kExPitch);
        const int half = lane & 1, t = (q & 1) * 16 + (lane >> 1), b = q >> 1, blk = U.wt * 2 + b;
        const float* xg = x + (32 * b + 16 * half) * kExPitch + t;
        uint8_t* tile = P.act + (size_t)(U.row0 / kMxRows) * mx_tile_bytes(nba);
        for (int c0 = 32 * grp; c0 < U.n; c0 += 64) {
          tmem_ld32(acc + c0, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) x[(32 * q + lane) * kExPitch + i] = __uint_as_float(r[i]);
          group_barrier(1 + grp);
          float v[16];
          uint32_t amax = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = geglu(xg[i * kExPitch], xg[(64 + i) * kExPitch]);
            amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
          }
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          float inv;
          const uint32_t s = mx_scale(amax, inv);
          if (c0 + t < U.n && blk < nba) {
            *reinterpret_cast<uint2*>(tile + mx_code_offset(nba, c0 + t, blk) + 8 * half) =
                make_uint2(mx_pack8(v, inv), mx_pack8(v + 8, inv));
            if (half == 0) tile[mx_scale_offset(c0 + t, blk)] = (uint8_t)s;
          }
          group_barrier(1 + grp);
        }
      } else {
        const int f = U.wt * kMxRows + 32 * q + lane;
        for (int c0 = 32 * grp; c0 < U.n; c0 += 64) {
          tmem_ld32(acc + c0, r);
          tmem_wait_ld();
          using E = Elem<MODE == kModeF32 ? kF32 : MODE == kModeF16 ? kF16 : kBF16>;
          typename E::T* o = static_cast<typename E::T*>(P.out) + (long long)(U.row0 + c0) * P.ldo + f;
          const int n = f < P.n_out ? min(32, U.n - c0) : 0;
          if (n == 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              *o = E::put(__uint_as_float(r[i]));
              o += P.ldo;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (i < n) *o = E::put(__uint_as_float(r[i]));
              o += P.ldo;
            }
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&B->acc_empty[a]);
      if (a ^= 1; a == 0) aph ^= 1;
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int MODE>
cudaError_t launch(const Params& P, int units, cudaStream_t s) {
  static SmemOptIn cache;
  const size_t smem = kBarBytes + kStages * kStageBytes + (MODE == kModeGated ? kExBytes : 0);
  const cudaError_t st = ensure_smem(mx4_gemm_kernel<MODE>, smem, cache);
  if (st != cudaSuccess) return st;
  return launch_pdl(mx4_gemm_kernel<MODE>, dim3(std::max(1, std::min(units, tc_num_sms()))), dim3(kThreads), smem, s, P);
}

}  // namespace mx

cudaError_t launch_mx4_gemm(int type, const uint8_t* w, const uint8_t* x, const int32_t* offsets,
                            const int32_t* counts, int E, int n_tokens, int rows, int cols, bool gated, void* out,
                            long long ldo, uint8_t* act, long long max_token_tiles, int* err, cudaStream_t s) {
  mx::Params P{};
  P.w = w;
  P.x = x;
  P.offsets = offsets;
  P.counts = counts;
  P.E = E;
  P.n_tokens = n_tokens;
  P.w_tiles = (rows + kMxRows - 1) / kMxRows;
  P.nb = mx_blocks(cols);
  P.n_out = gated ? rows / 2 : rows;
  P.out = out;
  P.ldo = ldo;
  P.act = act;
  P.err = err;
  const int units = (int)std::min<long long>(max_token_tiles * P.w_tiles, 1 << 20);
  if (gated) return mx::launch<mx::kModeGated>(P, units, s);
  switch (type) {
    case kF32: return mx::launch<mx::kModeF32>(P, units, s);
    case kF16: return mx::launch<mx::kModeF16>(P, units, s);
    default: return mx::launch<mx::kModeBF16>(P, units, s);
  }
}

}  // namespace mrml
