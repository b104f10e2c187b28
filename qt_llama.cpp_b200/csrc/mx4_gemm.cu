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
//   warps 0, 2 producers of the weights and of the tokens: a bulk copy per K
//              chunk (the matrix format is the shared-memory operand layout,
//              mx4.cuh)
//   warp 1     TMEM allocation; one lane copies the chunk's scales to tensor
//              memory and issues the MMAs
//   warps 4-11 epilogue, on the other of two accumulators
//
// With many tokens per expert those units are bound by the copies from L2 to
// shared memory: 34 KB per 128 x 128 x 256 step at the 64 bytes a cycle that
// an SM takes in is twice the tensor cores' time.  There, pairs of CTAs share
// a unit of 256 weight rows and 192 token rows (cta_group::2, M = 256): each
// copies its own 128 weight rows and half of the token rows, 31 KB per 128 x
// 192 x 256, and the first CTA's warp 1 issues for both.  The second CTA's
// warp 1 passes on that its stage has landed.
//
// A few tokens come unquantised: every CTA quantises them all into its own
// shared memory and, in the expert layer, sorts their (token, slot) pairs by
// itself: launches for it cost more than the repeated work.  The gate and up
// product multiplies all of them by each expert that has a pair (N = 16 is the
// least that the tensor cores take) and keeps the pairs' columns.
//
// Measured (weights of a 128-expert layer, H = 2816, I = 704): 64 tokens' gate
// and up product 40 us for 270 MB of weights and activations, 6.7 TB/s, the
// copy rate; 8192 tokens' 155 us, 3.4 PFLOP/s, no unit at its limit (of 64 bytes
// a cycle 41 copied in, the shared-memory pipe at 60 %: 34 for the tensor cores,
// 26 for the GeGLU's exchange; the tensor pipe at 48 %), and the down product 158
// us, bound by writing its 738 MB of f32 rows (5.4 TB/s over all its DRAM
// traffic).  Dense bf16: 4096 x 4224 x 2816 27 us, 3.6 PFLOP/s, 374 units for 74
// pairs, so five waves and a sixth of four units; 8192^3 200 us, 5.5 PFLOP/s.
//
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
constexpr int kThreads = 384;
constexpr int kFewTokens = 16, kFewWarps = 10;                   // tokens that a CTA quantises itself, and its warps for it
constexpr int kFewChunkBytes = 1024 + kFewTokens * kMxChunk * 16;  // their scales and codes per K chunk
constexpr int kFewCols = 8192;
constexpr int kFewPairs = 128;  // (token, slot) pairs that a CTA sorts itself: one expert's fit a tile
constexpr int kExPitch = 33;                          // f32 per row of the GeGLU exchange
constexpr int kExBytes = 2 * kMxRows * kExPitch * 4;  // two groups' 128 rows x 32 tokens

// Shapes of one CTA (kPair = false) and of a pair.  A stage holds the weights'
// chunk, then the tokens' scales (one group of 1024 bytes per 128-row tile
// that the unit touches) and codes.  Tensor memory holds two accumulators,
// then each stage's scales: 8 columns of weights, then per four blocks one
// group of four columns per token tile.
template <bool kPair>
struct Shape {
  static constexpr int kTokens = kPair ? 192 : 128;             // token rows of a unit
  static constexpr int kTokenTiles = kPair ? 2 : 1;             // 128-row tiles they touch
  static constexpr int kTokenScales = kTokenTiles * 1024;
  static constexpr int kStageBytes = kMxChunkBytes + kTokenScales + (kPair ? kTokens / 2 : kTokens) * kMxChunk * 16;
  static constexpr uint32_t kSf0 = 2 * kTokens, kSfCols = 8 + 8 * kTokenTiles;
  static_assert(kSf0 + kStages * kSfCols <= 512, "tensor memory has 512 columns");
  // A unit's first row sets the column where its scales start in their group of
  // four (Issue::shift); only even columns are supported, so units start at
  // multiples of 64 rows (and with one token tile at that tile's start).
  static_assert(kTokens % 64 == 0 && kMxRows % 64 == 0 && (kPair || kTokens % kMxRows == 0),
                "units start at even columns of the token scales");
};

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
  // A few (token, slot) pairs instead of sorted rows: every CTA sorts them
  // itself, the experts in the order of their first pairs, one tile each.
  const int32_t* ids;
  int32_t* pos;            // [pairs] each pair's row or -1, written by one CTA; or null
  int pairs, K;
  const void* raw;         // unquantised tokens [n_tokens][ldx], cols columns (QT >= 0)
  long long ldx;
  int cols, raw_vec;
  // Nothing but the tokens (and, for the GeGLU's result, earlier readers of
  // act) comes from the kernel right before this one or runs beside it; the
  // unit list and the weights are older than a launch that waited before it let
  // its successors start (kernels.h), and need no wait here.
  int early;
  // `out` is the caller's: the next launch may read it without waiting
  // (kernels.h), and does not start early.
  int last;
};

struct __align__(8) Bars {
  uint64_t full[kStages], empty[kStages], peer_full[kStages], acc_full[2], acc_empty[2], drain, tokens;
  uint32_t tmem_base;
  int abort;
  int first[kMaxExperts + 1];  // token tiles of earlier experts
  int row0[kMaxExperts], count[kMaxExperts];  // each expert's first row and rows
  // of a few pairs: experts that have some; each one's id; pairs' tokens,
  // expert by expert, and (row0) where an expert's start among them
  int experts;
  uint8_t expert[kFewPairs], token[kFewPairs];
};
static_assert(kMaxExperts <= 256 && kFewTokens <= 256, "expert and token numbers are kept in bytes");
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
// scales (bit 23), M = 128 or 256; N in bits 17-22 (N / 8), the scales' pair
// within their 32-bit column in bits 4-5 (B) and 29-30 (A).
__device__ __forceinline__ uint32_t idesc(int M, int N, int sf) {
  return (uint32_t)sf << 4 | 1u << 7 | 1u << 10 | (uint32_t)(N >> 3) << 17 | 1u << 23 | (uint32_t)(M >> 4) << 24 |
         (uint32_t)sf << 29;
}

#define MRML_MMA_MXF4(GROUP)                                                                              \
  asm volatile(                                                                                           \
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"                                                  \
      "tcgen05.mma.cta_group::" #GROUP                                                                    \
      ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),              \
      "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"((uint32_t)add))
template <bool kPair>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb,
                                         bool add) {
  if constexpr (kPair) MRML_MMA_MXF4(2);
  else MRML_MMA_MXF4(1);
}
#undef MRML_MMA_MXF4

// 32 lanes x 16 bytes of shared memory to four TMEM columns, the same in each
// of the four lane quarters (in a pair: each CTA's memory to its own TMEM).
template <bool kPair>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t lo) {
  if constexpr (kPair)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc(lo, 128)) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc(lo, 128)) : "memory");
}

// Arrives on a barrier (in a pair: on both CTAs') once the MMAs and copies
// issued so far have completed.
template <bool kPair>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (kPair)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  else
    mma_commit(bar);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrives on the first CTA's barrier at the same offset.
// ... with what this CTA's copies have brought to its shared memory, which the
// first CTA's MMAs read: this thread has acquired it from the copies' own
// barrier and passes it on by a release over the cluster.  Only shared memory
// changes hands, so the fence is restricted to that; `arrive.release.cluster`,
// which covers global memory too, takes 900 cycles, longer than a chunk's MMAs
// (8192^3: 333 us against 200).
__device__ __forceinline__ void release_to_leader(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
      "fence.release.sync_restrict::shared::cta.cluster;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// ... and after reads of tensor memory, which the tcgen05 fences on the two
// sides of the barrier order; no memory changes hands, so it is relaxed.
__device__ __forceinline__ void arrive_leader(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, 0;\n\t"
      "mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
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
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
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

// A producer's place in the ring of stages.
struct Ring {
  uint32_t empty0, full0, ring0;
  int s;
  uint32_t ph;
  __device__ __forceinline__ uint32_t empty() const { return empty0 + 8 * s; }
  __device__ __forceinline__ uint32_t full() const { return full0 + 8 * s; }
  __device__ __forceinline__ uint32_t stage(int bytes) const { return ring0 + s * bytes; }
  __device__ __forceinline__ void next() {
    if (++s == kStages) {
      s = 0;
      ph ^= 1;
    }
  }
};

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

// The units of a CTA (or pair) in turn (each role walks them by itself): weight tile,
// first token row, tokens.  Within an expert, units that follow one another
// share the weight tile.  The expert only moves forward, by steps through
// shared memory; searching for it in the offsets in global memory cost each
// role 1000 to 1700 cycles per unit.
template <bool kPair>
struct Units {
  static constexpr int kTokens = Shape<kPair>::kTokens;
  int u, e, w_units, first, next;  // unit; expert, its first unit and the next expert's
  int wt, row0, n, list;           // list: the first pair's place in Bars::token
  size_t w_tile;

  __device__ __forceinline__ void start(const Params& P, const Bars* B) {
    u = (int)blockIdx.x / (kPair ? 2 : 1);
    w_units = kPair ? (P.w_tiles + 1) / 2 : P.w_tiles;
    e = 0;
    first = 0;
    next = P.offsets ? B->first[1] * w_units : 0x7fffffff;
  }
  __device__ __forceinline__ void locate(const Params& P, const Bars* B) {
    if (P.ids) {
      const unsigned j = (unsigned)u / (unsigned)P.w_tiles;
      wt = (int)(u - j * P.w_tiles);
      e = B->expert[j];
      row0 = (int)j * kMxRows;
      n = B->count[j];
      list = B->row0[j];
    } else if (P.offsets) {
      while (u >= next) {  // u is below the last expert's end
        ++e;
        first = next;
        next = B->first[e + 1] * w_units;
      }
      const unsigned tt = (unsigned)(B->first[e + 1] - B->first[e]), r = (unsigned)(u - first);
      wt = (int)(r / tt);
      const int t = (int)(r - wt * tt);
      row0 = B->row0[e] + t * kTokens;
      n = min(kTokens, B->count[e] - t * kTokens);
    } else {
      const unsigned tt = (unsigned)(P.n_tokens + kTokens - 1) / kTokens;
      wt = (int)((unsigned)u / tt);
      row0 = (int)(u - wt * tt) * kTokens;
      n = min(kTokens, P.n_tokens - row0);
    }
    if constexpr (kPair) wt = 2 * wt + (int)(blockIdx.x & 1);  // the last pair's second tile may not exist
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

// What the MMAs of a unit have in common.
struct Issue {
  uint32_t acc, id0, id2;
  uint32_t shift;  // column of the unit's first token row within its scales
  bool two;        // the unit touches two token tiles
};

// A chunk of n blocks (even): its scales to tensor memory, then n / 2 MMAs.
// wa, xs: descriptor low words of the weights' chunk and of the tokens' scales,
// which their codes follow; sf: the stage's scale columns.
template <bool kPair, int n>
__device__ __forceinline__ void chunk_mma(const Issue& I, uint32_t wa, uint32_t xs, uint32_t sf, bool add) {
  constexpr int kGroups = (n + 3) / 4, kTiles = Shape<kPair>::kTokenTiles;
  // one tile's scales are directly followed by its codes (mx4.cuh)
  const uint32_t xa = xs + (kPair ? Shape<kPair>::kTokenScales >> 4 : 32 * kGroups);
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    copy_scales<kPair>(sf + 4 * g, wa + 32 * g);
    copy_scales<kPair>(sf + 8 + 4 * kTiles * g, xs + 32 * g);
    if (kPair && I.two) copy_scales<kPair>(sf + 12 + 4 * kTiles * g, xs + 64 + 32 * g);
  }
#pragma unroll
  for (int j = 0; j < n / 2; ++j)
    mma_mxf4<kPair>(I.acc, desc(wa + 32 * kGroups + j * 16, n * 128), desc(xa + j * 16, n * 128), j & 1 ? I.id2 : I.id0,
                    sf + (j >> 1) * 4, sf + 8 + 4 * kTiles * (j >> 1) + (kPair ? I.shift : 0), add || j > 0);
}

// A few pairs sorted by one warp: groups of 32 in turn, the experts numbered as
// they appear (Bars::first holds the number, or -1), the pairs ranked within
// theirs by a warp match.
__device__ __forceinline__ void sort_few(const Params& P, Bars* B, int lane) {
  constexpr int kGroups = kFewPairs / 32;
  const unsigned below = (1u << lane) - 1;
  if (P.pairs <= 32) {  // one group: no counts to carry over, 0.6 us less in a one-token layer
    int id = lane < P.pairs ? P.ids[lane] : -1;
    if (id >= P.E) {
      if (blockIdx.x == 0) set_error(P.err, kDevBadExpert);
      id = -1;
    }
    const bool has = id >= 0;
    const unsigned same = __match_any_sync(0xffffffffu, has ? id : -1);
    const int n = __popc(same), leader = __ffs(same) - 1, rank = __popc(same & below);
    const bool lead = has && rank == 0;
    const unsigned leads = __ballot_sync(0xffffffffu, lead);
    const int j = __popc(leads & ((1u << leader) - 1));
    int start = lead ? n : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, start, o);
      if (lane >= o) start += y;
    }
    start = __shfl_sync(0xffffffffu, start - n, leader);
    if (lead) {
      B->expert[j] = (uint8_t)id;
      B->count[j] = n;
      B->row0[j] = start;
    }
    if (has) B->token[start + rank] = (uint8_t)(lane / P.K);
    if (lane == 0) B->experts = __popc(leads);
    if (P.pos && blockIdx.x == 0 && lane < P.pairs) P.pos[lane] = has ? j * kMxRows + rank : -1;
    return;
  }
  for (int e = lane; e < P.E; e += 32) B->first[e] = -1;
  for (int j = lane; j < kFewPairs; j += 32) B->count[j] = 0;
  int id[kGroups], j[kGroups], rank[kGroups], experts = 0;
#pragma unroll
  for (int g = 0; g < kGroups; ++g) id[g] = 32 * g + lane < P.pairs ? P.ids[32 * g + lane] : -1;
  __syncwarp();
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (32 * g >= P.pairs) break;
    if (id[g] >= P.E) {
      if (blockIdx.x == 0) set_error(P.err, kDevBadExpert);
      id[g] = -1;
    }
    const bool has = id[g] >= 0;
    if (!has) id[g] = -1;
    const unsigned same = __match_any_sync(0xffffffffu, id[g]);
    const bool lead = has && (same & below) == 0, fresh = lead && B->first[id[g]] < 0;
    const unsigned all = __ballot_sync(0xffffffffu, fresh);
    if (fresh) {
      const int n = experts + __popc(all & below);
      B->first[id[g]] = n;
      B->expert[n] = (uint8_t)id[g];
    }
    experts += __popc(all);
    __syncwarp();
    if (has) {
      j[g] = B->first[id[g]];
      rank[g] = B->count[j[g]] + __popc(same & below);
    }
    __syncwarp();
    if (lead) B->count[j[g]] += __popc(same);
    __syncwarp();
  }
  if (lane == 0) B->experts = experts;
  int c[kGroups], s = 0;  // where each expert's pairs start: kGroups experts per lane
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    c[i] = s;
    s += B->count[lane * kGroups + i];
  }
  int up = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, up, o);
    if (lane >= o) up += y;
  }
#pragma unroll
  for (int i = 0; i < kGroups; ++i) B->row0[lane * kGroups + i] = up - s + c[i];
  __syncwarp();
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    if (32 * g >= P.pairs) break;
    const int p = 32 * g + lane;
    if (id[g] >= 0) B->token[B->row0[j[g]] + rank[g]] = (uint8_t)(p / P.K);
    if (P.pos && blockIdx.x == 0 && p < P.pairs) P.pos[p] = id[g] >= 0 ? j[g] * kMxRows + rank[g] : -1;
  }
}

enum : int { kModeF32 = 0, kModeF16 = 1, kModeBF16 = 2, kModeGated = 3 };

// QT >= 0: the tokens come unquantised, as QT, at most kFewTokens of them in one
// matrix: every CTA quantises them all into its own shared memory, where they
// stay, and only the weights pass through the ring.  One launch instead of two.
template <int MODE, bool kPair, int QT = -1>
__global__ void __launch_bounds__(kThreads, 1) mx4_gemm_kernel(const Params P) {
  using S = Shape<kPair>;
  constexpr int kStageBytes = QT >= 0 ? kMxChunkBytes : S::kStageBytes;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Bars* B = reinterpret_cast<Bars*>(smem_raw);
  uint8_t* ring = smem_raw + kBarBytes;
  float* ex = reinterpret_cast<float*>(ring + kStages * kStageBytes +  // GeGLU exchange
                                       (QT >= 0 ? (P.nb + kMxChunk - 1) / kMxChunk * kFewChunkBytes : 0));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? (int)(blockIdx.x & 1) : 0;  // in the cluster of two

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&B->full[i], QT >= 0 ? 1 : 2);
      mbar_init(&B->empty[i], 1);
      mbar_init(&B->peer_full[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B->acc_full[i], 1);
      mbar_init(&B->acc_empty[i], kPair ? 16 : 8);
    }
    mbar_init(&B->drain, 1);
    mbar_init(&B->tokens, kFewWarps);
    B->abort = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&B->tmem_base)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&B->tmem_base)));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
  }
  if (!P.early) pdl_wait();
  if (!P.last) pdl_trigger();
  if (P.ids && warp == 3) sort_few(P, B, lane);
  if (P.offsets && warp == 3) {  // token tiles before each expert
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
        s += (n + S::kTokens - 1) / S::kTokens;
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
  if constexpr (kPair) cluster_sync();  // both CTAs' barriers are initialised
  else __syncthreads();
  fence_after();
  const uint32_t tmem = B->tmem_base;
  const int n_units = (P.ids       ? B->experts
                       : P.offsets ? B->first[P.E]
                                   : (P.n_tokens + S::kTokens - 1) / S::kTokens) *
                      (kPair ? (P.w_tiles + 1) / 2 : P.w_tiles);
  const int step = (int)gridDim.x / (kPair ? 2 : 1);
  const size_t tile_bytes = mx_tile_bytes(P.nb);

  // The producer's and the issuer's loops run in one thread each, where every
  // instruction costs its latency: addresses advance instead of being
  // computed, and whole chunks have constant sizes.
  const int n_full = P.nb / kMxChunk, n_tail = P.nb % kMxChunk;
  const uint32_t ring0 = smem_u32(ring), full0 = smem_u32(&B->full[0]), empty0 = smem_u32(&B->empty[0]);
  if (QT >= 0 && warp >= 2) {
    // the tokens: a thread per (token, block); then to their other roles
    constexpr int kType = QT >= 0 ? QT : kF32;
    uint8_t* few = ring + kStages * kStageBytes;
    for (int i = threadIdx.x - 64; i < P.n_tokens * P.nb; i += 32 * kFewWarps) {
      const int t = i / P.nb, b = i % P.nb, c = b / kMxChunk, bl = b % kMxChunk;
      MxPart<kType, 32> v;
      if (b * 32 < P.cols)
        load_block<kType>(static_cast<const typename Elem<kType>::T*>(P.raw) + t * P.ldx, b, P.cols, P.raw_vec, v);
      else
        v.zero();
      uint4 q;
      const uint32_t s = quantize_block(v, q);
      const int n = min(kMxChunk, P.nb - c * kMxChunk);
      uint8_t* chunk = few + c * kFewChunkBytes;
      *reinterpret_cast<uint4*>(chunk + mx_scale_bytes(n) + (t >> 3) * (n * 128) + bl * 128 + (t & 7) * 16) = q;
      chunk[(bl >> 2) * 512 + t * 16 + (bl & 3)] = (uint8_t)s;
    }
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&B->tokens);
  }
  if (warp == 0 || (QT < 0 && warp == 2)) {
    if (elect_one()) {
      // Warp 0 copies the weights, warp 2 the tokens: one thread for both was
      // what bounded the pairs' chunks (up to five copies each).
      if (warp == 2) pdl_wait();
      Ring R{empty0, full0, ring0, 0, 0};
      int issued = 0;
      bool ok = true;
      Units<kPair> U;
      for (U.start(P, B); U.u < n_units && ok; U.u += step) {
        U.locate(P, B);
        if (warp == 0) {
          const bool some = !kPair || U.wt < P.w_tiles;
          const uint8_t* w = P.w + U.w_tile * tile_bytes;
          auto load = [&](int n, uint32_t bytes) {
            if (!(ok = wait_at(R.empty(), R.ph ^ 1, B, P.err))) return;
            expect_at(R.full(), some ? bytes : 0);
            if (some) copy_at(R.stage(kStageBytes), w, bytes, R.full());
            w += kMxChunkBytes;
            R.next();
            ++issued;
          };
          for (int c = 0; c < n_full && ok; ++c) load(kMxChunk, kMxChunkBytes);
          if (n_tail && ok) load(n_tail, mx_chunk_bytes(n_tail));
        } else {
          const uint8_t* x = P.x + (size_t)(U.row0 / kMxRows) * tile_bytes;
          const int N = (U.n + 15) & ~15;
          // the CTA's row groups: all, or in a pair half of them, which may
          // start in either tile (group gi) and continue in the next (g1 more)
          const int groups = N / (kPair ? 16 : 8), from = U.row0 % kMxRows / 8 + rank * groups;
          const int gi = from % 16, g0 = min(groups, 16 - gi), g1 = groups - g0;
          const bool two = kPair && U.row0 % kMxRows + N > kMxRows;
          auto load = [&](int n, uint32_t sb) {
            if (!(ok = wait_at(R.empty(), R.ph ^ 1, B, P.err))) return;
            const uint32_t dst = R.stage(kStageBytes) + kMxChunkBytes, line = n * 128;
            if constexpr (kPair) {
              const uint8_t* xc = x + sb + (from >= 16 ? tile_bytes : 0);
              expect_at(R.full(), (two ? 2 * sb : sb) + groups * line);
              copy_at(dst, x, sb, R.full());
              copy_at(dst + S::kTokenScales, xc + gi * line, g0 * line, R.full());
              if (two) copy_at(dst + 1024, x + tile_bytes, sb, R.full());
              if (g1) copy_at(dst + S::kTokenScales + g0 * line, xc + tile_bytes, g1 * line, R.full());
            } else {  // scales and codes in one run
              expect_at(R.full(), sb + groups * line);
              copy_at(dst, x, sb + groups * line, R.full());
            }
            x += kMxChunkBytes;
            R.next();
            ++issued;
          };
          for (int c = 0; c < n_full && ok; ++c) load(kMxChunk, 1024);
          if (n_tail && ok) load(n_tail, mx_scale_bytes(n_tail));
        }
      }
      // Whatever happened, every copy lands before the block gives up its
      // shared memory; and so do the signals that the last stages are free
      // (unless the walk ended early: those stages may never be).
      for (int i = 0; i < min(issued, kStages); ++i) {
        if (--R.s < 0) {
          R.s = kStages - 1;
          R.ph ^= 1;
        }
        mbar_wait_bounded(&B->full[R.s], R.ph, nullptr);
        ok = ok && mbar_wait_bounded(&B->empty[R.s], R.ph, nullptr);
      }
    }
  } else if (warp == 1 && rank == 0) {
    if (elect_one()) {
      int s = 0, a = 0;
      uint32_t ph = 0, aph = 0;
      bool ok = true;
      if (QT >= 0) ok = wait_at(smem_u32(&B->tokens), 0, B, P.err);
      Units<kPair> U;
      for (U.start(P, B); U.u < n_units && ok; U.u += step) {
        U.locate(P, B);
        const int N = QT >= 0 ? kFewTokens : (U.n + 15) & ~15, M = kPair ? 2 * kMxRows : kMxRows;
        const Issue I{tmem + a * S::kTokens, idesc(M, N, 0), idesc(M, N, 2), (uint32_t)(U.row0 % kMxRows / 32),
                      U.row0 % kMxRows + N > kMxRows};
        if (!(ok = wait_at(smem_u32(&B->acc_empty[a]), aph ^ 1, B, P.err))) break;
        fence_after();
        uint32_t few = desc_lo(ring0 + kStages * kStageBytes);
        auto chunk = [&](auto issue, bool add) {
          if (!wait_at(full0 + 8 * s, ph, B, P.err)) return false;
          if (kPair && !wait_at(smem_u32(&B->peer_full[s]), ph, B, P.err)) return false;
          fence_after();
          const uint32_t wa = desc_lo(ring0 + s * kStageBytes);
          issue(I, wa, QT >= 0 ? few : wa + (kMxChunkBytes >> 4), tmem + S::kSf0 + s * S::kSfCols, add);
          few += kFewChunkBytes >> 4;
          commit<kPair>(&B->empty[s]);
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
          return true;
        };
        for (int c = 0; c < n_full && ok; ++c) ok = chunk(chunk_mma<kPair, kMxChunk>, c > 0);
        if (ok && n_tail == 2) ok = chunk(chunk_mma<kPair, 2>, n_full > 0);
        if (ok && n_tail == 4) ok = chunk(chunk_mma<kPair, 4>, n_full > 0);
        if (ok && n_tail == 6) ok = chunk(chunk_mma<kPair, 6>, n_full > 0);
        if (!ok) break;
        commit<kPair>(&B->acc_full[a]);
        if (a ^= 1; a == 0) aph ^= 1;
      }
      commit<kPair>(&B->drain);  // and every MMA ends before the TMEM goes
      mbar_wait_bounded(&B->drain, 0, nullptr);
    }
  } else if (kPair && warp == 1) {
    // the pair's second CTA: tells the first that a stage has landed here
    if (elect_one()) {
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      Units<kPair> U;
      const int chunks = n_full + (n_tail > 0);
      for (U.start(P, B); U.u < n_units && ok; U.u += step) {
        for (int c = 0; c < chunks; ++c) {
          if (!(ok = wait_at(full0 + 8 * s, ph, B, P.err))) break;
          release_to_leader(&B->peer_full[s]);
          if (++s == kStages) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // The first CTA's commits signal barriers of this one too, and an
      // arrival must not reach a CTA that has left: the last of them, which
      // the first CTA commits on every path, is waited for here as there.
      mbar_wait_bounded(&B->drain, 0, nullptr);
    }
  } else if (warp >= 4) {
    // Two groups of four warps; a group's warp q reads the lanes 32q..32q+31
    // of tensor memory (weight rows), the groups take 32 columns (tokens) in
    // turn.
    const int q = warp & 3, grp = (warp - 4) >> 2;
    pdl_wait();
    int a = 0;
    uint32_t aph = 0;
    Units<kPair> U;
    for (U.start(P, B); U.u < n_units; U.u += step) {
      U.locate(P, B);
      bool ok = wait_bar(&B->acc_full[a], aph, B, P.err);
      // All lanes leave together; the four warps of a group where they meet
      // at barriers.
      if constexpr (MODE == kModeGated) ok = all_of_group(ok, 1 + grp);
      else ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const uint32_t acc = tmem + ((uint32_t)(32 * q) << 16) + a * S::kTokens;
      uint32_t r[32];
      if constexpr (MODE == kModeGated) {
        // 32 tokens at a time: all rows to shared memory (rows 0..63 gate,
        // 64..127 up), then two threads per (token, block of 32 outputs).
        const int nba = mx_blocks(P.n_out);
        float* x = ex + grp * (kMxRows * kExPitch);
        const int half = lane & 1, t = (q & 1) * 16 + (lane >> 1), b = q >> 1, blk = U.wt * 2 + b;
        const float* xg = x + (32 * b + 16 * half) * kExPitch;
        const size_t act_tile = mx_tile_bytes(nba);
        for (int c0 = 32 * grp; c0 < U.n; c0 += 64) {
          // of unquantised tokens all were multiplied: each pair takes its own's column
          tmem_ld32(acc + (QT >= 0 ? 0 : c0), r);
          const int col = QT < 0 ? t : c0 + t < U.n ? B->token[U.list + c0 + t] : 0;
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) x[(32 * q + lane) * kExPitch + i] = __uint_as_float(r[i]);
          group_barrier(1 + grp);
          float v[16];
          uint32_t amax = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = geglu(xg[i * kExPitch + col], xg[(64 + i) * kExPitch + col]);
            amax = max(amax, __float_as_uint(v[i]) & 0x7fffffffu);
          }
          amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
          float inv;
          const uint32_t s = mx_scale(amax, inv);
          if (c0 + t < U.n && blk < nba) {
            const int row = U.row0 + c0 + t, rt = row % kMxRows;
            uint8_t* tile = P.act + (size_t)(row / kMxRows) * act_tile;
            *reinterpret_cast<uint2*>(tile + mx_code_offset(nba, rt, blk) + 8 * half) =
                make_uint2(mx_pack8(v, inv), mx_pack8(v + 8, inv));
            if (half == 0) tile[mx_scale_offset(rt, blk)] = (uint8_t)s;
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
      if (lane == 0) {
        if (rank == 0) mbar_arrive(&B->acc_empty[a]);
        else arrive_leader(&B->acc_empty[a]);
      }
      if (a ^= 1; a == 0) aph ^= 1;
    }
  }
  __syncwarp();
  fence_before();
  // In a pair, neither CTA leaves before the other's reads and arrivals.
  if constexpr (kPair) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    fence_after();
    if constexpr (kPair) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem));
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int MODE, bool kPair, int QT = -1>
cudaError_t launch(const Params& P, long long units, cudaStream_t s) {
  static SmemOptIn cache;
  const size_t smem = kBarBytes + (MODE == kModeGated ? kExBytes : 0) +
                      (QT >= 0 ? kStages * kMxChunkBytes + (P.nb + kMxChunk - 1) / kMxChunk * kFewChunkBytes
                               : kStages * Shape<kPair>::kStageBytes);
  const cudaError_t st = ensure_smem(mx4_gemm_kernel<MODE, kPair, QT>, smem, cache);
  if (st != cudaSuccess) return st;
  const int ctas = kPair ? 2 : 1;
  const int grid = ctas * (int)std::max<long long>(1, std::min<long long>(units, tc_num_sms() / ctas));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {2, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = kPair ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, mx4_gemm_kernel<MODE, kPair, QT>, P);
}

template <bool kPair>
cudaError_t launch_mode(int mode, const Params& P, long long units, cudaStream_t s) {
  switch (mode) {
    case kModeGated: return launch<kModeGated, kPair>(P, units, s);
    case kModeF32: return launch<kModeF32, kPair>(P, units, s);
    case kModeF16: return launch<kModeF16, kPair>(P, units, s);
    default: return launch<kModeBF16, kPair>(P, units, s);
  }
}

}  // namespace mx

cudaError_t launch_mx4_gemm(int type, const uint8_t* w, const uint8_t* x, const int32_t* offsets,
                            const int32_t* counts, int E, int n_tokens, int rows, int cols, bool gated, void* out,
                            long long ldo, uint8_t* act, long long tokens, bool early, int* err, cudaStream_t s) {
  mx::Params P{};
  P.early = early;
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
  P.last = offsets == nullptr;  // of the expert layer's products, both are read by launches of its own
  const int mode = gated ? mx::kModeGated : type == kF32 ? mx::kModeF32 : type == kF16 ? mx::kModeF16 : mx::kModeBF16;
  // Pairs of CTAs pay where there are enough units for several waves of them,
  // tokens to fill their tiles, and a sum long enough to be bound by the
  // operands and not by the results.  Measured, one CTA against pairs: 4096 x
  // 4224 x 2816 bf16 28.4 / 26.7 us (7 tiles per SM), 8192^3 234 / 200; 2048 x
  // 4224 x 2816 16.8 / 17.0 (3.6), 1024: 10.5 / 12.8, 256: 6.1 / 7.9; 65536
  // sorted tokens, gated K = 2816 162 / 155, f32 rows K = 704 158 / 168.
  const long long tiles = (tokens + 127) / 128 * P.w_tiles;
  if (tokens >= 192ll * E && 2 * tiles >= 9ll * tc_num_sms() && cols >= 1024)
    return mx::launch_mode<true>(mode, P, (tokens / 192 + E) * ((P.w_tiles + 1) / 2), s);
  return mx::launch_mode<false>(mode, P, (tokens / 128 + std::min<long long>(E, tokens)) * P.w_tiles, s);
}

// At most one block per quantising thread.  One launch against two, replayed in
// graphs (us, blocks in brackets):
//   704 -> 2816:   4 tokens (88) 4.4 / 4.9, 12 (264) 4.9 / 5.2, 16 (352) 5.4 / 5.2
//   1024 -> 1024:  8 (256) 5.4 / 5.5, 12 (384) 5.8 / 5.5
//   2816 -> 4224:  1 (88) 7.3 / 8.2, 3 (264) 7.7 / 8.3, 4 (352) 8.2 / 8.3, 6 (528) 8.3 / 7.8
//   4096 -> 4096:  2 (256) 8.9 / 9.0, 3 (384) 9.4 / 9.0
//   8192 -> 8192:  1 (256) 13.0 / 13.8, 2 (512) 13.6 / 13.8, 3 (768) 14.2 / 13.8
bool mx4_few_tokens(int tokens, int cols) {
  return tokens <= mx::kFewTokens && cols <= mx::kFewCols &&
         (long long)tokens * mx_blocks(cols) <= 32 * mx::kFewWarps;
}

cudaError_t launch_mx4_few(int type, const uint8_t* w, const void* x, long long ldx, int n_tokens, int rows, int cols,
                           void* out, long long ldo, int* err, cudaStream_t s) {
  mx::Params P{};
  P.w = w;
  P.E = 1;
  P.n_tokens = n_tokens;
  P.w_tiles = (rows + kMxRows - 1) / kMxRows;
  P.nb = mx_blocks(cols);
  P.n_out = rows;
  P.out = out;
  P.ldo = ldo;
  P.err = err;
  P.last = 1;
  P.raw = x;
  P.ldx = ldx;
  P.cols = cols;
  P.raw_vec = ((uintptr_t)x & 15) == 0 && (size_t)ldx * elem_bytes(type) % 16 == 0;
  switch (type) {
    case kF32: return mx::launch<mx::kModeF32, false, kF32>(P, P.w_tiles, s);
    case kF16: return mx::launch<mx::kModeF16, false, kF16>(P, P.w_tiles, s);
    default: return mx::launch<mx::kModeBF16, false, kBF16>(P, P.w_tiles, s);
  }
}

// Pairs that one warp sorts, and tokens that a CTA quantises itself: up to 2048
// blocks, as every CTA quantises them all.  Three launches against the five
// with a sort and a gather of their own, each step with other experts' weights,
// replayed in graphs (us):
//   H 2816, I 704, 128 experts top-8:  1 token 15.6 / 25.2, 8 39.6 / 47.0, 16 (1408 blocks) 58.6 / 62.5
//   H 1024, I 512, 16 top-2:           1 10.5 / 14.0, 16 13.2 / 15.5
//   H 4096, I 1024, 256 top-4:         1 17.3 / 31.6, 16 (2048) 74.6 / 83.9
//   H 5632, I 704, 32 top-4:           8 (1408) 35.6 / 37.8, 12 (2112) 44.2 / 43.1
//   H 8192, I 512, 64 top-8:           8 (2048) 64.9 / 67.9, 12 (3072) 73.6 / 73.3, 16 86.6 / 83.7
//   H 8192, I 2048, 16 top-2:          4 (1024) 43.8 / 45.4, 8 59.3 / 58.5, 16 81.2 / 75.6
bool mx4_few_pairs(int T, int K, int H) {
  return T <= mx::kFewTokens && H <= mx::kFewCols && T * K <= mx::kFewPairs && T * mx_blocks(H) <= 2048;
}

cudaError_t launch_mx4_few_gate_up(int type, const uint8_t* w, const void* x, long long ldx, const int32_t* ids,
                                   int32_t* pos, int T, int K, int E, int H, int I, uint8_t* act, int* err,
                                   cudaStream_t s) {
  mx::Params P{};
  P.w = w;
  P.E = E;
  P.n_tokens = T;
  P.w_tiles = (2 * I + kMxRows - 1) / kMxRows;
  P.nb = mx_blocks(H);
  P.n_out = I;
  P.act = act;
  P.err = err;
  P.ids = ids;
  P.pos = pos;
  P.pairs = T * K;
  P.K = K;
  P.raw = x;
  P.ldx = ldx;
  P.cols = H;
  P.raw_vec = ((uintptr_t)x & 15) == 0 && (size_t)ldx * elem_bytes(type) % 16 == 0;
  const long long units = (long long)std::min(E, T * K) * P.w_tiles;
  switch (type) {
    case kF32: return mx::launch<mx::kModeGated, false, kF32>(P, units, s);
    case kF16: return mx::launch<mx::kModeGated, false, kF16>(P, units, s);
    default: return mx::launch<mx::kModeGated, false, kBF16>(P, units, s);
  }
}

cudaError_t launch_mx4_few_down(const uint8_t* w, const uint8_t* act, const int32_t* ids, int T, int K, int E, int H,
                                int I, float* y, int* err, cudaStream_t s) {
  mx::Params P{};
  P.w = w;
  P.x = act;
  P.E = E;
  P.w_tiles = (H + kMxRows - 1) / kMxRows;
  P.nb = mx_blocks(I);
  P.n_out = H;
  P.out = y;
  P.ldo = H;
  P.err = err;
  P.ids = ids;
  P.pairs = T * K;
  P.K = K;
  P.early = 1;  // ids and weights are older than the launch before
  return mx::launch<mx::kModeF32, false>(P, (long long)std::min(E, T * K) * P.w_tiles, s);
}

}  // namespace mrml
