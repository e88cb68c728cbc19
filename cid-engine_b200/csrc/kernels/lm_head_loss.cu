// Softmax cross entropy of an LM head, without keeping the logits, and its
// gradient.  For rows h_r (16-bit, H wide), weight rows w_v and labels y_r:
//
//   z_rv = h_r . w_v            (f32 accumulation on the tensor cores, which truncates:
//                                loss and lse are 1e-6 to 2e-6 off at H = 4096, 1e-5 at
//                                16384)
//   lse_r = log sum_v exp z_rv,  loss_r = lse_r - z_{r, y_r}
//   d_rv = a_r exp(z_rv - lse_r) - b_r [v = y_r],   a = g_loss + g_lse, b = g_loss
//   dh = d W,   dW = d^T h
//
// Rows whose label is ignore_index take no part: a prepare kernel packs the
// other rows (count n, left on the device), the products run over n rows only,
// and nothing of an ignored row's hidden state is read, so NaN there reaches
// nothing.  The n rows keep their order, and every sum has a fixed order:
// repeated calls give identical bits.
//
// The backward goes over the vocabulary in pieces: a piece's logits are
// computed again, turned into d (16 bits) in a workspace, and multiplied with the
// weight (dh, summed in f32 over the pieces) and the hidden rows (that piece's rows
// of dW).  8 n V H flops a step (2 forward, 2
// again, 4 gradients) instead of 6 with kept logits, which would be n V floats.
//
// Roundings to 16 bits: d, because the tensor cores take 16-bit operands (the
// same step as a 16-bit gradient of the logits, at most half a step of each
// element; dh and dW get what the label's element lost back in f32, the largest
// of its row unless another token is favoured), and the outputs.  fp16 d is
// scaled by a power of two from the largest coefficient, so that neither a loss
// scale nor a division by the number of rows leaves fp16's range; elements below
// 2^-37 of that coefficient are lost.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace cid {
namespace {

constexpr int kCtaM = 128;  // rows of an output tile that one CTA holds
constexpr int kBN = 256;    // columns of an output tile
constexpr int kBK = 64;     // K elements a stage: one 128-byte swizzle row
constexpr int kUmmaK = 16;
constexpr int kAccBufs = 2;
constexpr uint32_t kTmemCols = kAccBufs * kBN;
constexpr uint32_t kBlockBytes = 64 * kBK * 2;  // one 64 x 64 block of an MN-major operand
constexpr uint32_t kStageA = kCtaM * kBK * 2;
// Output leaves through shared memory in boxes of 32 rows x 128 bytes, two for
// each epilogue warp.
constexpr uint32_t kBoxBytes = 32 * 128;
constexpr uint32_t kBoxRegion = 4 * 2 * kBoxBytes;
// Labels whose part of dW gets its rounding back: up to kLabelMost of a token, whatever
// the other tokens' labels.  Where a warp's 32 tokens have no more than kNear in all,
// the labels' hidden rows wait in registers.
constexpr int kNear = 4;
constexpr int kLabelMost = 4;
// Of each epilogue warp: a word for each of its tokens, and kNear rows and tokens.
constexpr uint32_t kHitBytes = 4 * (32 + 2 * kNear);
constexpr int kThreads = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
constexpr int kRowGroup = 4096;  // rows whose row blocks share weight tiles in L2
constexpr int kPrepRows = 8;   // rows a prepare block packs at a time, one a warp
constexpr int kPrepBlocks = 8;  // prepare blocks an SM, at most
constexpr int kMaxSplits = 64;
// Units the split of dh may make: with four waves of 148 SMs the last wave costs
// little, and the partial tiles stay within 155 MB (256 x 256; 78 MB of 128 x 256).
constexpr int64_t kSplitUnits = 592;
constexpr int kMinSlices = 8;

// A CTA pair (cluster of two, tcgen05.mma.cta_group::2) computes 256 x 256
// tiles: each CTA stages its own 128 rows of A and half of B, so operands cross
// from L2 into shared memory at two thirds of the rate that a 128 x 256 tile by
// one CTA needs, and each CTA keeps two accumulators in TMEM.
template <bool kPair>
constexpr int kTileM = kPair ? 256 : 128;
template <bool kPair>
constexpr uint32_t kStageB = (kPair ? 128 : 256) * kBK * 2;
template <bool kPair>
constexpr uint32_t kStageBytes = kStageA + kStageB<kPair>;
template <bool kPair>
constexpr int kStages = kPair ? 6 : 4;
template <bool kPair>
constexpr size_t kSmemBytes =
    kStages<kPair> * size_t{kStageBytes<kPair>} + kBoxRegion + 4 * kHitBytes + 1024 + 512;
static_assert(kSmemBytes<true> <= 227 * 1024 && kSmemBytes<false> <= 227 * 1024,
              "shared memory of one CTA");

// Where an epilogue of kDweight finds the hidden rows of its tokens' labels.
enum Labels { kNone, kClose, kFar };

enum Mode {
  kLoss,     // A = hidden rows, B = weight rows: (max, sum of exp) a row and tile, label logits
  kDlogits,  // the same product: d, 16 bits
  kDhidden,  // A = d, B = weight (K = vocabulary, N contiguous): partial sums of dh
  kDweight   // A = d^T, B = hidden (K = rows, both with M / N contiguous): dW
};

struct Params {
  const int* count;     // [0] kept rows, [2] K splits of dh
  int64_t hidden;       // H
  int64_t cols;         // vocabulary columns of this piece
  int64_t col0;         // first of them
  const int* labels;    // packed rows: label, lse, coefficients
  const float* lse;
  const float* ca;
  const float* cb;
  const uint32_t* top;  // bits of the largest finite |coefficient| (fp16), or NULL
  float2* records;      // [tiles][rec_stride]
  float* label_logit;   // [rec_stride]
  int64_t rec_stride;
  float* rest;          // what rounding took from d at the label, packed rows
  const void* packed;   // kDweight: the packed hidden rows
  int accumulate;       // kDhidden: add to the partial sums of the pieces before
  uint32_t* status;
};

// Power of two that brings the largest finite coefficient to [2^12, 2^13) (fp16 d).
__device__ __forceinline__ float coef_scale(const uint32_t* top) {
  if (top == nullptr) return 1.0f;
  const float m = __uint_as_float(*top);
  if (!(m > 0.0f) || !(m < INFINITY)) return 1.0f;
  int e = 12 - ilogbf(m);
  e = e > 120 ? 120 : (e < -120 ? -120 : e);
  return __int_as_float((e + 127) << 23);
}

// The unit grid of one launch, the same for every role of the kernel.
struct Grid {
  int64_t mt, nt, splits, units, kslices;
};

// K splits of dh: the number that makes the slowest worker's share of slices
// smallest, the lowest of equals.  A unit costs its slices and about kUnitCost
// slices of epilogue, and a part has kMinSlices at least.  The count is fixed by a
// whole piece's slices, so that every piece adds to the same partial tiles.  The lanes of a warp weigh 32 numbers each
// round (one thread alone took 7 us over them).
__device__ inline int dh_splits(int64_t tiles, int kslices, int workers, int lane) {
  constexpr int kUnitCost = 8;
  unsigned best = 0xffffffffu;  // cost << 7 | splits; lane 0 always weighs one
  if (tiles > kSplitUnits / 2) return 1;
  const int t = static_cast<int>(tiles);
  for (int s = lane + 1; s <= kMaxSplits; s += 32) {
    if (s > 1 && (t * s > kSplitUnits || s * kMinSlices > kslices)) continue;
    const int waves = (t * s + workers - 1) / workers;
    const int64_t cost = static_cast<int64_t>(waves) * ((kslices + s - 1) / s + kUnitCost);
    const unsigned key =
        (static_cast<unsigned>(cost < (1 << 24) ? cost : (1 << 24) - 1) << 7) | static_cast<unsigned>(s);
    best = key < best ? key : best;
  }
  return static_cast<int>(__reduce_min_sync(0xffffffffu, best) & 127u);
}

__device__ __forceinline__ Grid make_grid(Mode mode, const Params& p, int n, int tile_m) {
  Grid g;
  const int64_t rows = n > 0 ? n : 1;  // one block of zero rows writes zero gradients
  if (mode == kLoss || mode == kDlogits) {
    g.mt = (rows + tile_m - 1) / tile_m;
    g.nt = (p.cols + kBN - 1) / kBN;
    g.kslices = (p.hidden + kBK - 1) / kBK;
    g.splits = 1;
  } else if (mode == kDhidden) {
    g.mt = (rows + tile_m - 1) / tile_m;
    g.nt = (p.hidden + kBN - 1) / kBN;
    g.kslices = (p.cols + kBK - 1) / kBK;
    g.splits = p.count[2];
  } else {
    g.mt = (p.cols + tile_m - 1) / tile_m;
    g.nt = (p.hidden + kBN - 1) / kBN;
    g.kslices = (rows + kBK - 1) / kBK;
    g.splits = 1;
  }
  g.units = g.mt * g.nt * g.splits;
  return g;
}

struct Unit {
  int64_t m, n, split, k0, k1;  // tile coordinates, K slices [k0, k1)
};

__device__ __forceinline__ Unit unit_at(Mode mode, const Grid& g, int64_t u, int tile_m) {
  Unit x;
  if (mode == kLoss || mode == kDlogits) {
    // groups of row blocks; inside one, the row blocks of a weight tile run next
    // to each other
    const int64_t blocks = kRowGroup / tile_m;
    const int64_t per = blocks * g.nt;
    const int64_t gi = u / per, first = gi * blocks;
    const int64_t in = g.mt - first < blocks ? g.mt - first : blocks;
    const int64_t local = u - gi * per;
    x.m = first + local % in;
    x.n = local / in;
    x.split = 0;
  } else {
    const int64_t tiles = g.mt * g.nt;
    x.split = u / tiles;
    const int64_t t = u - x.split * tiles;
    x.m = t / g.nt;
    x.n = t - x.m * g.nt;
  }
  const int64_t each = (g.kslices + g.splits - 1) / g.splits;
  x.k0 = x.split * each;
  x.k1 = x.k0 + each < g.kslices ? x.k0 + each : g.kslices;
  if (x.k1 < x.k0) x.k1 = x.k0;
  return x;
}

// Shared-memory descriptor of an MN-major operand in 64 x 64 blocks, each 64 K
// rows of 128 bytes (64 M or N elements) in the 128-byte swizzle: 8-row atoms
// 1024 bytes apart along K (stride byte offset), blocks kBlockBytes apart along
// M or N (leading byte offset).
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3fffu) |
         (static_cast<uint64_t>(kBlockBytes >> 4) << 16) | (uint64_t{1024 >> 4} << 32) |
         (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

// Operands with M / N contiguous in memory (the others have K contiguous).
template <Mode kMode>
constexpr bool kAMn = kMode == kDweight;
template <Mode kMode>
constexpr bool kBMn = kMode == kDweight || kMode == kDhidden;

// Instruction descriptor of kind::f16: D f32, A and B of type T (0 fp16, 1
// bf16), bit 15 / 16: A / B with M / N contiguous, N >> 3 at 17, M >> 4 at 24.
template <typename T, Mode kMode, bool kPair>
__device__ __forceinline__ uint32_t idesc() {
  constexpr uint32_t t = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((kAMn<kMode> ? 1u : 0u) << 15) |
         ((kBMn<kMode> ? 1u : 0u) << 16) | (uint32_t(kBN >> 3) << 17) |
         (uint32_t(kTileM<kPair> >> 4) << 24);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename T>
__device__ __forceinline__ float round16(float x) {
  if (std::is_same<T, __nv_bfloat16>::value) return __bfloat162float(__float2bfloat16_rn(x));
  return __half2float(__float2half_rn(x));
}

__device__ __forceinline__ float2 pair_of(__nv_bfloat16, uint32_t u) {
  return make_float2(bf16_bits_lo(u), bf16_bits_hi(u));
}
__device__ __forceinline__ float2 pair_of(__half, uint32_t u) {
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

// ---- cluster and pair forms of the wrappers ----

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

// The shared::cluster address of `addr` (this CTA's shared memory) in CTA `rank`.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A load into this CTA's shared memory that counts on a barrier of the pair.
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, int32_t x,
                                              int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

template <bool kPair>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t desc,
                                    uint32_t accumulate) {
  if (kPair)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(desc), "r"(accumulate)
        : "memory");
  else
    umma_f16(d, a, b, desc, accumulate);
}

// Arrives on `bar`, in both CTAs of a pair, once the MMAs issued so far are done.
template <bool kPair>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (kPair)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        " [%0], %1;" ::"r"(smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    umma_commit(bar);
}

// A box from shared memory to the matrix of `map`, or added to it (f32); a group
// of its own either way, so that waits count boxes.
__device__ __forceinline__ void box_out(const CUtensorMap* map, int32_t x, int32_t y,
                                        uint32_t box, bool inside, bool add) {
  if (!inside) {
  } else if (add)
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group"
                 " [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(box)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group"
                 " [%0, {%1, %2}], [%3];" ::"l"(reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(box)
                 : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// ---------------------------------------------------------------------------
// The product kernel: persistent, warp-specialised, one CTA or one pair a tile
// ---------------------------------------------------------------------------
//
// In a pair, both CTAs load, and read back their half of the rows; the leader
// (rank 0) counts both CTAs' loads on its `full` barriers and issues the MMAs,
// whose commits arrive in both.
//
// Bound by the tensor cores and, at one to four waves of tiles, by the last wave:
// 2867 kept rows x 128256 x 4096 run loss, d, dh and dW at 1541, 1547, 1447
// and 1575 TFLOP/s one at a time (1270 to 1300 together, under the power cap);
// 512 x 32000 x 2048 take 54.6, 58, 52 and 63.9 us (tensor pipe 63, 59, 66, 53 %; of
// dW's few slices a tile the epilogue takes longer than the products).  Up to 128 rows
// it is bound by memory: 24 x 128256 x 4096, 1.05 GB a launch, 176, 188, 154 and 244 us.

template <typename T, Mode kMode, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                     const __grid_constant__ CUtensorMap map_b,
                     const __grid_constant__ CUtensorMap map_out, Params p) {
  constexpr int kS = kStages<kPair>;
  constexpr int kTM = kTileM<kPair>;
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  unsigned char* stage_a = smem;
  unsigned char* stage_b = smem + kS * kStageA;
  unsigned char* boxes = smem + kS * kStageBytes<kPair>;
  unsigned char* hits = boxes + kBoxRegion;
  uint64_t* full = reinterpret_cast<uint64_t*>(hits + 4 * kHitBytes);
  uint64_t* empty = full + kS;
  uint64_t* acc_full = empty + kS;
  uint64_t* acc_empty = acc_full + kAccBufs;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kAccBufs);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = kPair ? cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kS; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < kAccBufs; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], kPair ? 8 : 4);
    }
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // A pair takes its tensor memory as a pair: both CTAs have to be running before either
  // asks.  Beside another stream's kernels one can start well before the other.
  __syncthreads();
  if (kPair) cluster_sync();
  if (warp == 1) {
    if (kPair) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(tmem_slot)),
                   "r"(kTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                       smem_u32(tmem_slot)),
                   "r"(kTmemCols)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  __syncthreads();
  if (kPair) cluster_sync();  // the peer has its tensor memory
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  // every kernel of a call is a programmatic dependent of the one before: set-up
  // overlaps its tail, global memory waits for its end
  pdl_trigger();
  pdl_wait();
  const int n = *p.count;
  const Grid g = make_grid(kMode, p, n, kTM);
  const int64_t ksteps = (n > 0 ? n + kUmmaK - 1 : kUmmaK) / kUmmaK;  // of kDweight
  const int64_t first = kPair ? blockIdx.x >> 1 : blockIdx.x;
  const int64_t stride = kPair ? gridDim.x >> 1 : gridDim.x;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      int s = 0;
      uint32_t ph = 0, issued = 0, issue_par = 0;
      bool ok = true;
      for (int64_t u = first; ok && u < g.units; u += stride) {
        const Unit x = unit_at(kMode, g, u, kTM);
        const int32_t m0 = static_cast<int32_t>(x.m * kTM + rank * kCtaM);
        const int32_t n0 = static_cast<int32_t>(x.n * kBN + rank * 128);
        for (int64_t k = x.k0; k < x.k1; ++k) {
          if (!mbar_wait(&empty[s], ph ^ 1u, abort, kWaitNs)) {
            if (!*abort) raise_abort(abort, p.status);
            ok = false;
            break;
          }
          uint32_t bar = smem_u32(&full[s]);
          if (rank == 0) mbar_expect_tx(&full[s], (kPair ? 2 : 1) * kStageBytes<kPair>);
          if (kPair) bar = map_rank(bar, 0);
          auto load = [&](void* dst, const CUtensorMap* map, int32_t cx, int32_t cy) {
            if (kPair)
              tma_load_pair(dst, map, cx, cy, bar);
            else
              tma_load_2d(dst, map, cx, cy, &full[s]);
          };
          unsigned char* a = stage_a + s * kStageA;
          unsigned char* b = stage_b + s * kStageB<kPair>;
          const int32_t kx = static_cast<int32_t>(k * kBK);
          if (kAMn<kMode>) {
            for (int i = 0; i < 2; ++i) load(a + i * kBlockBytes, &map_a, m0 + i * 64, kx);
          } else {
            load(a, &map_a, kx, m0);
          }
          if (kBMn<kMode>) {
            const int32_t row = kx + (kMode == kDhidden ? static_cast<int32_t>(p.col0) : 0);
            for (int i = 0; i < (kPair ? 2 : 4); ++i)
              load(b + i * kBlockBytes, &map_b, n0 + i * 64, row);
          } else {
            for (int i = 0; i < (kPair ? 1 : 2); ++i)
              load(b + i * (128 * kBK * 2), &map_b, kx,
                   static_cast<int32_t>(p.col0) + n0 + i * 128);
          }
          issued |= 1u << s;
          issue_par = (issue_par & ~(1u << s)) | (ph << s);
          if (++s == kS) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      // what this CTA loaded has been multiplied, and every arrival of the MMAs'
      // commits on these barriers has landed, before the CTA exits
      for (int i = 0; i < kS; ++i)
        if (issued & (1u << i)) mbar_wait(&empty[i], (issue_par >> i) & 1u, nullptr, kDrainNs);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // ---------------- MMA issuer ----------------
      // The whole warp runs the loop and an elected lane issues: operands stay in
      // uniform registers, which keeps an MMA's issue short of its run time.
      int s = 0, buf = 0;
      uint32_t ph = 0, aph = 0;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        bool got = true;
        if (lane == 0) {
          got = mbar_wait(bar, parity, abort, kWaitNs);
          if (!got && !*abort) raise_abort(abort, p.status);
        }
        return __shfl_sync(0xffffffffu, static_cast<int>(got), 0) != 0;
      };
      for (int64_t u = first; ok && u < g.units; u += stride) {
        const Unit x = unit_at(kMode, g, u, kTM);
        if (!wait(&acc_empty[buf], aph ^ 1u)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(buf * kBN);
        for (int64_t k = x.k0; k < x.k1; ++k) {
          if (!wait(&full[s], ph)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(stage_a + s * kStageA);
          const uint32_t b0 = smem_u32(stage_b + s * kStageB<kPair>);
          // K advance: 32 bytes inside a K-major row, two 8-row atoms otherwise
          // (the address field counts 16 bytes)
          const uint64_t ad = kAMn<kMode> ? mn_desc(a0) : sw128_desc(a0);
          const uint64_t bd = kBMn<kMode> ? mn_desc(b0) : sw128_desc(b0);
          // rows past the last step of kDweight are not zero: they are not multiplied
          const int64_t left = kMode == kDweight ? ksteps - k * (kBK / kUmmaK) : kBK / kUmmaK;
          const uint32_t more = k > x.k0 ? 1u : 0u;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < kBK / kUmmaK; ++kk) {
              if (kk >= left) break;
              mma<kPair>(d, ad + kk * (kAMn<kMode> ? 128 : 2), bd + kk * (kBMn<kMode> ? 128 : 2),
                         idesc<T, kMode, kPair>(), kk > 0 ? 1u : more);
            }
            commit<kPair>(&empty[s]);
          }
          __syncwarp();
          if (++s == kS) {
            s = 0;
            ph ^= 1u;
          }
        }
        if (!ok) break;
        if (elect_one()) commit<kPair>(&acc_full[buf]);
        __syncwarp();
        last_bar = &acc_full[buf];
        last_par = aph;
        if (++buf == kAccBufs) {
          buf = 0;
          aph ^= 1u;
        }
      }
      // MMAs in flight finish before the TMEM is freed (immediate unless aborted)
      if (lane == 0 && last_bar != nullptr) mbar_wait(last_bar, last_par, nullptr, kDrainNs);
      __syncwarp();
    }
  } else {
    // ---------------- epilogue: thread = tile row, TMEM lane = tile row ----------------
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const float scale = coef_scale(p.top), inv = 1.0f / scale;
    const uint32_t box0 = smem_u32(boxes) + static_cast<uint32_t>(quarter) * (2 * kBoxBytes);
    uint32_t box = 0;  // the next of the warp's two boxes
    int buf = 0;
    uint32_t aph = 0;
    unsigned* seen = reinterpret_cast<unsigned*>(hits + quarter * kHitBytes);  // [32]
    int* mine = reinterpret_cast<int*>(seen + 32);                             // [kNear]
    int* tokens = mine + kNear;                                                // [kNear]
    if (kMode == kDweight) seen[lane] = 0;
    // the first 128 labels (the array is padded to as many)
    const int4 labels0 = kMode == kDweight ? reinterpret_cast<const int4*>(p.labels)[lane]
                                           : make_int4(-1, -1, -1, -1);
    for (int64_t u = first; u < g.units; u += stride) {
      const Unit x = unit_at(kMode, g, u, kTM);
      const int64_t row0 = x.m * kTM + rank * kCtaM;  // the CTA's first row
      const int64_t row = row0 + r;
      const bool valid = row < (kMode == kDweight ? p.cols : n);
      int label = -1;
      float lse2 = 0.0f, ca = 0.0f, cb = 0.0f;
      float top = -INFINITY, sum = 0.0f;
      if ((kMode == kLoss || kMode == kDlogits) && valid) {
        label = p.labels[row];
        if (kMode == kDlogits) {
          lse2 = p.lse[row] * kLog2e;
          ca = p.ca[row] * scale;
          cb = p.cb[row] * scale;
        }
      }
      // dW's rows of labels: the label's element of d is b (1 - p) large, and what its
      // rounding took is added back below, b times 2^-9 of a hidden row.  The warp looks
      // for its 32 tokens among the labels, and each lane keeps those of its own token
      // in ascending order, so that sums have one order.  A token with more than
      // kLabelMost keeps its elements' roundings and is looked for no further, so that a
      // frequent label takes nothing from its neighbours.
      const int token0 = static_cast<int>(p.col0 + row0) + quarter * 32;
      int found = 0, own_count = 0, own_slot[kLabelMost] = {};  // of all tokens, of the lane's
      if (kMode == kDweight) {
        __syncwarp();
        unsigned many = 0;  // tokens with more than kLabelMost
        for (int i0 = 0; i0 < n; i0 += 128) {
          const int i = i0 + lane * 4;
          const int4 y = i0 == 0 ? labels0 : *reinterpret_cast<const int4*>(p.labels + i);
          const int rel[4] = {y.x - token0, y.y - token0, y.z - token0, y.w - token0};
          unsigned own = 0;  // bits of this lane's four
#pragma unroll
          for (int k = 0; k < 4; ++k)
            own |= (static_cast<unsigned>(rel[k]) < 32u && i + k < n ? 1u : 0u) << k;
          if (!__any_sync(0xffffffffu, own != 0)) continue;
          if (many != 0) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((many >> (rel[k] & 31) & 1u) != 0) own &= ~(1u << k);
          }
          found = 1;
          // the lanes whose k-th label is this lane's token, by way of the token's word
          unsigned by[4], left_over = 0;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            by[k] = 0;
            if (!__any_sync(0xffffffffu, (own >> k & 1u) != 0)) continue;
            if ((own >> k & 1u) != 0) atomicOr(&seen[rel[k]], 1u << lane);
            __syncwarp();
            by[k] = seen[lane];
            seen[lane] = 0;
            left_over |= by[k];
            __syncwarp();
          }
          while (left_over != 0 && own_count <= kLabelMost) {
            const int from = __ffs(static_cast<int>(left_over)) - 1;
            left_over &= left_over - 1;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if ((by[k] >> from & 1u) != 0) {
#pragma unroll
                for (int e = 0; e < kLabelMost; ++e)
                  if (own_count == e) own_slot[e] = i0 + from * 4 + k;
                ++own_count;
              }
          }
          many = __ballot_sync(0xffffffffu, own_count > kLabelMost);
        }
        if (found != 0)
          found = static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(own_count)));
        if (found != 0 && found <= kNear) {
          int at = 0;
#pragma unroll
          for (int e = 0; e < kNear; ++e)
            at += __popc(__ballot_sync(0xffffffffu, own_count > e) & ((1u << lane) - 1u));
#pragma unroll
          for (int e = 0; e < kLabelMost; ++e)
            if (e < own_count) {
              mine[at + e] = own_slot[e];
              tokens[at + e] = lane;
            }
        }
        __syncwarp();
        if (own_count > kLabelMost) own_count = 0;
      }
      // Few labels: the tile's columns of their hidden rows, eight a lane, asked for
      // here, while the product runs, and handed around below.  More of them: each lane
      // reads the rows of its own token's as it comes to them.  (Read
      // one label after another by the whole warp, a backward of 512 rows x 4096 x 512
      // took 73 us, and of 64 rows with labels among 32 tokens 252; so 50 and 46.)
      uint4 seg[kNear];
      float left[kNear];
      int who[kNear];
      if (kMode == kDweight) {
#pragma unroll
        for (int e = 0; e < kNear; ++e) {
          seg[e] = make_uint4(0, 0, 0, 0);
          left[e] = 0.0f;
          who[e] = -1;
          if (e < found && found <= kNear) {
            const int slot = mine[e];
            const int64_t col = x.n * kBN + lane * 8;
            if (col < p.hidden)
              seg[e] = static_cast<const uint4*>(p.packed)[slot * (p.hidden / 8) + col / 8];
            left[e] = p.rest[slot];
            who[e] = tokens[e];
          }
        }
      }
      bool got = mbar_wait(&acc_full[buf], aph, abort, kWaitNs);
      got = __all_sync(0xffffffffu, got);
      if (!got) {
        if (lane == 0 && !*abort) raise_abort(abort, p.status);
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>(buf * kBN);
      const int64_t width = kMode == kLoss || kMode == kDlogits ? p.cols : p.hidden;
      const bool empty_split = kMode == kDhidden && x.k0 == x.k1;  // no product: zeros
      // d is written to the tile's end, zeros past the vocabulary
      const int64_t rest_cols = width - x.n * kBN;
      const int cols = kMode == kDlogits || rest_cols > kBN ? kBN : static_cast<int>(rest_cols);
      auto columns = [&](int c, auto corrected) {  // 32 of them
        const int64_t c0 = x.n * kBN + c;  // column of the output tile's matrix
        // the lane's next label: its hidden row's columns and what rounding took
        int next[kLabelMost], ahead = own_count;
#pragma unroll
        for (int e = 0; e < kLabelMost; ++e) next[e] = own_slot[e];
        uint4 far[4] = {};
        float far_by = 0.0f;
        bool fetched = false;
        auto fetch = [&] {
          fetched = ahead != 0;
          if (!fetched) return;
          const int slot = next[0];
#pragma unroll
          for (int e = 0; e + 1 < kLabelMost; ++e) next[e] = next[e + 1];
          --ahead;
          const uint4* h = static_cast<const uint4*>(p.packed) + slot * (p.hidden / 8) + c0 / 8;
          far_by = p.rest[slot];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (c0 + 8 * q < width) far[q] = h[q];
        };
        if constexpr (corrected.value == kFar) {
          fetch();
          __syncwarp();
        }
        uint32_t t[32];
        tmem_issue32(taddr + static_cast<uint32_t>(c), t);
        tmem_wait32(t);
        float v[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = empty_split ? 0.0f : __uint_as_float(t[j]);
        if (kMode == kLoss) {
          if (c0 + 32 > width) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c0 + j >= width) v[j] = -INFINITY;
          }
          const int64_t rel = label - p.col0 - c0;
          if (rel >= 0 && rel < 32) {
            float at = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == rel) at = v[j];
            p.label_logit[row] = at;
          }
          float cm = v[0];
#pragma unroll
          for (int j = 1; j < 32; ++j) cm = fmaxf(cm, v[j]);
          if (cm > top) {
            sum = top == -INFINITY ? (sum != sum ? sum : 0.0f) : sum * ex2((top - cm) * kLog2e);
            top = cm;
          }
          // a chunk of -inf alone adds nothing; NaN and +inf make the sum NaN
          const float off = top == -INFINITY ? 0.0f : -top * kLog2e;
          float a0 = 0.0f, a1 = 0.0f, b0 = 0.0f, b1 = 0.0f;
#pragma unroll
          for (int j = 0; j < 32; j += 4) {
            float x0, x1, x2, x3;
            fma2(x0, x1, v[j], v[j + 1], kLog2e, off);
            fma2(x2, x3, v[j + 2], v[j + 3], kLog2e, off);
            add2(a0, a1, ex2(x0), ex2(x1));
            add2(b0, b1, ex2(x2), ex2(x3));
          }
          sum += (a0 + a1) + (b0 + b1);
          return;
        }
        if (kMode == kDlogits) {
          const int64_t rel = label - p.col0 - c0;
#pragma unroll
          for (int j = 0; j < 32; ++j) {
            float q = ca * ex2(fmaf(v[j], kLog2e, -lse2));
            if (j == rel) q -= cb;
            v[j] = valid && c0 + j < width ? q : 0.0f;
          }
          if (valid && rel >= 0 && rel < 32) {
            float at = 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (j == rel) at = v[j];
            p.rest[row] = at - round16<T>(at);
          }
        } else if (kMode == kDweight) {
          if constexpr (corrected.value != kNone) {
            auto add = [&](float by, int q, uint32_t u0, uint32_t u1, uint32_t u2, uint32_t u3) {
              const uint32_t u[4] = {u0, u1, u2, u3};
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 f = pair_of(T{}, u[j]);
                v[8 * q + 2 * j] = fmaf(by, f.x, v[8 * q + 2 * j]);
                v[8 * q + 2 * j + 1] = fmaf(by, f.y, v[8 * q + 2 * j + 1]);
              }
            };
#pragma unroll
            for (int e = 0; e < (corrected.value == kClose ? kNear : 0); ++e) {
              if (e >= found) break;
              const float by = who[e] == lane ? left[e] : 0.0f;
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int from = c / 8 + q;
                add(by, q, __shfl_sync(0xffffffffu, seg[e].x, from),
                    __shfl_sync(0xffffffffu, seg[e].y, from),
                    __shfl_sync(0xffffffffu, seg[e].z, from),
                    __shfl_sync(0xffffffffu, seg[e].w, from));
              }
            }
            while (corrected.value == kFar && fetched) {
#pragma unroll
              for (int q = 0; q < 4; ++q) add(far_by, q, far[q].x, far[q].y, far[q].z, far[q].w);
              fetch();
            }
            __syncwarp();
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] *= inv;
        }
        // into the warp's box: 16-byte pieces of a row in the 128-byte swizzle
        constexpr bool wide = kMode == kDhidden;  // f32: 32 columns a box; 16 bits: 64
        const bool opens = wide || (c & 32) == 0;
        if (opens) {  // the store that read this box two boxes ago is done with it
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
          __syncwarp();
        }
        const uint32_t dst = box0 + box * kBoxBytes + static_cast<uint32_t>(lane) * 128;
#pragma unroll
        for (int j = 0; j < (wide ? 8 : 4); ++j) {
          const uint32_t piece = wide ? j : (c & 32 ? 4 : 0) + j;
          const uint32_t to = dst + ((piece ^ (lane & 7u)) << 4);
          uint32_t o[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            o[e] = wide ? __float_as_uint(v[4 * j + e]) : pack2<T>(v[(8 * j + 2 * e) & 31], v[(8 * j + 2 * e + 1) & 31]);
          asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(to), "r"(o[0]), "r"(o[1]),
                       "r"(o[2]), "r"(o[3])
                       : "memory");
        }
        const bool closes = wide || (c & 32) != 0 || (kMode != kDlogits && c0 + 32 >= width);
        if (closes) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            // columns past the matrix are clipped, boxes past its rows not issued
            int64_t oy = row0 + quarter * 32, ox = c0;
            if (kMode == kDhidden) {
              oy = ((x.split * g.mt + x.m) * g.nt + x.n) * kTM + rank * kCtaM + quarter * 32;
              ox = c;
            } else {
              ox = c0 - (c & 32);
              if (kMode == kDweight) oy += p.col0;
            }
            box_out(&map_out, static_cast<int32_t>(ox), static_cast<int32_t>(oy),
                    box0 + box * kBoxBytes,
                    kMode != kDweight || row0 + quarter * 32 < p.cols,
                    kMode == kDhidden && p.accumulate);
          }
          box ^= 1u;
        }
      };
      // the loop without labels stays short: of few rows, dW is bound by it
      if (kMode != kDweight || found == 0) {
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) columns(c, std::integral_constant<int, kNone>{});
      } else if (found <= kNear) {
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) columns(c, std::integral_constant<int, kClose>{});
      } else {
#pragma unroll 1
        for (int c = 0; c < cols; c += 32) columns(c, std::integral_constant<int, kFar>{});
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kPair)
          arrive_at(map_rank(smem_u32(&acc_empty[buf]), 0));
        else
          mbar_arrive(&acc_empty[buf]);
      }
      if (++buf == kAccBufs) {
        buf = 0;
        aph ^= 1u;
      }
      if (kMode == kLoss && valid) p.records[x.n * p.rec_stride + row] = make_float2(top, sum);
    }
    if (kMode != kLoss && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }

  __syncthreads();
  if (kPair) cluster_sync();  // no arrival or load for this CTA is under way
  if (warp == 1) {
    tc_fence_after();
    if (kPair)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "r"(kTmemCols)
                   : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                   "r"(kTmemCols)
                   : "memory");
  }
  // A pair gives its tensor memory back as a pair: neither CTA leaves its SM to another
  // kernel's while the other's deallocation is under way.
  if (kPair) cluster_sync();
}

// ---------------------------------------------------------------------------
// Packing the kept rows
// ---------------------------------------------------------------------------

constexpr int kIgnored = -1;  // slot of a row without a label
constexpr int kBadLabel = -2;  // slot of a row whose label is no token

struct PrepParams {
  const uint4* hidden;     // [rows][vecs]
  int64_t rows, vecs;      // vecs = H / 8
  const int64_t* labels;
  int64_t ignore, vocab;
  const float* lse;        // per row (backward), or NULL
  const float* grad_loss;  // per row, or NULL for zero
  const float* grad_lse;
  uint4* packed;           // [padded rows][vecs]
  int* slot_of;            // [rows]
  int* plabel;             // packed
  float* plse;
  float* pa;
  float* pb;
  uint32_t* top;           // fp16 backward: bits of the largest finite |coefficient|
  int* count;              // [0] kept rows, [2] K splits of dh
  int piece_slices, tile_m, workers;  // K slices of a whole piece of dh, rows of a tile, CTAs or pairs
  uint32_t* status;
};

// One block packs kPrepRows rows at a time: it counts the kept rows before its own
// (reading their labels, 8 bytes each from L2), then copies them.  Of many rows a
// block packs several such groups one after the other, so that the labels are
// read by kPrepBlocks blocks an SM at most.
// The last block leaves the count and zeroes the rows up to the next multiple
// of 16, the K step of dW = d^T h.  Bound by latency, 7 to 8 us at 1024 rows and 14 at
// 4096.
__global__ void __launch_bounds__(32 * kPrepRows) head_prepare_kernel(PrepParams p) {
  __shared__ int warp_sum[kPrepRows];
  __shared__ int slots[kPrepRows];
  __shared__ int total;
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t groups = (p.rows + kPrepRows - 1) / kPrepRows;
  const int64_t each = (groups + gridDim.x - 1) / gridDim.x;
  const int64_t g0 = blockIdx.x * each, g1 = g0 + each < groups ? g0 + each : groups;
  if (g0 >= g1) return;
  int before = 0;
  for (int64_t i = threadIdx.x; i < g0 * kPrepRows; i += blockDim.x) {
    const int64_t y = p.labels[i];
    before += (y != p.ignore && y >= 0 && y < p.vocab) ? 1 : 0;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) warp_sum[warp] = before;
  __syncthreads();
  int base = lane < kPrepRows ? warp_sum[lane] : 0;  // kept rows before the group
  base = __reduce_add_sync(0xffffffffu, base);
  for (int64_t g = g0; g < g1; ++g) {
    const int64_t r0 = g * kPrepRows;
    if (warp == 0) {
      const int64_t r = r0 + lane;
      const bool mine = lane < kPrepRows && r < p.rows;
      const int64_t y = mine ? p.labels[r] : p.ignore;
      const bool ignored = y == p.ignore;
      const bool kept = mine && !ignored && y >= 0 && y < p.vocab;
      const unsigned mask = __ballot_sync(0xffffffffu, kept);
      const int slot =
          kept ? base + __popc(mask & ((1u << lane) - 1u)) : (ignored ? kIgnored : kBadLabel);
      if (mine) {
        p.slot_of[r] = slot;
        if (slot == kBadLabel && p.status) atomicOr(p.status, CID_STATUS_TOKEN_ID_OUT_OF_RANGE);
      }
      if (kept) {
        p.plabel[slot] = static_cast<int>(y);
        if (p.lse != nullptr) {
          const float gl = p.grad_loss ? p.grad_loss[r] : 0.0f;
          const float ge = p.grad_lse ? p.grad_lse[r] : 0.0f;
          p.plse[slot] = p.lse[r];
          p.pa[slot] = gl + ge;
          p.pb[slot] = gl;
          // one that is not finite spoils its own row and dW, not the scale of the others
          const float most = fmaxf(fabsf(gl + ge), fabsf(gl));
          if (p.top && most < INFINITY) atomicMax(p.top, __float_as_uint(most));
        }
      }
      if (lane < kPrepRows) slots[lane] = mine ? slot : kIgnored;
      if (lane == 0) total = base + __popc(mask);
    }
    __syncthreads();
    // the block's kept rows, piece by piece: eight loads of a thread in flight
    constexpr int kFlight = 8;
    const uint32_t vecs = static_cast<uint32_t>(p.vecs), units = kPrepRows * vecs;
    for (uint32_t i0 = threadIdx.x; i0 < units; i0 += kFlight * blockDim.x) {
      uint4 v[kFlight];
      int to[kFlight];
#pragma unroll
      for (int j = 0; j < kFlight; ++j) {
        const uint32_t i = i0 + j * blockDim.x;
        to[j] = i < units ? slots[i / vecs] : kIgnored;
        if (to[j] >= 0) v[j] = p.hidden[r0 * p.vecs + i];
      }
#pragma unroll
      for (int j = 0; j < kFlight; ++j)
        if (to[j] >= 0) p.packed[to[j] * p.vecs + (i0 + j * blockDim.x) % vecs] = v[j];
    }
    base = total;
    __syncthreads();  // slots and total are free for the next group
  }
  if (g1 == groups) {
    const int n = base;
    const int64_t pad = n > 0 ? (static_cast<int64_t>(n) + 15) / 16 * 16 : 16;
    for (int64_t i = n * p.vecs + threadIdx.x; i < pad * p.vecs; i += blockDim.x)
      p.packed[i] = make_uint4(0, 0, 0, 0);
    if (warp == 0) {
      const int64_t mt = ((n > 0 ? n : 1) + p.tile_m - 1) / p.tile_m;
      const int64_t nt = (p.vecs * 8 + kBN - 1) / kBN;
      const int splits = dh_splits(mt * nt, p.piece_slices, p.workers, lane);
      if (lane == 0) {
        p.count[0] = n;
        p.count[2] = splits;
      }
    }
  }
}

// loss and log-sum-exp of 32 rows a block from the tiles' (max, sum of exp), the
// tiles dealt to kLossParts warps: 7.5 us for 512 rows of 125 tiles, 11 us for 2867
// rows of 501.  The sums' merges chain, so more warps a row, not more bytes, count.
constexpr int kLossParts = 32;

__global__ void __launch_bounds__(32 * kLossParts)
    head_loss_kernel(const float2* records, int64_t tiles, int64_t rec_stride,
                     const float* label_logit, const int* slot_of, int64_t rows, float* loss,
                     float* lse) {
  __shared__ float sm[kLossParts][32], ss[kLossParts][32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, part = threadIdx.x >> 5;
  const int64_t r = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int slot = r < rows ? slot_of[r] : kIgnored;
  float m = -INFINITY, s = 0.0f;
  auto merge = [&](float om, float os) {
    const float nm = fmaxf(m, om);
    // the difference first: a side that keeps its maximum keeps its sum exactly;
    // an empty side has s = 0 and m = -inf
    if (nm == -INFINITY)
      s += os;
    else
      s = s * ex2((m - nm) * kLog2e) + os * ex2((om - nm) * kLog2e);
    m = nm;
  };
  if (slot >= 0)
    for (int64_t t = part; t < tiles; t += 4 * kLossParts) {
      float2 q[4];  // four loads in flight
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[i] = t + i * kLossParts < tiles ? records[(t + i * kLossParts) * rec_stride + slot]
                                          : make_float2(-INFINITY, 0.0f);
#pragma unroll
      for (int i = 0; i < 4; ++i) merge(q[i].x, q[i].y);
    }
  sm[part][lane] = m;
  ss[part][lane] = s;
  __syncthreads();
  if (part == 0 && r < rows) {
    for (int i = 1; i < kLossParts; ++i) merge(sm[i][lane], ss[i][lane]);
    if (slot >= 0) {
      const float l = m + logf(s);
      lse[r] = l;
      loss[r] = l - label_logit[slot];
    } else {
      const float q = slot == kIgnored ? 0.0f : __int_as_float(0x7fffffff);
      lse[r] = q;
      loss[r] = q;
    }
  }
}

// dh of every row: the splits' partial sums in ascending order, and what rounding
// took from d at the label times the label's weight row (d is largest there, and
// its rounding is most of what the sum would be off by); 16 bits.  Zero for an
// ignored row, NaN for a label that is no token.  Bound by memory and latency: 12 us
// for 1024 rows x 2048, 35 us for 4096 x 4096.
template <typename T>
__global__ void __launch_bounds__(256)
    head_dhidden_kernel(const float* partial, const int* slot_of, const int* plabel,
                        const float* rest, const uint4* weight, const int* count,
                        int64_t hidden, int tile_m, const uint32_t* top, T* out) {
  pdl_trigger();
  pdl_wait();
  const int64_t r = blockIdx.x;
  const int slot = slot_of[r];
  const int64_t n = *count;
  const int64_t mt = ((n > 0 ? n : 1) + tile_m - 1) / tile_m, nt = (hidden + kBN - 1) / kBN;
  const int splits = count[2];
  const float inv = 1.0f / coef_scale(top);
  const float left = slot >= 0 ? rest[slot] : 0.0f;
  const uint4* own = weight + (slot >= 0 ? plabel[slot] : 0) * (hidden / 8);
  for (int64_t c = threadIdx.x * 8; c < hidden; c += blockDim.x * 8) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = slot == kBadLabel ? __int_as_float(0x7fffffff) : 0.0f;
    if (slot >= 0) {
      const int64_t tile = (slot / tile_m) * nt + c / kBN, size = tile_m * kBN;
      const float* q = partial + tile * size + (slot % tile_m) * kBN + c % kBN;
#pragma unroll 4
      for (int s = 0; s < splits; ++s, q += mt * nt * size) {
        const float4 x = reinterpret_cast<const float4*>(q)[0];
        const float4 y = reinterpret_cast<const float4*>(q)[1];
        v[0] += x.x;
        v[1] += x.y;
        v[2] += x.z;
        v[3] += x.w;
        v[4] += y.x;
        v[5] += y.y;
        v[6] += y.z;
        v[7] += y.w;
      }
      if (left != 0.0f) {
        const uint4 w = own[c / 8];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = pair_of(T{}, u[j]);
          v[2 * j] = fmaf(left, f.x, v[2 * j]);
          v[2 * j + 1] = fmaf(left, f.y, v[2 * j + 1]);
        }
      }
    }
    uint4 o;
    o.x = pack2<T>(v[0] * inv, v[1] * inv);
    o.y = pack2<T>(v[2] * inv, v[3] * inv);
    o.z = pack2<T>(v[4] * inv, v[5] * inv);
    o.w = pack2<T>(v[6] * inv, v[7] * inv);
    *reinterpret_cast<uint4*>(out + r * hidden + c) = o;
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxLossRows = INT32_MAX - 512;

int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// Rows above which a pair computes a tile: at most 128 rows fill half a pair's
// tile, and then memory is what counts.
bool use_pair(int64_t rows) { return rows > kCtaM; }

int64_t padded_rows(int64_t rows) { return round_up(rows, use_pair(rows) ? 256 : 128); }

// Vocabulary columns of a piece of the backward.  A piece costs three launches,
// each with a last wave that leaves SMs idle; a small one keeps d in L2 between
// them.  Backward measured with d of 64 / 128 / 256 MB and whole: 7.65 / 7.12 /
// 7.21 / 6.97 ms at 2867 kept rows x 128256 x 4096, 5.27 / 4.66 / 4.24 / 4.17 ms at
// 8192 x 32000 x 4096: 256 MB, and no fewer than 4096 columns.
int64_t piece_cols(int64_t rows, int64_t vocab) {
  constexpr int64_t kPieceBytes = 256 << 20;
  int64_t c = kPieceBytes / (2 * padded_rows(rows)) / kBN * kBN;
  if (c < 4096) c = 4096;
  const int64_t all = round_up(vocab, kBN);
  return c < all ? c : all;
}

// Partial tiles of dh: what dh_splits makes of up to `tiles` tiles (fewer rows may be
// kept) and a piece's K slices, at most.
int64_t partial_tiles(int64_t tiles, int64_t slices) {
  int64_t splits = slices / kMinSlices;
  splits = splits < 1 ? 1 : (splits > kMaxSplits ? kMaxSplits : splits);
  const int64_t most = tiles * splits < kSplitUnits ? tiles * splits : kSplitUnits;
  return tiles > most ? tiles : most;
}

// Byte offsets of the workspace's parts.
struct Layout {
  size_t count, slot_of, plabel, plse, pa, pb, label_logit, rest, packed, records, d, partial, bytes;
  int64_t partial_rows;
};

Layout layout(int64_t rows, int64_t hidden, int64_t vocab, bool backward) {
  Layout l = {};
  size_t at = 0;
  auto take = [&](int64_t bytes) {
    const size_t here = at;
    at += static_cast<size_t>(round_up(bytes, 1024));
    return here;
  };
  const int64_t padded = padded_rows(rows), tile_m = use_pair(rows) ? 256 : 128;
  l.count = take(16);  // count, top, splits
  l.slot_of = take(rows * 4);
  l.plabel = take(padded * 4);
  l.packed = take(padded * hidden * 2);
  if (!backward) {
    l.label_logit = take(padded * 4);
    l.records = take((vocab + kBN - 1) / kBN * padded * 8);
  } else {
    l.plse = take(padded * 4);
    l.pa = take(padded * 4);
    l.pb = take(padded * 4);
    l.rest = take(padded * 4);
    l.d = take(padded * piece_cols(rows, vocab) * 2);
    const int64_t tiles = padded / tile_m * ((hidden + kBN - 1) / kBN);
    l.partial_rows = partial_tiles(tiles, piece_cols(rows, vocab) / kBK) * tile_m;
    l.partial = take(l.partial_rows * kBN * 4);
  }
  l.bytes = at;
  return l;
}

bool loss_extents_ok(int64_t rows, int64_t hidden, int64_t vocab) {
  int64_t n = 0, tiles = 0;
  if (!(rows >= 0 && rows <= kMaxLossRows && hidden > 0 && hidden % 8 == 0 &&
        hidden <= INT32_MAX / 2 && vocab > 0 && vocab <= INT32_MAX - kBN &&
        count_ok(rows, hidden, &n) && n <= kMaxCount && count_ok(vocab, hidden, &n) &&
        n <= kMaxCount && count_ok((vocab + kBN - 1) / kBN, rows, &n) && n <= kMaxCount))
    return false;
  // rows of the partial tiles of dh: a tensor map's extent
  tiles = (rows + 127) / 128 * ((hidden + kBN - 1) / kBN);
  return tiles <= INT32_MAX / 512;
}

template <typename T, Mode kMode, bool kPair>
int launch_gemm(const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& out,
                const Params& p, int64_t units, cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(head_gemm_kernel<T, kMode, kPair>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(kSmemBytes<kPair>));
  if (e != cudaSuccess) return record_cuda_error(e);
  const int64_t workers = kPair ? sm_count() / 2 : sm_count();
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((units < workers ? units : workers) * (kPair ? 2 : 1)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes<kPair>;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kPair ? 2 : 1;
  return record_cuda_error(
      cudaLaunchKernelEx(&cfg, head_gemm_kernel<T, kMode, kPair>, a, b, out, p));
}

// 2-D f32 map of the partial tiles, boxes of 32 x 32.
int make_partial_map(CUtensorMap* map, void* base, int64_t rows) {
  auto encode = tensor_map_encoder();
  if (encode == nullptr) return record_cuda_error(cudaErrorNotSupported);
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(kBN), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(kBN) * 4};
  cuuint32_t box[2] = {32, 32};
  cuuint32_t estr[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, base, dims, strides, box, estr,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? CID_OK
             : CID_ERR_INVALID_ARGUMENT;
}

struct Call {
  cid_dtype_t dtype;
  const void* hidden;
  int64_t rows, dim;
  const void* weight;
  int64_t vocab;
  const int64_t* labels;
  int64_t ignore;
  unsigned char* ws;
  uint32_t* status;
  cudaStream_t stream;
};

int launch_prepare(const Call& c, const Layout& l, const float* lse, const float* grad_loss,
                   const float* grad_lse, bool scaled) {
  PrepParams q = {};
  q.hidden = static_cast<const uint4*>(c.hidden);
  q.rows = c.rows;
  q.vecs = c.dim / 8;
  q.labels = c.labels;
  q.ignore = c.ignore;
  q.vocab = c.vocab;
  q.lse = lse;
  q.grad_loss = grad_loss;
  q.grad_lse = grad_lse;
  q.packed = reinterpret_cast<uint4*>(c.ws + l.packed);
  q.slot_of = reinterpret_cast<int*>(c.ws + l.slot_of);
  q.plabel = reinterpret_cast<int*>(c.ws + l.plabel);
  q.plse = reinterpret_cast<float*>(c.ws + l.plse);
  q.pa = reinterpret_cast<float*>(c.ws + l.pa);
  q.pb = reinterpret_cast<float*>(c.ws + l.pb);
  q.count = reinterpret_cast<int*>(c.ws + l.count);
  q.piece_slices = static_cast<int>(piece_cols(c.rows, c.vocab) / kBK);
  q.tile_m = use_pair(c.rows) ? 256 : 128;
  q.workers = use_pair(c.rows) ? sm_count() / 2 : sm_count();
  q.status = c.status;
  if (scaled) {
    q.top = reinterpret_cast<uint32_t*>(c.ws + l.count) + 1;
    const cudaError_t e = cudaMemsetAsync(q.top, 0, 4, c.stream);
    if (e != cudaSuccess) return record_cuda_error(e);
  }
  int64_t blocks = (c.rows + kPrepRows - 1) / kPrepRows;
  if (blocks > int64_t{kPrepBlocks} * sm_count()) blocks = int64_t{kPrepBlocks} * sm_count();
  return launch_pdl(head_prepare_kernel, dim3(static_cast<unsigned>(blocks)),
                    dim3(32 * kPrepRows), 0, c.stream, q);
}

template <typename T, bool kPair>
int run_loss(const Call& c, float* loss, float* lse) {
  const Layout l = layout(c.rows, c.dim, c.vocab, false);
  const int64_t padded = padded_rows(c.rows);
  int rc = launch_prepare(c, l, nullptr, nullptr, nullptr, false);
  if (rc != CID_OK) return rc;
  CUtensorMap map_a, map_b;
  rc = make_map_sw128(&map_a, c.dtype, c.ws + l.packed, c.dim, padded, c.dim, kBK, 128);
  if (rc == CID_OK)
    rc = make_map_sw128(&map_b, c.dtype, c.weight, c.dim, c.vocab, c.dim, kBK, 128);
  if (rc != CID_OK) return rc;
  Params p = {};
  p.count = reinterpret_cast<const int*>(c.ws + l.count);
  p.hidden = c.dim;
  p.cols = c.vocab;
  p.labels = reinterpret_cast<const int*>(c.ws + l.plabel);
  p.records = reinterpret_cast<float2*>(c.ws + l.records);
  p.label_logit = reinterpret_cast<float*>(c.ws + l.label_logit);
  p.rec_stride = padded;
  p.status = c.status;
  const int64_t tiles = (c.vocab + kBN - 1) / kBN;
  rc = launch_gemm<T, kLoss, kPair>(map_a, map_b, map_a, p, padded / kTileM<kPair> * tiles,
                                    c.stream);
  if (rc != CID_OK) return rc;
  return launch_pdl(head_loss_kernel, dim3(static_cast<unsigned>((c.rows + 31) / 32)),
                    dim3(32 * kLossParts), 0, c.stream, static_cast<const float2*>(p.records),
                    tiles, padded, static_cast<const float*>(p.label_logit),
                    reinterpret_cast<const int*>(c.ws + l.slot_of), c.rows, loss, lse);
}

template <typename T, bool kPair>
int run_backward(const Call& c, const float* lse, const float* grad_loss, const float* grad_lse,
                 void* grad_hidden, void* grad_weight) {
  const Layout l = layout(c.rows, c.dim, c.vocab, true);
  const int64_t padded = padded_rows(c.rows);
  const int64_t piece = piece_cols(c.rows, c.vocab);
  const bool scaled = c.dtype == CID_DTYPE_F16;
  int rc = launch_prepare(c, l, lse, grad_loss, grad_lse, scaled);
  if (rc != CID_OK) return rc;
  unsigned char* d = c.ws + l.d;
  CUtensorMap h_k, h_mn, w_k, w_mn, d_k, d_mn, d_out, dw_out, dh_out;
  auto map = [&](CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int box) {
    if (rc == CID_OK) rc = make_map_sw128(m, c.dtype, base, inner, outer, inner, 64, box);
  };
  map(&h_k, c.ws + l.packed, c.dim, padded, 128);
  map(&h_mn, c.ws + l.packed, c.dim, padded, kBK);
  map(&w_k, c.weight, c.dim, c.vocab, 128);
  map(&w_mn, c.weight, c.dim, c.vocab, kBK);
  map(&d_k, d, piece, padded, 128);
  map(&d_mn, d, piece, padded, kBK);
  map(&d_out, d, piece, padded, 32);
  if (grad_weight != nullptr) map(&dw_out, grad_weight, c.dim, c.vocab, 32);
  if (rc == CID_OK) rc = make_partial_map(&dh_out, c.ws + l.partial, l.partial_rows);
  if (rc != CID_OK) return rc;
  Params p = {};
  p.count = reinterpret_cast<const int*>(c.ws + l.count);
  p.hidden = c.dim;
  p.labels = reinterpret_cast<const int*>(c.ws + l.plabel);
  p.lse = reinterpret_cast<const float*>(c.ws + l.plse);
  p.ca = reinterpret_cast<const float*>(c.ws + l.pa);
  p.cb = reinterpret_cast<const float*>(c.ws + l.pb);
  p.top = scaled ? reinterpret_cast<const uint32_t*>(c.ws + l.count) + 1 : nullptr;
  p.rest = reinterpret_cast<float*>(c.ws + l.rest);
  p.packed = c.ws + l.packed;
  p.status = c.status;
  constexpr int kTM = kTileM<kPair>;
  const int64_t mt = padded / kTM, ht = (c.dim + kBN - 1) / kBN;
  for (int64_t c0 = 0; c0 < c.vocab; c0 += piece) {
    p.col0 = c0;
    p.cols = c.vocab - c0 < piece ? c.vocab - c0 : piece;
    p.accumulate = c0 > 0;
    rc = launch_gemm<T, kDlogits, kPair>(h_k, w_k, d_out, p, mt * ((p.cols + kBN - 1) / kBN),
                                         c.stream);
    if (rc == CID_OK && grad_hidden != nullptr)
      rc = launch_gemm<T, kDhidden, kPair>(d_k, w_mn, dh_out, p, INT32_MAX, c.stream);
    if (rc == CID_OK && grad_weight != nullptr)
      rc = launch_gemm<T, kDweight, kPair>(d_mn, h_mn, dw_out, p, (p.cols + kTM - 1) / kTM * ht,
                                           c.stream);
    if (rc != CID_OK) return rc;
  }
  if (grad_hidden == nullptr) return CID_OK;
  return launch_pdl(head_dhidden_kernel<T>, dim3(static_cast<unsigned>(c.rows)), dim3(256), 0,
                    c.stream, reinterpret_cast<const float*>(c.ws + l.partial),
                    reinterpret_cast<const int*>(c.ws + l.slot_of), p.labels,
                    static_cast<const float*>(p.rest), static_cast<const uint4*>(c.weight),
                    p.count, c.dim, kTM, p.top,
                    static_cast<T*>(grad_hidden));
}

template <typename T>
int run_loss(const Call& c, float* loss, float* lse) {
  return use_pair(c.rows) ? run_loss<T, true>(c, loss, lse) : run_loss<T, false>(c, loss, lse);
}

template <typename T>
int run_backward(const Call& c, const float* lse, const float* grad_loss, const float* grad_lse,
                 void* grad_hidden, void* grad_weight) {
  return use_pair(c.rows)
             ? run_backward<T, true>(c, lse, grad_loss, grad_lse, grad_hidden, grad_weight)
             : run_backward<T, false>(c, lse, grad_loss, grad_lse, grad_hidden, grad_weight);
}

int check_loss(cid_dtype_t dtype, const void* hidden, int64_t rows, int64_t dim,
               const void* weight, int64_t vocab, const int64_t* labels, const void* workspace,
               const uint32_t* status) {
  if (dtype != CID_DTYPE_BF16 && dtype != CID_DTYPE_F16) return CID_ERR_UNSUPPORTED_DTYPE;
  if (!loss_extents_ok(rows, dim, vocab)) return CID_ERR_INVALID_ARGUMENT;
  if (misaligned({{hidden, 16}, {weight, 16}, {labels, 8}, {workspace, 16}, {status, 4}}))
    return CID_ERR_MISALIGNED;
  return CID_OK;
}

}  // namespace
}  // namespace cid

using namespace cid;

extern "C" size_t cid_lm_head_cross_entropy_workspace_bytes(int64_t rows, int64_t hidden_dim,
                                                            int64_t vocab, int backward) {
  if (rows <= 0 || !loss_extents_ok(rows, hidden_dim, vocab)) return 0;
  return layout(rows, hidden_dim, vocab, backward != 0).bytes;
}

extern "C" int cid_lm_head_cross_entropy(cid_dtype_t dtype, const void* hidden, int64_t rows,
                                         int64_t hidden_dim, const void* weight, int64_t vocab,
                                         const int64_t* labels, int64_t ignore_index, float* loss,
                                         float* log_sum_exp, void* workspace,
                                         size_t workspace_bytes, uint32_t* status, void* stream) {
  const int rc =
      check_loss(dtype, hidden, rows, hidden_dim, weight, vocab, labels, workspace, status);
  if (rc != CID_OK) return rc;
  if (misaligned({{loss, 4}, {log_sum_exp, 4}})) return CID_ERR_MISALIGNED;
  if (rows == 0) return CID_OK;
  if (any_null({hidden, weight, labels, loss, log_sum_exp, workspace}))
    return CID_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < cid_lm_head_cross_entropy_workspace_bytes(rows, hidden_dim, vocab, 0))
    return CID_ERR_SCRATCH_LIMIT;
  const Call c{dtype, hidden,       rows,
               hidden_dim, weight,  vocab,
               labels, ignore_index, static_cast<unsigned char*>(workspace),
               status, as_stream(stream)};
  return dtype == CID_DTYPE_F16 ? run_loss<__half>(c, loss, log_sum_exp)
                                : run_loss<__nv_bfloat16>(c, loss, log_sum_exp);
}

extern "C" int cid_lm_head_cross_entropy_backward(
    cid_dtype_t dtype, const void* hidden, int64_t rows, int64_t hidden_dim, const void* weight,
    int64_t vocab, const int64_t* labels, int64_t ignore_index, const float* log_sum_exp,
    const float* grad_loss, const float* grad_log_sum_exp, void* grad_hidden, void* grad_weight,
    void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
  const int rc =
      check_loss(dtype, hidden, rows, hidden_dim, weight, vocab, labels, workspace, status);
  if (rc != CID_OK) return rc;
  if (misaligned({{log_sum_exp, 4},
                  {grad_loss, 4},
                  {grad_log_sum_exp, 4},
                  {grad_hidden, 16},
                  {grad_weight, 16}}))
    return CID_ERR_MISALIGNED;
  if (grad_hidden == nullptr && grad_weight == nullptr) return CID_OK;
  if (rows == 0) {
    if (grad_weight == nullptr) return CID_OK;
    return record_cuda_error(cudaMemsetAsync(
        grad_weight, 0, static_cast<size_t>(vocab) * hidden_dim * 2, as_stream(stream)));
  }
  if (any_null({hidden, weight, labels, log_sum_exp, workspace})) return CID_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < cid_lm_head_cross_entropy_workspace_bytes(rows, hidden_dim, vocab, 1))
    return CID_ERR_SCRATCH_LIMIT;
  const Call c{dtype, hidden,       rows,
               hidden_dim, weight,  vocab,
               labels, ignore_index, static_cast<unsigned char*>(workspace),
               status, as_stream(stream)};
  return dtype == CID_DTYPE_F16
             ? run_backward<__half>(c, log_sum_exp, grad_loss, grad_log_sum_exp, grad_hidden,
                                    grad_weight)
             : run_backward<__nv_bfloat16>(c, log_sum_exp, grad_loss, grad_log_sum_exp,
                                           grad_hidden, grad_weight);
}
