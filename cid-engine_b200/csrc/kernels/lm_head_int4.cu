// The LM head with a weight of 4 bits: each group of `group` (32, 64 or 128)
// consecutive columns of a weight row holds codes q in [-8, 7] and one 16-bit
// scale s, standing for w = s q.
//
//   quantize:   s = round16(max |w| / 7),  q = clamp(rint(w / s), -8, 7)
//   dequantize: round16(s q)
//   products:   z_nv = sum_g s_vg (sum_{k in g} q_vk h_nk), f32
//   statistics: max softmax probability, argmax and the current token's
//               probability over z, without writing z
//
// Codes are stored as q + 8, eight to a 32-bit word: column 8 j + 2 i at bits
// 4 i and column 8 j + 2 i + 1 at bits 16 + 4 i of word j.  One shift and one
// masked OR then give a pair of neighbouring columns in the halves of a
// register, with the exponent that makes them 128 + q + 8 (bf16) or 1024 + q + 8
// (fp16); one subtraction leaves q exactly.
//
// Product kernel.  The weight's bytes bound it up to some 64 rows (128256 x
// 4096: 270 MB, 42 us at the copy peak), so every SM streams weight tiles of
// 128 rows with TMA, whatever the number of hidden rows.  The contraction runs
// on the tensor cores with the weight as A: a thread owns one weight row, turns
// 128 of its codes into 64 registers of 16-bit pairs and stores them to TMEM,
// which tcgen05.mma takes as its A operand; hidden rows are B (N = 16 to 64
// columns of the accumulator).  q is exact in 16 bits and the scale is applied
// in f32 to each group's sum when it is read back from TMEM, so nothing is
// rounded between the inputs and the f32 result.  Two warpgroups take turns:
// one's MMAs run while the other unpacks.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace cid {
namespace {

constexpr int kTileV = 128;       // weight rows of a tile: UMMA M, one a thread
constexpr int kChunk = 128;       // columns a warpgroup unpacks at a time
constexpr int kStageK = 256;      // columns of a stage: a chunk for each warpgroup
constexpr int kUmmaK = 16;
constexpr uint32_t kStageW = kTileV * kStageK / 2;  // 16 KiB of codes
constexpr int kChunkCols = kChunk / 2;              // TMEM columns of a chunk of A
constexpr int kMaxStages = 8;
constexpr int kThreads = 384;  // warp 0 TMA, warp 1 MMA, warps 2-3 idle, warps 4-11 two warpgroups
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxParts = 256;  // vocabulary parts of the statistics: record combine limit

struct Int4Params {
  int64_t rows, vocab;
  int64_t groups;       // scales a weight row
  int64_t stages_k;     // stages a tile: ceil(H / kStageK)
  int64_t tiles;        // weight tiles
  int64_t parts;        // vocabulary parts, one a CTA
  int64_t row_blocks;   // blocks of the kernel's N rows
  const void* scales;
  void* out;            // logits [rows][vocab], or NULL
  cid_shard_record_t* records;  // statistics: [parts][rows]
  const int64_t* ids;
  uint32_t* status;
  int round_bf16;
  int stages;           // shared-memory stages
};

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

// Stores 64 registers to 64 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_store64(uint32_t taddr, const uint32_t (&r)[64]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t* q = r + 32 * h;
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
        "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
            taddr + 32 * h),
        "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]), "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7]),
        "r"(q[8]), "r"(q[9]), "r"(q[10]), "r"(q[11]), "r"(q[12]), "r"(q[13]), "r"(q[14]),
        "r"(q[15]), "r"(q[16]), "r"(q[17]), "r"(q[18]), "r"(q[19]), "r"(q[20]), "r"(q[21]),
        "r"(q[22]), "r"(q[23]), "r"(q[24]), "r"(q[25]), "r"(q[26]), "r"(q[27]), "r"(q[28]),
        "r"(q[29]), "r"(q[30]), "r"(q[31])
        : "memory");
  }
}

__device__ __forceinline__ void tmem_wait_store() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 16 consecutive f32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// D[tmem] (+)= A[tmem] * B[shared], K = 16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

// The four pairs of columns of a word of codes as 16-bit pairs.
template <typename T>
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t* out) {
  constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t magic = bf ? 0x43004300u : 0x64006400u;  // 128 or 1024 in both halves
  constexpr uint32_t bias = bf ? 0x43084308u : 0x64086408u;   // 136 or 1032
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = ((w >> (4 * i)) & 0x000f000fu) | magic;
    if (bf) {
      const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&t),
                                       *reinterpret_cast<const __nv_bfloat162*>(&bias));
      out[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&t),
                                *reinterpret_cast<const __half2*>(&bias));
      out[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
  }
}

// Running statistics of one hidden row over the columns a lane has seen.
struct LaneState {
  float m, s;
  int where, nan;
};

__device__ __forceinline__ void lane_merge(LaneState& a, float m, float s, int where, int nan) {
  if (m > a.m || (m == a.m && where >= 0 && (a.where < 0 || where < a.where))) a.where = where;
  const float nm = fmaxf(a.m, m);
  const float off = nm == -INFINITY ? 0.0f : nm * kLog2e;
  a.s = a.s * ex2(fmaf(a.m, kLog2e, -off)) + s * ex2(fmaf(m, kLog2e, -off));
  a.m = nm;
  if (nan >= 0 && (a.nan < 0 || nan < a.nan)) a.nan = nan;
}

// N: hidden rows of a pass (accumulator columns); S: groups in a chunk of 128
// columns, each with an accumulator of its own.
template <typename T, int N, int S>
__global__ void __launch_bounds__(kThreads, 1)
    int4_head_kernel(const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_h, Int4Params p) {
  constexpr int kDCols = N * S;
  constexpr int kDBufs = kDCols <= 64 ? 2 : 1;  // accumulators of a warpgroup
  static_assert(kDCols <= 128 && 2 * 2 * kChunkCols + 2 * kDBufs * kDCols <= int(kTmemCols),
                "A chunks and accumulators share TMEM");
  constexpr uint32_t kStageH = N * kStageK * 2;
  constexpr uint32_t kStage = kStageW + kStageH;
  constexpr uint32_t kType = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  constexpr uint32_t kDesc = (1u << 4) | (kType << 7) | (kType << 10) |
                             (uint32_t(N >> 3) << 17) | (uint32_t(kTileV >> 4) << 24);

  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const int stages = p.stages;
  unsigned char* stage0 = smem;
  float* xch = reinterpret_cast<float*>(smem + stages * kStage);  // [N][kTileV]
  uint64_t* full = reinterpret_cast<uint64_t*>(xch + N * kTileV);
  uint64_t* empty = full + kMaxStages;
  uint64_t* a_full = empty + kMaxStages;  // [2 warpgroups][2]
  uint64_t* d_full = a_full + 4;          // [2 warpgroups][2]
  uint64_t* joined = d_full + 4;          // the eight unpacking warps meet
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(joined + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 2 * 4 + 1);  // the unpacking warps' reads and the MMAs'
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&a_full[i], 4);
      mbar_init(&d_full[i], 1);
    }
    mbar_init(joined, 8);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const uint32_t d_base = tmem_base + 4 * kChunkCols;

  const int64_t part = blockIdx.x;
  const int64_t t0 = part * p.tiles / p.parts, t1 = (part + 1) * p.tiles / p.parts;
  const int64_t turns = p.row_blocks * (t1 - t0);  // tiles this CTA runs through

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- TMA producer ----------------
      int s = 0;
      uint32_t ph = 0, issued = 0, issue_par = 0;
      bool ok = true;
      for (int64_t i = 0; ok && i < turns; ++i) {
        const int64_t rb = i / (t1 - t0), t = t0 + i % (t1 - t0);
        for (int64_t k = 0; k < p.stages_k; ++k) {
          if (!mbar_wait(&empty[s], ph ^ 1u, abort, kWaitNs)) {
            if (!*abort) raise_abort(abort, p.status);
            ok = false;
            break;
          }
          mbar_expect_tx(&full[s], kStage);
          unsigned char* w = stage0 + s * kStage;
          tma_load_2d(w, &map_w, static_cast<int32_t>(k * (kStageK / 4)),
                      static_cast<int32_t>(t * kTileV), &full[s]);
          for (int b = 0; b < kStageK / 64; ++b)
            tma_load_2d(w + kStageW + b * (N * 128), &map_h,
                        static_cast<int32_t>(k * kStageK + b * 64), static_cast<int32_t>(rb * N),
                        &full[s]);
          issued |= 1u << s;
          issue_par = (issue_par & ~(1u << s)) | (ph << s);
          if (++s == stages) {
            s = 0;
            ph ^= 1u;
          }
        }
      }
      for (int i = 0; i < stages; ++i)
        if (issued & (1u << i)) mbar_wait(&full[i], (issue_par >> i) & 1u, nullptr, kDrainNs);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- MMA issuer ----------------
      int s = 0;
      uint32_t ph = 0;
      uint64_t* last_bar = nullptr;
      uint32_t last_par = 0;
      bool ok = true;
      int64_t n = 0;  // stages so far: the chunk count of each warpgroup
      for (int64_t i = 0; ok && i < turns * p.stages_k; ++i, ++n) {
        const uint32_t b0 = smem_u32(stage0 + s * kStage + kStageW);
        const int ab = static_cast<int>(n & 1);
        const uint32_t par = static_cast<uint32_t>(n >> 1) & 1u;
        if (!mbar_wait(&full[s], ph, abort, kWaitNs)) {
          if (!*abort) raise_abort(abort, p.status);
          break;
        }
        for (int wg = 0; wg < 2; ++wg) {
          // the codes of this chunk are in TMEM, and the accumulator it will use
          // has been read
          if (!mbar_wait(&a_full[wg * 2 + ab], par, abort, kWaitNs)) {
            if (!*abort) raise_abort(abort, p.status);
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = tmem_base + static_cast<uint32_t>((wg * 2 + ab) * kChunkCols);
          const uint32_t d =
              d_base + static_cast<uint32_t>((wg * kDBufs + (kDBufs == 2 ? ab : 0)) * kDCols);
#pragma unroll
          for (int kk = 0; kk < kChunk / kUmmaK; ++kk) {
            constexpr int per = kChunk / kUmmaK / S;  // MMAs of a group
            const uint64_t bd = sw128_desc(b0 + (wg * 2 + kk / 4) * (N * 128) + (kk % 4) * 32);
            umma_f16_ts(d + (kk / per) * N, a + kk * (kUmmaK / 2), bd, kDesc,
                        kk % per != 0 ? 1u : 0u);
          }
          umma_commit(&d_full[wg * 2 + ab]);
          last_bar = &d_full[wg * 2 + ab];
          last_par = par;
        }
        if (!ok) break;
        umma_commit(&empty[s]);
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (last_bar != nullptr) mbar_wait(last_bar, last_par, nullptr, kDrainNs);
    }
  } else if (warp >= 4) {
    // ---------------- two warpgroups: thread = weight row ----------------
    const int wg = (warp - 4) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const T* scales = static_cast<const T*>(p.scales);
    int s = 0;
    uint32_t ph = 0;
    int64_t n = 0;  // chunks of this warpgroup so far
    bool ok = true;
    constexpr int kOwn = (N + 7) / 8;  // hidden rows whose statistics a warp keeps
    LaneState st[kOwn];
    float cur[kOwn];

    float acc[N];
    // adds the sums of chunk c (stage k of the tile of row v) to acc
    auto drain = [&](int64_t c, const float (&sc)[S]) {
      const int ab = static_cast<int>(c & 1);
      bool got = mbar_wait(&d_full[wg * 2 + ab], static_cast<uint32_t>(c >> 1) & 1u, abort,
                           kWaitNs);
      got = __all_sync(0xffffffffu, got);
      if (!got) {
        if (lane == 0 && !*abort) raise_abort(abort, p.status);
        return false;
      }
      tc_fence_after();
      const uint32_t d = d_base + lane_off +
                         static_cast<uint32_t>((wg * kDBufs + (kDBufs == 2 ? ab : 0)) * kDCols);
#pragma unroll
      for (int g = 0; g < S; ++g)
#pragma unroll
        for (int j = 0; j < N; j += 16) {
          uint32_t x[16];
          tmem_load16(d + static_cast<uint32_t>(g * N + j), x);
#pragma unroll
          for (int q = 0; q < 16; ++q) acc[j + q] = fmaf(__uint_as_float(x[q]), sc[g], acc[j + q]);
        }
      tc_fence_before();
      return true;
    };

    uint32_t join_par = 0;
    auto join = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(joined);
      bool got = mbar_wait(joined, join_par, abort, kWaitNs);
      got = __all_sync(0xffffffffu, got);
      join_par ^= 1u;
      if (!got && lane == 0 && !*abort) raise_abort(abort, p.status);
      return got;
    };

    for (int64_t i = 0; ok && i < turns; ++i) {
      const int64_t rb = i / (t1 - t0), ti = i % (t1 - t0), t = t0 + ti;
      const int64_t v = t * kTileV + r;
      const bool valid = v < p.vocab;
      if (ti == 0) {
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          st[j] = LaneState{-INFINITY, 0.0f, -1, -1};
          cur[j] = 0.0f;
        }
      }
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] = 0.0f;
      float sc_prev[S];
      for (int64_t k = 0; k < p.stages_k; ++k, ++n) {
        float sc[S];
#pragma unroll
        for (int g = 0; g < S; ++g) {
          const int64_t gi = (k * 2 + wg) * S + g;
          sc[g] = valid && gi < p.groups ? to_float(scales[v * p.groups + gi]) : 0.0f;
        }
        bool got = mbar_wait(&full[s], ph, abort, kWaitNs);
        got = __all_sync(0xffffffffu, got);
        if (!got) {
          if (lane == 0 && !*abort) raise_abort(abort, p.status);
          ok = false;
          break;
        }
        const unsigned char* row = stage0 + s * kStage + r * 128;
        uint32_t a[64];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 w =
              *reinterpret_cast<const uint4*>(row + (((wg * 4 + c) ^ (r & 7)) << 4));
          unpack8<T>(w.x, a + c * 16);
          unpack8<T>(w.y, a + c * 16 + 4);
          unpack8<T>(w.z, a + c * 16 + 8);
          unpack8<T>(w.w, a + c * 16 + 12);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
        // A buffer n & 1 was last read by the MMAs of chunk n - 2, whose sums
        // have been drained; with one accumulator chunk n - 1's must be too
        if (kDBufs == 1 && k > 0 && !drain(n - 1, sc_prev)) {
          ok = false;
          break;
        }
        tmem_store64(tmem_base + lane_off + static_cast<uint32_t>((wg * 2 + (n & 1)) * kChunkCols),
                     a);
        tmem_wait_store();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&a_full[wg * 2 + (n & 1)]);
        if (kDBufs == 2 && k > 0 && !drain(n - 1, sc_prev)) {
          ok = false;
          break;
        }
#pragma unroll
        for (int g = 0; g < S; ++g) sc_prev[g] = sc[g];
      }
      if (!ok || !drain(n - 1, sc_prev)) {
        ok = false;
        break;
      }
      // ---- the tile's sums: warpgroup 1's halves join warpgroup 0's ----
      if (wg == 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) xch[j * kTileV + r] = acc[j];
      }
      if (!join()) break;
      const int64_t row0 = rb * N;
      if (wg == 0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
          float z = acc[j] + xch[j * kTileV + r];
          if (p.out != nullptr) {
            if (valid && row0 + j < p.rows) {
              T* o = static_cast<T*>(p.out) + (row0 + j) * p.vocab + v;
              if (std::is_same<T, __nv_bfloat16>::value)
                *reinterpret_cast<__nv_bfloat16*>(o) = __float2bfloat16_rn(z);
              else
                *reinterpret_cast<__half*>(o) = __float2half_rn(z);
            }
          } else {
            if (p.round_bf16) z = __bfloat162float(__float2bfloat16_rn(z));
            xch[j * kTileV + r] = valid ? z : -INFINITY;
          }
        }
      }
      if (!join()) break;
      if (p.out == nullptr) {
        const int w = warp - 4;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          const int nrow = w + j * 8;
          if (nrow >= N || row0 + nrow >= p.rows) break;
          const float4 q = *reinterpret_cast<const float4*>(xch + nrow * kTileV + lane * 4);
          const float x[4] = {q.x, q.y, q.z, q.w};
          const int c0 = static_cast<int>(t * kTileV) + lane * 4;
          const int64_t rel = p.ids[row0 + nrow] - c0;
          float cm = -INFINITY;
          int cw = -1, cn = -1;
#pragma unroll
          for (int e = 3; e >= 0; --e) {
            if (x[e] >= cm && c0 + e < p.vocab) {
              cm = x[e];
              cw = c0 + e;
            }
            if (x[e] != x[e]) cn = c0 + e;
            if (rel == e && c0 + e < p.vocab) cur[j] = x[e];
          }
          const float off = cm == -INFINITY ? 0.0f : cm * kLog2e;
          float cs = 0.0f;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            cs += x[e] == -INFINITY ? 0.0f : ex2(fmaf(x[e], kLog2e, -off));
          lane_merge(st[j], cm, cs, cw, cn);
        }
        if (ti + 1 == t1 - t0) {
          // ---- the part's record of each row ----
#pragma unroll
          for (int j = 0; j < kOwn; ++j) {
            const int nrow = w + j * 8;
            if (nrow >= N || row0 + nrow >= p.rows) break;
            LaneState a = st[j];
            float c = cur[j];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
              const float om = __shfl_xor_sync(0xffffffffu, a.m, d);
              const float os = __shfl_xor_sync(0xffffffffu, a.s, d);
              const int ow = __shfl_xor_sync(0xffffffffu, a.where, d);
              const int on = __shfl_xor_sync(0xffffffffu, a.nan, d);
              const float oc = __shfl_xor_sync(0xffffffffu, c, d);
              lane_merge(a, om, os, ow, on);
              c += oc;  // one lane at most has seen the token
            }
            if (lane == 0) {
              cid_shard_record_t rec;
              rec.max_logit = a.m;
              const bool special = !(a.m > -INFINITY && a.m < INFINITY) || a.s != a.s;
              const int first = static_cast<int>(t0 * kTileV);
              if (special) {
                const int at = a.nan >= 0 ? a.nan : (a.where >= 0 ? a.where : first);
                rec.sum_exp = a.m == -INFINITY ? 0.0f : __int_as_float(0x7fffffff);
                rec.index = at | (a.nan >= 0 ? static_cast<int32_t>(0x80000000u) : 0);
              } else {
                rec.sum_exp = a.s;
                rec.index = a.where;
              }
              rec.current = c;
              p.records[part * p.rows + row0 + nrow] = rec;
            }
          }
        }
      }
      if (!join()) break;  // xch is free
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base),
                 "r"(kTmemCols)
                 : "memory");
  }
}

// ---------------------------------------------------------------------------
// Quantiser
// ---------------------------------------------------------------------------

constexpr int kQuantThreads = 256;

// A lane holds 8 columns (16 bytes) and writes their word; the group's lanes
// (4, 8 or 16) share the maximum.  |w| compares as its bits, NaN above all, so
// a NaN or infinite weight leaves its group's scale NaN or infinite.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_kernel(const uint4* weight, int64_t words, int lanes, uint32_t* packed, T* scales) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kQuantThreads + threadIdx.x;
  // words is a multiple of 4, a group's lanes are in range together
  const uint4 v = i < words ? weight[i] : make_uint4(0, 0, 0, 0);
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) top = max(top, max(u[j] & 0x7fffu, (u[j] >> 16) & 0x7fffu));
  for (int d = 1; d < lanes; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
  if (i >= words) return;
  const uint16_t bits = static_cast<uint16_t>(top);
  const float amax = to_float(*reinterpret_cast<const T*>(&bits));
  T scale;
  if (std::is_same<T, __nv_bfloat16>::value)
    *reinterpret_cast<__nv_bfloat16*>(&scale) = __float2bfloat16_rn(__fdiv_rn(amax, 7.0f));
  else
    *reinterpret_cast<__half*>(&scale) = __float2half_rn(__fdiv_rn(amax, 7.0f));
  const float s = to_float(scale);
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint16_t b = static_cast<uint16_t>(u[j] >> (16 * h));
      float q = 0.0f;
      if (s > 0.0f && s < INFINITY) {
        q = rintf(__fdiv_rn(to_float(*reinterpret_cast<const T*>(&b)), s));
        q = fminf(fmaxf(q, -8.0f), 7.0f);
      }
      word |= static_cast<uint32_t>(static_cast<int>(q) + 8) << (4 * j + 16 * h);
    }
  }
  packed[i] = word;
  if (i % lanes == 0) scales[i / lanes] = scale;
}

template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_kernel(const uint32_t* packed, const T* scales, int64_t words, int lanes,
                      uint4* weight) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kQuantThreads + threadIdx.x;
  if (i >= words) return;
  const uint32_t w = packed[i];
  const float s = to_float(scales[i / lanes]);
  uint32_t u[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float lo = s * static_cast<float>(static_cast<int>((w >> (4 * j)) & 15u) - 8);
    const float hi = s * static_cast<float>(static_cast<int>((w >> (4 * j + 16)) & 15u) - 8);
    if (std::is_same<T, __nv_bfloat16>::value)
      asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(u[j]) : "f"(hi), "f"(lo));
    else
      asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(u[j]) : "f"(hi), "f"(lo));
  }
  weight[i] = make_uint4(u[0], u[1], u[2], u[3]);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxInt4Rows = INT32_MAX - 64;

bool int4_weight_ok(int64_t vocab, int64_t dim, int group) {
  int64_t n = 0;
  return (group == 32 || group == 64 || group == 128) && vocab > 0 &&
         vocab <= INT32_MAX - kTileV && dim > 0 && dim % group == 0 &&
         dim <= INT32_MAX - kStageK && count_ok(vocab, dim, &n) && n <= kMaxCount &&
         n / (8 * kQuantThreads) < INT32_MAX;
}

int64_t int4_parts(int64_t vocab) {
  const int64_t tiles = (vocab + kTileV - 1) / kTileV;
  int64_t parts = sm_count() < kMaxParts ? sm_count() : kMaxParts;
  return tiles < parts ? tiles : parts;
}

template <typename T, int N, int S>
int launch_int4(const CUtensorMap& map_w, const CUtensorMap& map_h, Int4Params p,
                cudaStream_t stream) {
  constexpr size_t stage = kStageW + size_t{N} * kStageK * 2;
  constexpr size_t fixed = size_t{N} * kTileV * 4 + 1024 + 512;
  constexpr size_t fit = (227 * 1024 - fixed) / stage;
  p.stages = static_cast<int>(fit < kMaxStages ? fit : kMaxStages);
  p.row_blocks = (p.rows + N - 1) / N;
  const size_t smem = p.stages * stage + fixed;
  const cudaError_t e =
      cudaFuncSetAttribute(int4_head_kernel<T, N, S>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem));
  if (e != cudaSuccess) return record_cuda_error(e);
  int4_head_kernel<T, N, S>
      <<<static_cast<unsigned>(p.parts), kThreads, smem, stream>>>(map_w, map_h, p);
  return launch_result();
}

// Hidden rows of a pass: the accumulators of a chunk's groups are at most 64
// columns wide, so a group of 128 takes up to 64 rows a pass, one of 64 up to
// 32, one of 32 sixteen; more rows read the weight again.
template <typename T>
int dispatch_int4(cid_dtype_t dtype, const void* hidden, int64_t dim, const void* packed,
                  int group, Int4Params p, cudaStream_t stream) {
  const int most = group / 2;
  const int n = p.rows > 32 && most >= 64 ? 64 : (p.rows > 16 && most >= 32 ? 32 : 16);
  CUtensorMap map_w, map_h;
  // codes copied as 16-bit elements, four columns each
  int rc = make_map_sw128(&map_w, CID_DTYPE_F16, packed, dim / 4, p.vocab, dim / 4, 64, kTileV);
  if (rc == CID_OK) rc = make_map_sw128(&map_h, dtype, hidden, dim, p.rows, dim, 64, n);
  if (rc != CID_OK) return rc;
  p.groups = dim / group;
  p.stages_k = (dim + kStageK - 1) / kStageK;
  p.tiles = (p.vocab + kTileV - 1) / kTileV;
  p.parts = int4_parts(p.vocab);
  switch (group) {
    case 128:
      return n == 64   ? launch_int4<T, 64, 1>(map_w, map_h, p, stream)
             : n == 32 ? launch_int4<T, 32, 1>(map_w, map_h, p, stream)
                       : launch_int4<T, 16, 1>(map_w, map_h, p, stream);
    case 64:
      return n == 32 ? launch_int4<T, 32, 2>(map_w, map_h, p, stream)
                     : launch_int4<T, 16, 2>(map_w, map_h, p, stream);
    default:
      return launch_int4<T, 16, 4>(map_w, map_h, p, stream);
  }
}

// Checks shared by the two products; rows == 0 is left to the caller.
int check_int4(cid_dtype_t dtype, const void* hidden, int64_t rows, int64_t dim,
               const uint32_t* packed, const void* scales, int group, int64_t vocab,
               const uint32_t* status) {
  if (dtype != CID_DTYPE_BF16 && dtype != CID_DTYPE_F16) return CID_ERR_UNSUPPORTED_DTYPE;
  int64_t n = 0;
  if (rows < 0 || rows > kMaxInt4Rows || !int4_weight_ok(vocab, dim, group) ||
      !count_ok(rows, dim, &n) || n > kMaxCount || !count_ok(rows, vocab, &n) || n > kMaxCount)
    return CID_ERR_INVALID_ARGUMENT;
  if (misaligned({{hidden, 16}, {packed, 16}, {scales, 2}, {status, 4}}))
    return CID_ERR_MISALIGNED;
  return CID_OK;
}

}  // namespace
}  // namespace cid

using namespace cid;

extern "C" int cid_lm_head_quantize(cid_dtype_t dtype, const void* weight, int64_t vocab,
                                    int64_t hidden_dim, int group_size, uint32_t* packed,
                                    void* scales, void* stream) {
  if (dtype != CID_DTYPE_BF16 && dtype != CID_DTYPE_F16) return CID_ERR_UNSUPPORTED_DTYPE;
  if (!int4_weight_ok(vocab, hidden_dim, group_size)) return CID_ERR_INVALID_ARGUMENT;
  if (misaligned({{weight, 16}, {packed, 16}, {scales, 2}})) return CID_ERR_MISALIGNED;
  if (any_null({weight, packed, scales})) return CID_ERR_INVALID_ARGUMENT;
  const int64_t words = vocab * (hidden_dim / 8);
  const unsigned blocks = static_cast<unsigned>((words + kQuantThreads - 1) / kQuantThreads);
  const auto* w = static_cast<const uint4*>(weight);
  if (dtype == CID_DTYPE_F16)
    quantize_kernel<__half><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        w, words, group_size / 8, packed, static_cast<__half*>(scales));
  else
    quantize_kernel<__nv_bfloat16><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        w, words, group_size / 8, packed, static_cast<__nv_bfloat16*>(scales));
  return launch_result();
}

extern "C" int cid_lm_head_dequantize(cid_dtype_t dtype, const uint32_t* packed,
                                      const void* scales, int64_t vocab, int64_t hidden_dim,
                                      int group_size, void* weight, void* stream) {
  if (dtype != CID_DTYPE_BF16 && dtype != CID_DTYPE_F16) return CID_ERR_UNSUPPORTED_DTYPE;
  if (!int4_weight_ok(vocab, hidden_dim, group_size)) return CID_ERR_INVALID_ARGUMENT;
  if (misaligned({{weight, 16}, {packed, 16}, {scales, 2}})) return CID_ERR_MISALIGNED;
  if (any_null({weight, packed, scales})) return CID_ERR_INVALID_ARGUMENT;
  const int64_t words = vocab * (hidden_dim / 8);
  const unsigned blocks = static_cast<unsigned>((words + kQuantThreads - 1) / kQuantThreads);
  auto* w = static_cast<uint4*>(weight);
  if (dtype == CID_DTYPE_F16)
    dequantize_kernel<__half><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        packed, static_cast<const __half*>(scales), words, group_size / 8, w);
  else
    dequantize_kernel<__nv_bfloat16><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        packed, static_cast<const __nv_bfloat16*>(scales), words, group_size / 8, w);
  return launch_result();
}

extern "C" int cid_lm_head_quantized_logits(cid_dtype_t dtype, const void* hidden, int64_t rows,
                                            int64_t hidden_dim, const uint32_t* packed,
                                            const void* scales, int group_size, int64_t vocab,
                                            void* logits, uint32_t* status, void* stream) {
  const int rc =
      check_int4(dtype, hidden, rows, hidden_dim, packed, scales, group_size, vocab, status);
  if (rc != CID_OK) return rc;
  if (misaligned({{logits, 2}})) return CID_ERR_MISALIGNED;
  if (rows == 0) return CID_OK;
  if (any_null({hidden, packed, scales, logits})) return CID_ERR_INVALID_ARGUMENT;
  Int4Params p = {};
  p.rows = rows;
  p.vocab = vocab;
  p.scales = scales;
  p.out = logits;
  p.status = status;
  return dtype == CID_DTYPE_F16
             ? dispatch_int4<__half>(dtype, hidden, hidden_dim, packed, group_size, p,
                                     as_stream(stream))
             : dispatch_int4<__nv_bfloat16>(dtype, hidden, hidden_dim, packed, group_size, p,
                                            as_stream(stream));
}

extern "C" size_t cid_lm_head_quantized_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows <= 0 || rows > kMaxInt4Rows || vocab <= 0 || vocab > INT32_MAX - kTileV) return 0;
  const int64_t tiles = (vocab + kTileV - 1) / kTileV;
  return static_cast<size_t>(tiles < kMaxParts ? tiles : kMaxParts) * static_cast<size_t>(rows) *
         sizeof(cid_shard_record_t);
}

extern "C" int cid_lm_head_quantized_display_statistics(
    cid_dtype_t dtype, const void* hidden, int64_t rows, int64_t hidden_dim,
    const uint32_t* packed, const void* scales, int group_size, int64_t vocab,
    const int64_t* token_ids, int round_bf16, float* confidence, int64_t* predicted,
    float* current_confidence, void* workspace, size_t workspace_bytes, uint32_t* status,
    void* stream) {
  int rc = check_int4(dtype, hidden, rows, hidden_dim, packed, scales, group_size, vocab, status);
  if (rc != CID_OK) return rc;
  if (misaligned({{token_ids, 8},
                  {confidence, 4},
                  {predicted, 8},
                  {current_confidence, 4},
                  {workspace, 16}}))
    return CID_ERR_MISALIGNED;
  if (rows == 0) return CID_OK;
  if (any_null({hidden, packed, scales, token_ids, confidence, predicted, current_confidence,
                workspace}))
    return CID_ERR_INVALID_ARGUMENT;
  if (workspace_bytes < cid_lm_head_quantized_workspace_bytes(rows, vocab))
    return CID_ERR_SCRATCH_LIMIT;
  Int4Params p = {};
  p.rows = rows;
  p.vocab = vocab;
  p.scales = scales;
  p.records = static_cast<cid_shard_record_t*>(workspace);
  p.ids = token_ids;
  p.status = status;
  p.round_bf16 = round_bf16 ? 1 : 0;
  rc = dtype == CID_DTYPE_F16
           ? dispatch_int4<__half>(dtype, hidden, hidden_dim, packed, group_size, p,
                                   as_stream(stream))
           : dispatch_int4<__nv_bfloat16>(dtype, hidden, hidden_dim, packed, group_size, p,
                                          as_stream(stream));
  if (rc != CID_OK) return rc;
  // merge the parts of every row (ascending column ranges) into its statistics
  int64_t offsets[kMaxParts + 1];
  const int64_t parts = int4_parts(vocab), tiles = (vocab + kTileV - 1) / kTileV;
  for (int64_t i = 0; i < parts; ++i) offsets[i] = i * tiles / parts * kTileV;
  offsets[parts] = vocab;
  return cid_display_combine_records(static_cast<const cid_shard_record_t*>(workspace),
                                     static_cast<int>(parts), offsets, token_ids, rows,
                                     confidence, predicted, current_confidence, status, stream);
}
