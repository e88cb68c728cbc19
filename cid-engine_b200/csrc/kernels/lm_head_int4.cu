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
// Codes are stored as c = q + 8, eight to a 32-bit word: column 8 j + 2 i at bits
// 4 i and column 8 j + 2 i + 1 at bits 16 + 4 i of word j.  Masked where they
// stand, a word's nibbles 0 and 1 of each half are fp16 numbers as they are:
// c and 16 c times the smallest subnormal 2^-24.  One shift by 8 brings the
// other two there, so eight columns cost five integer instructions.
//
// The MMAs therefore run in fp16 whatever the hidden rows' type: each hidden row
// is first turned into fp16 times a power of two that brings its largest
// value to [2^14, 2^15), with the columns that meet 16 c divided by 16.  A value
// keeps all its bits unless it is below 2^-24 of its row's largest, and then
// loses less than 2^-35 of that largest, far under the f32 sum's own rounding.
// 8 sum h of every group is kept beside and subtracted from the group's sum:
// sum c h - 8 sum h = sum q h, with roundings of 8 sum |h| in f32.
//
// Two product kernels; the weight's bytes bound both up to some 64 rows (128256 x
// 4096: 270 MB, 42 us at the copy peak).
//
// * Up to 8 hidden rows (int4_rows_kernel): every warp multiplies on its own,
//   with mma.sync (16 weight rows x 16 columns times 8 hidden rows).  A thread's
//   16 bytes of codes from memory are its A fragments after masking, since the
//   MMA's columns may be taken in any order that the hidden rows in shared
//   memory follow.  No buffer changes hands between warps until a tile's sums
//   meet, and the legacy tensor path is fast enough for 8 columns.
// * More rows (int4_head_kernel): tcgen05 with the weight as A.  Every SM
//   streams weight tiles with TMA; a thread owns one weight row, masks 128 of
//   its codes into 64 registers and stores them to TMEM, which tcgen05.mma takes
//   as its A operand; hidden rows are B (N = 16 to 64 columns of the
//   accumulator).  The scale is applied in f32 to each group's sum when it is
//   read back from TMEM.  Unpacking, MMAs and read-back are warps of their own,
//   joined by rings of TMEM buffers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "tcgen05.cuh"

namespace cid {
namespace {

constexpr int kTileV = 128;       // weight rows of an accumulator: UMMA M, one a thread
constexpr int kChunk = 128;       // columns of a stage, unpacked by a warpgroup at a time
constexpr int kUmmaK = 16;
constexpr uint32_t kStageW = kTileV * kChunk / 2;   // 8 KiB of codes for 128 weight rows
constexpr int kChunkCols = kChunk / 2;              // TMEM columns of a chunk of A
constexpr int kMaxStages = 16;
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kDRegion = kTmemCols - 4 * kChunkCols;  // columns left for accumulators
constexpr int kMaxParts = 256;  // vocabulary parts of the statistics: record combine limit
constexpr int kXchRows = 32;           // hidden rows that a tile is transposed in at a time
constexpr int kXchMost = kTileV + 8;   // floats between them, at most
constexpr size_t kSmemLimit = 227 * 1024;

struct Int4Params {
  int64_t rows, vocab;
  int64_t groups;      // scales a weight row
  int chunks;          // stages a tile: ceil(H / kChunk)
  int64_t tiles;       // tiles of R * kTileV weight rows
  int64_t parts;       // vocabulary parts, one a CTA
  int64_t row_blocks;  // blocks of the kernel's N rows
  const void* scales;
  const float* sums;       // 8 sum h: [row blocks][groups][N]
  const float* row_scale;  // what undoes a hidden row's power of two: [row blocks][N]
  void* out;                    // logits [rows][vocab], or NULL
  cid_shard_record_t* records;  // statistics: [parts][rows]
  const int64_t* ids;
  uint32_t* status;
  int round_bf16;
  int stages;  // shared-memory stages
};

__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ float2 pair_floats(uint32_t u) {
  if (std::is_same<T, __nv_bfloat16>::value) return make_float2(bf16_bits_lo(u), bf16_bits_hi(u));
  return __half22float2(*reinterpret_cast<const __half2*>(&u));
}

template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  if (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Stores 32 registers to 32 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* q) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,"
      "%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(
          taddr),
      "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]), "r"(q[4]), "r"(q[5]), "r"(q[6]), "r"(q[7]),
      "r"(q[8]), "r"(q[9]), "r"(q[10]), "r"(q[11]), "r"(q[12]), "r"(q[13]), "r"(q[14]),
      "r"(q[15]), "r"(q[16]), "r"(q[17]), "r"(q[18]), "r"(q[19]), "r"(q[20]), "r"(q[21]),
      "r"(q[22]), "r"(q[23]), "r"(q[24]), "r"(q[25]), "r"(q[26]), "r"(q[27]), "r"(q[28]),
      "r"(q[29]), "r"(q[30]), "r"(q[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_store() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 16 consecutive f32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15}, [%16];\n tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// The same of 32 columns.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
  tmem_issue32(taddr, r);
  tmem_wait32(r);
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

// {a0, a1} += ({x0, x1} 2^24 - {s0, s1}) b
__device__ __forceinline__ void group_add2(float& a0, float& a1, uint32_t x0, uint32_t x1,
                                           float s0, float s1, float b) {
  asm("{\n .reg .b64 ra, rx, rb, rs, rk;\n mov.b64 ra, {%0, %1};\n mov.b64 rx, {%2, %3};\n"
      " mov.b64 rs, {%4, %5};\n mov.b64 rb, {%6, %6};\n mov.b64 rk, {%7, %7};\n"
      " fma.rn.f32x2 rx, rx, rk, rs;\n fma.rn.f32x2 ra, rx, rb, ra;\n"
      " mov.b64 {%0, %1}, ra;\n}"
      : "+f"(a0), "+f"(a1)
      : "r"(x0), "r"(x1), "f"(s0), "f"(s1), "f"(b), "f"(16777216.0f));
}

// The four pairs of columns of a word of codes, c 2^-24 and 16 c 2^-24 in fp16.
__device__ __forceinline__ void unpack8(uint32_t w, uint32_t* out) {
  out[0] = w & 0x000f000fu;
  out[1] = w & 0x00f000f0u;
  out[2] = (w >> 8) & 0x000f000fu;
  out[3] = (w >> 8) & 0x00f000f0u;
}

// A logit from the sum over its groups and the hidden row's power of two.  A group
// with an infinite scale has codes of zero, and its part is 0 x inf; but sum c h and
// 8 sum h are rounded apart, and infinity times what is left of them is an infinity of
// either sign as often as NaN.  An infinite sum is therefore NaN.
__device__ __forceinline__ float logit_of(float sum, float row_scale) {
  return fmaf(sum, 0.0f, sum * row_scale);
}

// Running statistics of one hidden row over the columns a thread has seen.
struct RowStats {
  float m, s;
  int where, nan;  // first column of the maximum, first NaN column; -1: none
};

__device__ __forceinline__ void merge_stats(RowStats& a, const RowStats& b) {
  if (b.m > a.m || (b.m == a.m && b.where >= 0 && (a.where < 0 || b.where < a.where)))
    a.where = b.where;
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) {
    a.s += b.s;  // nothing, or NaN
  } else {
    // the difference first: a side that keeps its maximum keeps its sum exactly
    a.s = a.s * ex2((a.m - m) * kLog2e) + b.s * ex2((b.m - m) * kLog2e);
  }
  a.m = m;
  if (b.nan >= 0 && (a.nan < 0 || b.nan < a.nan)) a.nan = b.nan;
}

// The shard record of merged statistics; `first` is the part's first column.
__device__ __forceinline__ cid_shard_record_t record_of(const RowStats& a, float current,
                                                        int first) {
  cid_shard_record_t rec;
  rec.max_logit = a.m;
  if (!(a.m > -INFINITY && a.m < INFINITY) || a.s != a.s) {
    const int at = a.nan >= 0 ? a.nan : (a.where >= 0 ? a.where : first);
    rec.sum_exp = a.m == -INFINITY ? 0.0f : __int_as_float(0x7fffffff);
    rec.index = at | (a.nan >= 0 ? static_cast<int32_t>(0x80000000u) : 0);
  } else {
    rec.sum_exp = a.s;
    rec.index = a.where;
  }
  rec.current = current;
  return rec;
}

// Roles of a CTA: warps 0-3 control (0 codes' TMA, 1 and 2 MMA, 3 hidden rows' TMA), then R warpgroups that read
// the accumulators back, then two that unpack.
__host__ __device__ constexpr int int4_threads(int r) { return 128 * (3 + r); }

// With two row blocks (640 threads, 96 registers each at launch) the read-back warps
// hold 64 accumulators apiece: registers move to them from the others.  The build
// checks that every such kernel has the 96: a launch with fewer would wait for the
// rest for good.  The shares add up to no more than the launch's, and on each SM
// sub-partition (a warp of control, two of read-back, two of unpacking) to 32 x 472 of
// 16384.
constexpr int kLaunchRegs = 96;
constexpr int kCtrlRegs = 40;
constexpr int kReadRegs = 144;
constexpr int kUnpackRegs = 72;
static_assert(128 * kCtrlRegs + 256 * kReadRegs + 256 * kUnpackRegs <=
                  int4_threads(2) * kLaunchRegs,
              "setmaxnreg.inc draws only on the registers the CTA was launched with");

// N: hidden rows of a pass (accumulator columns); S: groups in a chunk of 128
// columns, each with an accumulator of its own; R: blocks of 128 weight rows a
// tile; kResident: the hidden rows stay in shared memory for the whole pass
// (otherwise their slices travel with the codes).
//
// Chunks are numbered q along the CTA's work: for every stage the tile's R row
// blocks.  Unpacking warpgroup q & 1 fills A buffer (q & 1, (q >> 1) & 1), so with
// one row block the warpgroups take turns at the stages, whose number is even then;
// the accumulators form a ring.
//
// No unit is full at 16 rows x 128256 x 4096 (77 us, 272 MB from memory: 43 % of DRAM,
// 10 % of the tensor pipe, 53 % of the issue slots with the polling among them): the
// roles wait for one another.  At 64 rows (147 us with the statistics) the read-back
// of each group's 64 sums a weight row sets the pace.  Three A buffers a warpgroup
// (104 us at 16 rows), four unpacking warpgroups (87) and MMAs issued by the unpacking
// warps (201) were slower.
template <typename T, int N, int S, int R, bool kResident>
__global__ void __launch_bounds__(int4_threads(R), 1)
    int4_head_kernel(const __grid_constant__ CUtensorMap map_w,
                     const __grid_constant__ CUtensorMap map_h, Int4Params p) {
  constexpr int kDCols = N * S;
  constexpr int kDBufs = int(kDRegion) / kDCols < 4 ? int(kDRegion) / kDCols : 4;
  static_assert(kDBufs == 4 || kDBufs == 2, "the accumulator ring is a power of two");
  constexpr uint32_t kHidden = uint32_t(N) * kChunk * 2;  // hidden rows of a stage
  constexpr uint32_t kStage = R * kStageW + (kResident ? 0u : kHidden);
  // D f32, A and B fp16 (0), both K-major, N >> 3 at bit 17, M >> 4 at bit 24
  constexpr uint32_t kDesc =
      (1u << 4) | (uint32_t(N >> 3) << 17) | (uint32_t(kTileV >> 4) << 24);
  constexpr int kXN = N < kXchRows ? N : kXchRows;
  constexpr int kPer = kTileV / kXN;  // threads of a warpgroup that keep one hidden row's statistics
  constexpr int kXchPitch = kTileV + kPer;  // a warp's reads fall on 32 banks

  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  unsigned char* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  const int stages = p.stages;
  unsigned char* stage0 = smem;
  unsigned char* resident = smem + stages * kStage;  // [2 * chunks][N][64] of the hidden rows
  float* xch = reinterpret_cast<float*>(
      resident + (kResident ? size_t(p.chunks) * kHidden : 0));  // [R][kXN][kXchPitch]
  float* sums = xch + R * kXN * kXchPitch;  // [groups][N] of -8 sum h, then [N] row scales
  const int64_t group_slots = static_cast<int64_t>(p.chunks) * S;
  uint64_t* full = reinterpret_cast<uint64_t*>(sums + group_slots * N + N);
  uint64_t* empty = full + kMaxStages;
  uint64_t* a_full = empty + kMaxStages;  // [warpgroup][2]
  uint64_t* a_empty = a_full + 4;
  uint64_t* d_full = a_empty + 4;         // [kDBufs]
  uint64_t* d_empty = d_full + 4;
  uint64_t* h_full = d_empty + 4;
  uint64_t* h_empty = h_full + 1;
  uint64_t* joined = h_empty + 1;         // [R]: a read-back warpgroup's warps meet
  uint64_t* joined_all = joined + 2;      // all of the read-back warps
  uint64_t* mma_done = joined_all + 1;    // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 2);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      // the warps that unpack the stage, and the MMA warps that use its hidden rows
      mbar_init(&empty[s], kResident ? 4 * R : 5 * R);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&a_full[i], 4);
      mbar_init(&a_empty[i], 1);
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 4);
    }
    mbar_init(h_full, 1);
    mbar_init(h_empty, 2);
    for (int i = 0; i < 2; ++i) mbar_init(&mma_done[i], 1);
    for (int i = 0; i < R; ++i) mbar_init(&joined[i], 4);
    mbar_init(joined_all, 4 * R);
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
  const int chunks = p.chunks;

  // A bounded wait of a whole warp; false when it ran out or another role did.
  // One lane polls: thirty-two take turns at the barrier and slow every role.  The
  // others' accesses are issued after the shuffle that waits for it.
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) {
    bool got = true;
    if (lane == 0) {
      got = mbar_wait(bar, parity, abort, kWaitNs);
      if (!got && !*abort) raise_abort(abort, p.status);
    }
    return __shfl_sync(0xffffffffu, static_cast<int>(got), 0) != 0;
  };
  auto thread_wait = [&](uint64_t* bar, uint32_t parity) {
    const bool got = mbar_wait(bar, parity, abort, kWaitNs);
    if (!got && !*abort) raise_abort(abort, p.status);
    return got;
  };

  if (warp < 4) {
    if (R == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kCtrlRegs));
    if (warp == 0) {
      if (lane == 0) {
        // ---------------- TMA producer ----------------
        // codes need no wait for the kernel that prepares the hidden rows: it was
        // launched in stream order, so what it follows, the codes' writer too, is done
        int s = 0;
        uint32_t ph = 0, issued = 0, issue_par = 0;
        bool ok = true, prepared = false;
        for (int64_t rb = 0; ok && rb < p.row_blocks; ++rb) {
          for (int64_t t = t0; ok && t < t1; ++t) {
            for (int k = 0; k < chunks; ++k) {
              if (!thread_wait(&empty[s], ph ^ 1u)) {
                ok = false;
                break;
              }
              mbar_expect_tx(&full[s], kStage);
              unsigned char* w = stage0 + s * kStage;
              for (int r = 0; r < R; ++r)
                tma_load_2d(w + r * kStageW, &map_w, k * (kChunk / 4),
                            static_cast<int32_t>((t * R + r) * kTileV), &full[s]);
              if (!kResident) {
                if (!prepared) pdl_wait();
                prepared = true;
                for (int b = 0; b < kChunk / 64; ++b)
                  tma_load_2d(w + R * kStageW + b * (N * 128), &map_h, k * kChunk + b * 64,
                              static_cast<int32_t>(rb * N), &full[s]);
              }
              issued |= 1u << s;
              issue_par = (issue_par & ~(1u << s)) | (ph << s);
              if (++s == stages) {
                s = 0;
                ph ^= 1u;
              }
            }
          }
        }
        // copies in flight land before the CTA exits (immediate unless aborted)
        for (int i = 0; i < stages; ++i)
          if (issued & (1u << i)) mbar_wait(&full[i], (issue_par >> i) & 1u, nullptr, kDrainNs);
      }
    } else if (warp == 3) {
      if (kResident && lane == 0) {
        // ---------------- resident hidden rows: one load a pass ----------------
        pdl_wait();
        int64_t loads = 0;
        for (int64_t rb = 0; rb < p.row_blocks; ++rb, ++loads) {
          if (rb > 0 && !thread_wait(h_empty, static_cast<uint32_t>(rb - 1) & 1u)) break;
          mbar_expect_tx(h_full, static_cast<uint32_t>(chunks) * kHidden);
          for (int b = 0; b < chunks * (kChunk / 64); ++b)
            tma_load_2d(resident + b * (N * 128), &map_h, b * 64, static_cast<int32_t>(rb * N),
                        h_full);
        }
        if (loads > 0)
          mbar_wait(h_full, static_cast<uint32_t>(loads - 1) & 1u, nullptr, kDrainNs);
      }
    } else if (warp == 1 || warp == 2) {
      // ---------------- MMA issuers: one for each unpacking warpgroup ----------------
      // The whole warp runs the loop, so that addresses and descriptors stay
      // warp-uniform; one lane issues.
      const uint32_t mw = static_cast<uint32_t>(warp) - 1u;
      int s = 0;
      uint32_t ph = 0;
      bool ok = true;
      uint32_t q = mw, turn = 0;  // chunk number (parities need its low bits only), whose stage it is
      for (int64_t rb = 0; ok && rb < p.row_blocks; ++rb) {
        if (kResident && !warp_wait(h_full, static_cast<uint32_t>(rb) & 1u)) break;
        for (int64_t t = t0; ok && t < t1; ++t) {
          for (int k = 0; ok && k < chunks; ++k, turn ^= 1u) {
            if (R == 2 || turn == mw) {
              // the codes reach this role through TMEM; with resident hidden rows a
              // stage is refilled without it and its barrier must not be waited for
              const uint32_t ab = mw * 2 + ((q >> 1) & 1u), db = q % kDBufs;
              if ((!kResident && !warp_wait(&full[s], ph)) ||
                  !warp_wait(&a_full[ab], (q >> 2) & 1u) ||
                  !warp_wait(&d_empty[db], (q / kDBufs & 1u) ^ 1u)) {
                ok = false;
                break;
              }
              tc_fence_after();
              const uint32_t a = tmem_base + ab * kChunkCols, d = d_base + db * kDCols;
              const uint64_t bd = sw128_desc(kResident ? smem_u32(resident + size_t(k) * kHidden)
                                                       : smem_u32(stage0 + s * kStage + R * kStageW));
              if (elect_one()) {
#pragma unroll
                for (int kk = 0; kk < kChunk / kUmmaK; ++kk) {
                  constexpr int per = kChunk / kUmmaK / S;  // MMAs of a group
                  // the descriptor's address field counts 16 bytes
                  umma_f16_ts(d + (kk / per) * N, a + kk * (kUmmaK / 2),
                              bd + (kk / 4) * (N * 128 / 16) + (kk % 4) * 2, kDesc,
                              kk % per != 0 ? 1u : 0u);
                }
                umma_commit(&a_empty[ab]);
                umma_commit(&d_full[db]);
                if (!kResident) umma_commit(&empty[s]);
              }
              __syncwarp();
              q += 2;
            }
            if (++s == stages) {
              s = 0;
              ph ^= 1u;
            }
          }
        }
        if (kResident && ok && elect_one()) umma_commit(h_empty);
      }
      // every arrival of this warp's MMAs lands before the CTA may exit and the
      // TMEM is freed, also those that no one waits for any more
      if (elect_one()) {
        umma_commit(&mma_done[mw]);
        mbar_wait(&mma_done[mw], 0, nullptr, kDrainNs);
      }
      __syncwarp();
    }
  } else if (warp >= 4 + 4 * R) {
    // ---------------- unpacking: thread = weight row ----------------
    if (R == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kUnpackRegs));
    const int wg = (warp - 4 - 4 * R) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    int s = 0;
    uint32_t ph = 0, n = 0;  // n: chunks of this warpgroup so far, q = 2 n + wg
    auto next_stage = [&]() {
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    };
    const int64_t total = p.row_blocks * (t1 - t0) * chunks;
    if (R == 1 && wg == 1) next_stage();
    for (int64_t i = R == 1 ? wg : 0; i < total; i += R == 1 ? 2 : 1, ++n) {
      if (!warp_wait(&full[s], ph)) break;
      // 64 bytes of codes a weight row, in the 64-byte swizzle
      const unsigned char* row = stage0 + s * kStage + (R == 2 ? wg * kStageW : 0) + r * 64;
      uint4 w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        w[j] = *reinterpret_cast<const uint4*>(row + ((j ^ ((r >> 1) & 3)) << 4));
      const uint32_t ab = static_cast<uint32_t>(wg) * 2 + (n & 1u);
      if (!warp_wait(&a_empty[ab], (n >> 1 & 1u) ^ 1u)) break;
      tc_fence_after();
      const uint32_t dst = tmem_base + lane_off + ab * kChunkCols;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        uint32_t a[32];
        unpack8(w[2 * j].x, a);
        unpack8(w[2 * j].y, a + 4);
        unpack8(w[2 * j].z, a + 8);
        unpack8(w[2 * j].w, a + 12);
        unpack8(w[2 * j + 1].x, a + 16);
        unpack8(w[2 * j + 1].y, a + 20);
        unpack8(w[2 * j + 1].z, a + 24);
        unpack8(w[2 * j + 1].w, a + 28);
        tmem_store32(dst + 32 * j, a);
      }
      // The stage is handed back only now that every lane's codes have come in and been
      // used, and its reads are fenced against the refill's writes.  An arrival right
      // after the loads' issue overtook them: they wait their turn behind the read-back's
      // scales, up to 2048 lines for its four warps, about a microsecond, and a refill
      // takes less.  (147 us for 16 rows of groups of 32 then, 149 now; 137 and 141 for 32
      // rows of groups of 64, 77.1 and 77.8 for 16 of 128.)
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tmem_wait_store();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&empty[s]);
        mbar_arrive(&a_full[ab]);
      }
      next_stage();
      if (R == 1) next_stage();
    }
  } else {
    // ---------------- read-back: thread = weight row ----------------
    if (R == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kReadRegs));
    const int wg = (warp - 4) >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint16_t* scales = static_cast<const uint16_t*>(p.scales);
    float* tile_xch = xch + wg * (kXN * kXchPitch);
    constexpr int kParts = N / kXN;            // of the hidden rows, transposed one after another
    const int own = r / kPer, sub = r % kPer;  // this thread's row of a part and share of columns
    uint32_t join_par = 0;
    auto join = [&](uint64_t* bar, uint32_t par) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
      return warp_wait(bar, par);
    };

    // The scales of four chunks are loaded while the four before are used.
    constexpr int kAhead = 4;
    uint16_t next[kAhead * S], now[kAhead * S];
    auto load_scales = [&](int64_t v, int kc) {
#pragma unroll
      for (int i = 0; i < kAhead * S; ++i) {
        const int64_t g = static_cast<int64_t>(kc) * S + i;
        next[i] = v < p.vocab && g < p.groups ? scales[v * p.groups + g] : uint16_t{0};
      }
    };
    auto scale_of = [](uint16_t bits) { return to_float(*reinterpret_cast<const T*>(&bits)); };

    uint32_t q = static_cast<uint32_t>(wg);  // R == 2: every other chunk is this warpgroup's
    uint32_t all_par = 0;
    bool ok = true;
    load_scales((t0 * R + wg) * kTileV + r, 0);
    pdl_wait();
    for (int64_t rb = 0; ok && rb < p.row_blocks; ++rb) {
      const int64_t row0 = rb * N;
      // the group sums and row scales of this pass's hidden rows
      for (int64_t i = threadIdx.x - 128; i < group_slots * N; i += 128 * R)
        sums[i] = i < p.groups * N ? -p.sums[rb * p.groups * N + i] : 0.0f;
      if (threadIdx.x - 128 < N)
        sums[group_slots * N + threadIdx.x - 128] = p.row_scale[row0 + threadIdx.x - 128];
      if (!join(joined_all, all_par)) break;
      all_par ^= 1u;
      RowStats st[kParts];
      float cur[kParts];
      int64_t id[kParts];
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        st[h] = RowStats{-INFINITY, 0.0f, -1, -1};
        cur[h] = 0.0f;
        const int64_t hr = row0 + h * kXN + own;
        id[h] = p.out == nullptr && hr < p.rows ? p.ids[hr] : -1;
      }
      for (int64_t t = t0; ok && t < t1; ++t) {
        const int64_t v0 = (t * R + wg) * kTileV, v = v0 + r;
        float acc[N];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        for (int kc = 0; ok && kc < chunks; kc += kAhead) {
#pragma unroll
          for (int i = 0; i < kAhead * S; ++i) now[i] = next[i];
          if (kc + kAhead < chunks)
            load_scales(v, kc + kAhead);
          else
            load_scales(t + 1 < t1 ? v + R * kTileV : (t0 * R + wg) * kTileV + r, 0);
#pragma unroll
          for (int i = 0; i < kAhead; ++i) {
            if (kc + i >= chunks) break;
            const uint32_t db = q % kDBufs;
            if (!warp_wait(&d_full[db], q / kDBufs & 1u)) {
              ok = false;
              break;
            }
            tc_fence_after();
            const uint32_t d = d_base + lane_off + db * kDCols;
            const float* gs = sums + static_cast<int64_t>(kc + i) * (S * N);
#pragma unroll
            for (int g = 0; g < S; ++g) {
              const float sc = scale_of(now[i * S + g]);
              constexpr int kStep = N < 32 ? N : 32;
#pragma unroll
              for (int j = 0; j < N; j += kStep) {
                uint32_t x[kStep];
                tmem_load(d + g * N + j, x);
#pragma unroll
                for (int e = 0; e < kStep; e += 4) {
                  const float4 h8 = *reinterpret_cast<const float4*>(gs + g * N + j + e);
                  group_add2(acc[j + e], acc[j + e + 1], x[e], x[e + 1], h8.x, h8.y, sc);
                  group_add2(acc[j + e + 2], acc[j + e + 3], x[e + 2], x[e + 3], h8.z, h8.w, sc);
                }
              }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&d_empty[db]);
            q += R;
          }
        }
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = logit_of(acc[j], sums[group_slots * N + j]);
        // ---- the tile's logits: 128 weight rows x N hidden rows ----
        if (p.out != nullptr) {
          if (v < p.vocab) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
              if (row0 + j >= p.rows) break;
              T* o = static_cast<T*>(p.out) + (row0 + j) * p.vocab + v;
              if (std::is_same<T, __nv_bfloat16>::value)
                *reinterpret_cast<__nv_bfloat16*>(o) = __float2bfloat16_rn(acc[j]);
              else
                *reinterpret_cast<__half*>(o) = __float2half_rn(acc[j]);
            }
          }
          continue;
        }
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
#pragma unroll
          for (int j = 0; j < kXN; ++j) {
            float z = acc[h * kXN + j];
            if (p.round_bf16) z = __bfloat162float(__float2bfloat16_rn(z));
            tile_xch[j * kXchPitch + r] = v < p.vocab ? z : -INFINITY;
          }
          if (!join(&joined[wg], join_par)) {
            ok = false;
            break;
          }
          join_par ^= 1u;
          // columns sub, sub + kPer, ... of the tile: the maximum, then the
          // exponentials; where they stand is looked up only when it matters
          const float* x = tile_xch + own * kXchPitch + sub;
          constexpr int kShare = kTileV / kPer;
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 8
          for (int e = 0; e < kShare; ++e) m4[e & 3] = fmaxf(m4[e & 3], x[e * kPer]);
          RowStats b{fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), 0.0f, -1, -1};
          const float off = b.m == -INFINITY ? 0.0f : b.m;
          float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
          for (int e = 0; e < kShare; ++e) s4[e & 3] += ex2((x[e * kPer] - off) * kLog2e);
          b.s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
          const int c0 = static_cast<int>(v0) + sub;
          if (b.m > st[h].m || st[h].where < 0) {
            for (int e = kShare - 1; e >= 0; --e)
              if (x[e * kPer] == b.m && c0 + e * kPer < p.vocab) b.where = c0 + e * kPer;
          }
          if (b.s != b.s) {  // a NaN, or an infinite maximum
            for (int e = kShare - 1; e >= 0; --e)
              if (x[e * kPer] != x[e * kPer]) b.nan = c0 + e * kPer;
          }
          merge_stats(st[h], b);
          const int64_t rel = id[h] - v0;
          if (rel >= 0 && rel < kTileV && rel % kPer == sub) cur[h] = x[rel - sub];
          if (!join(&joined[wg], join_par)) {  // the part may be overwritten
            ok = false;
            break;
          }
          join_par ^= 1u;
        }
      }
      if (!ok) break;
      if (p.out != nullptr) {
        // the next pass's sums wait for every reader of these
        if (!join(joined_all, all_par)) break;
        all_par ^= 1u;
        continue;
      }
      // ---- the part's record of each row: over the row's threads, then the warpgroups ----
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
#pragma unroll
        for (int d = 1; d < kPer; d <<= 1) {
          RowStats o;
          o.m = __shfl_xor_sync(0xffffffffu, st[h].m, d);
          o.s = __shfl_xor_sync(0xffffffffu, st[h].s, d);
          o.where = __shfl_xor_sync(0xffffffffu, st[h].where, d);
          o.nan = __shfl_xor_sync(0xffffffffu, st[h].nan, d);
          merge_stats(st[h], o);
          cur[h] += __shfl_xor_sync(0xffffffffu, cur[h], d);  // one thread at most has seen it
        }
      }
      if (R == 2) {
        float* slots = xch + kXN * kXchPitch;  // the second warpgroup's tile is free
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          float* slot = slots + (h * kXN + own) * 8;
          if (wg == 1 && sub == 0) {
            slot[0] = st[h].m;
            slot[1] = st[h].s;
            slot[2] = __int_as_float(st[h].where);
            slot[3] = __int_as_float(st[h].nan);
            slot[4] = cur[h];
          }
        }
        if (!join(joined_all, all_par)) break;
        all_par ^= 1u;
        if (wg == 0) {
#pragma unroll
          for (int h = 0; h < kParts; ++h) {
            const float* slot = slots + (h * kXN + own) * 8;
            merge_stats(st[h], RowStats{slot[0], slot[1], __float_as_int(slot[2]),
                                        __float_as_int(slot[3])});
            cur[h] += slot[4];
          }
        }
      }
      // the next pass overwrites the slots and sums
      if (!join(joined_all, all_par)) break;
      all_par ^= 1u;
#pragma unroll
      for (int h = 0; h < kParts; ++h) {
        const int64_t hr = row0 + h * kXN + own;
        if (wg == 0 && sub == 0 && hr < p.rows)
          p.records[part * p.rows + hr] =
              record_of(st[h], cur[h], static_cast<int>(t0 * R * kTileV));
      }
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
// Hidden rows in fp16
// ---------------------------------------------------------------------------

// Bits of the largest |value| of eight: |h| compares as its bits, NaN above all.
__device__ __forceinline__ uint32_t top_bits(uint4 v) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) top = max(top, max(u[j] & 0x7fffu, (u[j] >> 16) & 0x7fffu));
  return top;
}

// e that brings a row's largest value to [2^14, 2^15) by 2^e.  A row of zeros or
// one that is not finite keeps its values (the latter's logits are NaN: an
// infinity times a code, less eight times it).
template <typename T>
__device__ __forceinline__ int row_exponent(uint32_t top) {
  const uint16_t bits = static_cast<uint16_t>(top);
  const float most = to_float(*reinterpret_cast<const T*>(&bits));
  const int e = most > 0.0f && most < INFINITY ? 14 - ilogbf(most) : 0;
  return e > 126 ? 126 : e;  // |h| < 2^-112
}

// Eight columns times `up` in fp16, those that meet 16 c (pairs 1 and 3)
// divided by 16; adds what the MMAs will see of them to `sum`.
template <typename T>
__device__ __forceinline__ uint4 scaled_columns(uint4 v, float up, float& sum) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint16_t b0 = static_cast<uint16_t>(u[j]), b1 = static_cast<uint16_t>(u[j] >> 16);
    const float k = j & 1 ? 0.0625f : 1.0f;
    const __half2 h = __floats2half2_rn(to_float(*reinterpret_cast<const T*>(&b0)) * up * k,
                                        to_float(*reinterpret_cast<const T*>(&b1)) * up * k);
    o[j] = *reinterpret_cast<const uint32_t*>(&h);
    const float2 f = __half22float2(h);
    sum += (f.x + f.y) * (j & 1 ? 16.0f : 1.0f);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// ---------------------------------------------------------------------------
// Up to 8 hidden rows
// ---------------------------------------------------------------------------

constexpr int kRowsThreads = 512;
// Warps of a tile: four along its 128 weight rows, four along the columns.
constexpr int kRowWarps = 4;
constexpr int kColWarps = kRowsThreads / 32 / kRowWarps;
constexpr int kRowsTile = 32 * kRowWarps;
constexpr int kRowsN = 8;  // hidden rows: the MMA's columns
// Blocks of codes a thread holds ahead.  Measured at 8 rows x 128256 x 4096 with 2 /
// 3 / 4: groups of 128 70.4 / 66.7 / 64.3 us, of 64 94.8 / 98.9 / 103.0 us.
template <int S>
constexpr int kRowsRing = S == 1 ? 4 : 2;
constexpr int kRowsPad = 64;  // bytes between hidden rows in shared memory, past whole blocks

struct RowsParams {
  const uint32_t* packed;
  const uint16_t* scales;
  const uint4* hidden;  // [rows][words]
  int64_t rows, vocab;
  int words, groups, blocks;  // a weight row's words, groups and blocks of 128 columns
  int64_t tiles, parts;
  void* out;
  cid_shard_record_t* records;
  const int64_t* ids;
  int round_bf16;
};

// Place of 8 columns (unit u of a block of 128) in the order of the fragments: a
// quad's thread t takes word i of its codes as columns `first + 8 t'`, see
// int4_rows_kernel; unit (t, i) goes to 4 i + t.
__device__ __forceinline__ int fragment_place(int u, int lanes) {
  if (lanes == 16) return (u & 3) * 4 + (u >> 2);              // groups of 128
  return ((u >> 3) * 2 + (u & 1)) * 4 + ((u >> 1) & 3);        // of 64
}

// A thread's codes and scales of 32 weight rows x 128 columns: rows g, g + 8,
// g + 16, g + 24 (g = lane / 4), in each four words; the scales are those of row
// g + 8 t (t = lane % 4).
template <int S>
struct CodeBlock {
  uint32_t w[4][4];
  uint16_t scale[S];
};

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                          uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes are read once: no line of them stays in L1.
template <int B>
__device__ __forceinline__ void load_codes(uint32_t* to, const uint32_t* from) {
  static_assert(B == 4 || B == 2, "16 or 8 bytes");
  if (B == 4)
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(to[0]), "=r"(to[1]), "=r"(to[2]), "=r"(to[3])
                 : "l"(from));
  else
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];"
                 : "=r"(to[0]), "=r"(to[1])
                 : "l"(from));
}

// kStats: statistics instead of logits (their state costs registers).
// Bound by the codes' bytes and the instructions that mask them, about evenly:
// 8 rows x 128256 x 4096 in groups of 128 take 62 us (270 MB, 4.4 TB/s), in groups
// of 64 95 us; 1 row x 32000 x 2048 is 15.7 us, most of it the call's own issue.
template <typename T, int S, bool kStats>
__global__ void __launch_bounds__(kRowsThreads, 1) int4_rows_kernel(RowsParams p) {
  constexpr int N = kRowsN;
  constexpr int kRun = 4 / S;    // consecutive words of a group a thread takes
  extern __shared__ unsigned char smem[];
  const int pitch = p.blocks * 256 + kRowsPad;
  constexpr int rw = kRowWarps, kws = kColWarps, tile_rows = kRowsTile;
  unsigned char* hid = smem;                                     // [N][pitch]
  float* sums = reinterpret_cast<float*>(smem + N * pitch);      // [blocks * S][N] of -8 sum h
  float* rscale = sums + p.blocks * S * N;                       // [N]
  float* red = rscale + N;                                       // [2][kws][N][tile_rows]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rwi = warp / kws, kw = warp % kws;  // neighbours share a weight row's lines
  const int64_t t0 = blockIdx.x * p.tiles / p.parts, t1 = (blockIdx.x + 1) * p.tiles / p.parts;
  const int per_tile = (p.blocks + kws - 1) / kws;  // blocks of a warp, the last perhaps empty
  const int64_t total = (t1 - t0) * per_tile;

  // The load's position: a tile's first row for this thread (row g of the warp's
  // 32, its words of a group), the bytes from there to rows g + 8 r, and the block
  // of columns.  Rows and columns past the ends read the last ones instead: such
  // rows are not stored, such columns meet hidden values of zero.
  const int words = p.words, groups = p.groups;
  const int last_word = (words - kRun) * 4;
  int64_t l_v = t0 * tile_rows + rwi * 32 + g;
  const unsigned char* l_row = nullptr;
  const uint16_t* l_scale = nullptr;
  int l_off[4], l_k = 0, l_kb = kw;
  int64_t l_tiles = t1 - t0;  // left to load
  auto seek = [&]() {
    const int64_t left = p.vocab - 1 - l_v;  // < 0 for a row past the last
    const int64_t v = left < 0 ? p.vocab - 1 : l_v;
    l_row = reinterpret_cast<const unsigned char*>(p.packed + v * words) + t * (kRun * 4);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int down = left < 8 * r ? (left < 0 ? 0 : static_cast<int>(left)) : 8 * r;
      l_off[r] = down * words * 4;
    }
    const int64_t sv = l_v + 8 * t;
    l_scale = p.scales + (sv < p.vocab ? sv : p.vocab - 1) * groups;
  };
  seek();
  auto load = [&](CodeBlock<S>& b) {
    const int kb = l_kb < p.blocks ? l_kb : p.blocks - 1;
#pragma unroll
    for (int i = 0; i < 4; i += kRun) {
      // words of a group stand together: group i / kRun, words t * kRun + 0..
      const int at = kb * 64 + i * 16;
      const unsigned char* from = l_row + (at < last_word - t * (kRun * 4) ? at : last_word - t * (kRun * 4));
#pragma unroll
      for (int r = 0; r < 4; ++r)
        load_codes<kRun>(&b.w[r][i], reinterpret_cast<const uint32_t*>(from + l_off[r]));
    }
#pragma unroll
    for (int i = 0; i < S; ++i) {
      const int gi = kb * S + i;
      b.scale[i] = l_scale[gi < groups ? gi : groups - 1];
    }
    l_kb += kws;
    if (++l_k == per_tile) {
      l_k = 0;
      l_kb = kw;
      if (--l_tiles > 0) {
        l_v += tile_rows;
        seek();
      }
    }
  };

  constexpr int kRing = kRowsRing<S>;
  CodeBlock<S> ring[kRing];
#pragma unroll
  for (int i = 0; i < kRing; ++i) load(ring[i]);

  // ---- the hidden rows, two warps each, while the first codes are on their way ----
  {
    constexpr int lanes = 16 / S;  // that hold a group's columns
    const int n = warp >> 1, half = warp & 1, units = p.blocks * 16;
    uint32_t* tops = reinterpret_cast<uint32_t*>(red);
    const uint4* src = p.hidden + static_cast<int64_t>(n) * words;
    uint32_t top = 0;
    if (n < p.rows)
      for (int i = half * 32 + lane; i < words; i += 64) top = max(top, top_bits(src[i]));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    const int e = row_exponent<T>(max(tops[n * 2], tops[n * 2 + 1]));
    const float up = __int_as_float((e + 127) << 23);
    if (half == 0 && lane == 0) rscale[n] = __int_as_float((127 - e) << 23);
    for (int i0 = half * 32; i0 < units; i0 += 64) {
      const int i = i0 + lane;
      float sum = 0.0f;
      uint4 x = make_uint4(0, 0, 0, 0);
      if (n < p.rows && i < words) x = scaled_columns<T>(src[i], up, sum);
      if (i < units)
        *reinterpret_cast<uint4*>(hid + n * pitch +
                                  ((i & ~15) + fragment_place(i & 15, lanes)) * 16) = x;
#pragma unroll
      for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      if (i < units && i % lanes == 0) sums[i / lanes * N + n] = -8.0f * sum;
    }
    __syncthreads();
  }

  // outputs of this thread: tile row tid % tile_rows, hidden rows tid / tile_rows, + step, ...
  constexpr int kOwn = tile_rows * N / kRowsThreads;
  const int orow = threadIdx.x % tile_rows, on = threadIdx.x / tile_rows;
  constexpr int step = kRowsThreads / tile_rows;
  RowStats st[kOwn];
  float cur[kOwn];
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    st[j] = RowStats{-INFINITY, 0.0f, -1, -1};
    cur[j] = 0.0f;
  }

  float acc[2][4] = {};
  int64_t tile = t0;
  int k = 0, buf = 0;
  auto compute = [&](const CodeBlock<S>& b) {
    const int kb = kw + k * kws;
    if (kb < p.blocks) {
      const unsigned char* h = hid + g * pitch + kb * 256 + t * 16;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const float own = to_float(*reinterpret_cast<const T*>(&b.scale[s]));
        float c[2][4] = {};
#pragma unroll
        for (int i = s * kRun; i < (s + 1) * kRun; ++i) {
          const uint4 x = *reinterpret_cast<const uint4*>(h + i * 64);
#pragma unroll
          for (int m = 0; m < 2; ++m) {
            uint32_t a0[4], a1[4];
            unpack8(b.w[2 * m][i], a0);
            unpack8(b.w[2 * m + 1][i], a1);
            mma_16816(c[m], a0[0], a1[0], a0[1], a1[1], x.x, x.y);
            mma_16816(c[m], a0[2], a1[2], a0[3], a1[3], x.z, x.w);
          }
        }
        const float2 h8 = *reinterpret_cast<const float2*>(sums + (kb * S + s) * N + 2 * t);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const float s0 = __shfl_sync(0xffffffffu, own, (lane & ~3) + 2 * m);
          const float s1 = __shfl_sync(0xffffffffu, own, (lane & ~3) + 2 * m + 1);
          group_add2(acc[m][0], acc[m][1], __float_as_uint(c[m][0]), __float_as_uint(c[m][1]),
                     h8.x, h8.y, s0);
          group_add2(acc[m][2], acc[m][3], __float_as_uint(c[m][2]), __float_as_uint(c[m][3]),
                     h8.x, h8.y, s1);
        }
      }
    }
    if (++k < per_tile) return;
    // ---- the tile's sums over the warps along K ----
    k = 0;
    float* rb = red + buf * (kws * N * tile_rows);
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = rwi * 32 + m * 16 + (e >> 1) * 8 + g, n = 2 * t + (e & 1);
        rb[(kw * N + n) * tile_rows + row] = acc[m][e];
        acc[m][e] = 0.0f;
      }
    __syncthreads();
    // the other buffer was read before this barrier, this one is before the next
    const int64_t v = tile * tile_rows + orow;
#pragma unroll
    for (int j = 0; j < kOwn; ++j) {
      const int n = on + j * step;
      if (n < N && n < p.rows) {
        float z = 0.0f;
#pragma unroll
        for (int q = 0; q < kws; ++q) z += rb[(q * N + n) * tile_rows + orow];
        z = logit_of(z, rscale[n]);
        if (!kStats) {
          if (v < p.vocab) {
            if (std::is_same<T, __nv_bfloat16>::value)
              static_cast<__nv_bfloat16*>(p.out)[n * p.vocab + v] = __float2bfloat16_rn(z);
            else
              static_cast<__half*>(p.out)[n * p.vocab + v] = __float2half_rn(z);
          }
        } else if (v < p.vocab) {
          if (p.round_bf16) z = __bfloat162float(__float2bfloat16_rn(z));
          const int c = static_cast<int>(v);
          merge_stats(st[j], z != z ? RowStats{-INFINITY, z, -1, c}
                                    : RowStats{z, z == INFINITY ? NAN : (z == -INFINITY ? 0.0f : 1.0f),
                                               c, -1});
          if (p.ids[n] == v) cur[j] = z;
        }
      }
    }
    buf ^= 1;
    ++tile;
  };

  for (int64_t i = 0; i < total; i += kRing) {
#pragma unroll
    for (int r = 0; r < kRing; ++r) {
      if (i + r >= total) break;
      compute(ring[r]);
      load(ring[r]);
    }
  }
  if (!kStats) return;

  // ---- the part's record of each hidden row: over the tile's rows ----
  __syncthreads();
  float* slots = red;  // [N][rw][8]
#pragma unroll
  for (int j = 0; j < kOwn; ++j) {
    const int n = on + j * step;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      RowStats o;
      o.m = __shfl_xor_sync(0xffffffffu, st[j].m, d);
      o.s = __shfl_xor_sync(0xffffffffu, st[j].s, d);
      o.where = __shfl_xor_sync(0xffffffffu, st[j].where, d);
      o.nan = __shfl_xor_sync(0xffffffffu, st[j].nan, d);
      merge_stats(st[j], o);
      cur[j] += __shfl_xor_sync(0xffffffffu, cur[j], d);  // one thread at most has seen the token
    }
    if (lane == 0 && n < N) {
      float* s = slots + (n * rw + orow / 32) * 8;
      s[0] = st[j].m;
      s[1] = st[j].s;
      s[2] = __int_as_float(st[j].where);
      s[3] = __int_as_float(st[j].nan);
      s[4] = cur[j];
    }
  }
  __syncthreads();
  if (threadIdx.x < N && threadIdx.x < p.rows) {
    const int n = threadIdx.x;
    RowStats a{-INFINITY, 0.0f, -1, -1};
    float c = 0.0f;
    for (int q = 0; q < rw; ++q) {
      const float* s = slots + (n * rw + q) * 8;
      merge_stats(a, RowStats{s[0], s[1], __float_as_int(s[2]), __float_as_int(s[3])});
      c += s[4];
    }
    p.records[blockIdx.x * p.rows + n] = record_of(a, c, static_cast<int>(t0 * tile_rows));
  }
}

// One block turns one hidden row into the fp16 row of the products, its group
// sums (8 sum h) and its scale 2^-e; rows past the last get zero sums.  Bound by
// latency, which the product kernel waits out: it starts when every block of this one
// has exited.
constexpr int kPrepThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kPrepThreads)
    int4_prepare_kernel(const uint4* hidden, int64_t rows, int vecs, int lanes, int n,
                        uint4* out, float* sums, float* row_scale) {
  __shared__ uint32_t tops[kPrepThreads / 32];
  const int64_t r = blockIdx.x;
  const int groups = vecs / lanes;
  float* my_sums = sums + (r / n * groups) * n + r % n;
  if (r >= rows) {
    for (int g = threadIdx.x; g < groups; g += kPrepThreads) my_sums[int64_t{g} * n] = 0.0f;
    if (threadIdx.x == 0) row_scale[r] = 0.0f;
    return;
  }
  const uint4* src = hidden + r * vecs;
  uint32_t top = 0;
  for (int i = threadIdx.x; i < vecs; i += kPrepThreads) top = max(top, top_bits(src[i]));
  top = __reduce_max_sync(0xffffffffu, top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPrepThreads / 32; ++i) top = max(top, tops[i]);
  const int e = row_exponent<T>(top);
  const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
  if (threadIdx.x == 0) row_scale[r] = down;
  // whole warps step together: a group's lanes share its sum
  for (int i0 = 0; i0 < vecs; i0 += kPrepThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    float sum = 0.0f;
    if (i < vecs) {
      out[r * vecs + i] = scaled_columns<T>(src[i], up, sum);
    }
    for (int d = 1; d < lanes; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (i < vecs && i % lanes == 0) my_sums[int64_t{i / lanes} * n] = 8.0f * sum;
  }
}

// ---------------------------------------------------------------------------
// Quantiser
// ---------------------------------------------------------------------------

constexpr int kQuantThreads = 256;
constexpr int kQuantWords = 4;  // words a thread, a block apart: loads in flight
constexpr int64_t kQuantBlock = kQuantThreads * kQuantWords;

// rint(w / s) + 8, ties to even, as the low bits of a float; r is 1 / s to a few
// units.  The first sum rounds w r to a multiple of 2^-14: a quotient that is a tie
// becomes one exactly, and no other can, since a quotient of two 11-bit numbers is
// a tie or 2^-12 away from it.  The second rounds to an integer, ties to even.
__device__ __forceinline__ float code_float(float w, float r) {
  return fmaf(w, r, 768.0f) + (12582920.0f - 768.0f);  // 1.5 2^9, then 1.5 2^23 + 8
}

// The word of eight columns.  kClamp: a quotient may leave [-8, 7].
template <typename T, bool kClamp>
__device__ __forceinline__ uint32_t code_word(uint4 v, float r, float grow) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t word = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 w = pair_floats<T>(u[j]);
    float lo = code_float(kClamp ? w.x * grow : w.x, r);
    float hi = code_float(kClamp ? w.y * grow : w.y, r);
    if (kClamp) {
      lo = fminf(fmaxf(lo, 12582912.0f), 12582927.0f);
      hi = fminf(fmaxf(hi, 12582912.0f), 12582927.0f);
    }
    word |= (__float_as_uint(lo) & 15u) << (4 * j);
    word |= (__float_as_uint(hi) & 15u) << (4 * j + 16);
  }
  return word;
}

// A lane holds 8 columns (16 bytes) and writes their word; the group's lanes
// (4, 8 or 16) share the maximum.  |w| compares as its bits, NaN above all, so
// a NaN or infinite weight leaves its group's scale NaN or infinite.
// Bound by memory, 2.5 bytes a weight, once the divisions are gone: with them, and
// a word every thread, 128256 x 4096 took 720 us; with one reciprocal a group and
// exact remainders for the ties 493 us, 90 % of the issue slots; with the two
// roundings 270 to 290 us, 4.6 to 4.9 TB/s.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    quantize_kernel(const uint4* weight, int64_t words, int lanes_log2, uint32_t* packed,
                    T* scales) {
  const int64_t first = blockIdx.x * kQuantBlock + threadIdx.x;
  const int lanes = 1 << lanes_log2;
  uint4 v[kQuantWords];
#pragma unroll
  for (int k = 0; k < kQuantWords; ++k) {
    const int64_t i = first + k * kQuantThreads;
    // words is a multiple of 4, a group's lanes are in range together
    v[k] = i < words ? __ldcs(weight + i) : make_uint4(0, 0, 0, 0);
  }
#pragma unroll
  for (int k = 0; k < kQuantWords; ++k) {
    const int64_t i = first + k * kQuantThreads;
    uint32_t top = __vmaxu2(__vmaxu2(v[k].x & 0x7fff7fffu, v[k].y & 0x7fff7fffu),
                            __vmaxu2(v[k].z & 0x7fff7fffu, v[k].w & 0x7fff7fffu));
    top = max(top & 0xffffu, top >> 16);
    for (int d = 1; d < lanes; d <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    if (i >= words) continue;
    const float amax = pair_floats<T>(top).x;
    // times 1/7 rounds to 16 bits as the quotient does: 7 times an odd number of
    // half steps has more bits than a maximum, so no quotient is a tie, and the
    // nearest to one is 2^-16 away
    T scale;
    if (std::is_same<T, __nv_bfloat16>::value)
      *reinterpret_cast<__nv_bfloat16*>(&scale) = __float2bfloat16_rn(amax * (1.0f / 7.0f));
    else
      *reinterpret_cast<__half*>(&scale) = __float2half_rn(amax * (1.0f / 7.0f));
    const float s = to_float(scale);
    // a scale of the 16-bit type's last binades has few bits: quotients may pass 7,
    // and the reciprocal f32's range (scale and weights then grow alike)
    constexpr bool bf = std::is_same<T, __nv_bfloat16>::value;
    uint32_t word = 0x88888888u;
    if (s >= (bf ? 1e-30f : 1e-3f) && s < INFINITY) {
      word = code_word<T, false>(v[k], __fdividef(1.0f, s), 1.0f);
    } else if (s > 0.0f && s < INFINITY) {
      const float grow = bf ? 1.2676506e30f : 1.0f;  // 2^100
      word = code_word<T, true>(v[k], __frcp_rn(s * grow), grow);
    }
    packed[i] = word;
    if ((i & (lanes - 1)) == 0) scales[i >> lanes_log2] = scale;
  }
}

// Bound by memory: 128256 x 4096 in 199 us, 1.32 GB at 6.6 TB/s.
template <typename T>
__global__ void __launch_bounds__(kQuantThreads)
    dequantize_kernel(const uint32_t* packed, const T* scales, int64_t words, int lanes_log2,
                      uint4* weight) {
  const int64_t first = blockIdx.x * kQuantBlock + threadIdx.x;
  uint32_t w[kQuantWords];
  float s[kQuantWords];
#pragma unroll
  for (int k = 0; k < kQuantWords; ++k) {
    const int64_t i = first + k * kQuantThreads;
    w[k] = i < words ? packed[i] : 0;
    s[k] = i < words ? to_float(scales[i >> lanes_log2]) : 0.0f;
  }
#pragma unroll
  for (int k = 0; k < kQuantWords; ++k) {
    const int64_t i = first + k * kQuantThreads;
    if (i >= words) break;
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // 2^23 + code as float bits, less 2^23 + 8: q
      const float lo =
          __uint_as_float(0x4b000000u | ((w[k] >> (4 * j)) & 15u)) - 8388616.0f;
      const float hi =
          __uint_as_float(0x4b000000u | ((w[k] >> (4 * j + 16)) & 15u)) - 8388616.0f;
      u[j] = pack_pair<T>(s[k] * lo, s[k] * hi);
    }
    __stcs(weight + i, make_uint4(u[0], u[1], u[2], u[3]));
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxInt4Rows = INT32_MAX - 64;


// log2 of the words, and so lanes, of a group of 32, 64 or 128.
int lanes_log2(int group) { return group == 32 ? 2 : (group == 64 ? 3 : 4); }

bool int4_weight_ok(int64_t vocab, int64_t dim, int group) {
  int64_t n = 0;
  return (group == 32 || group == 64 || group == 128) && vocab > 0 &&
         vocab <= INT32_MAX - 2 * kTileV && dim > 0 && dim % group == 0 &&
         dim <= INT32_MAX / 2 && count_ok(vocab, dim, &n) && n <= kMaxCount &&
         n / (8 * kQuantThreads) < INT32_MAX;
}

// A launch's shape: R blocks of 128 weight rows a tile, its tiles and its parts
// (one a CTA).
struct Int4Plan {
  int n, r;        // r: 0 for int4_rows_kernel
  bool resident;
  int stages;
  int tile_rows;
  int64_t tiles, parts;
};

size_t rows_smem(int64_t blocks, int group) {
  constexpr int n = kRowsN;
  return n * (blocks * 256 + kRowsPad) + (blocks * (kChunk / group) * n + n) * 4 +
         size_t{2} * kColWarps * n * kRowsTile * 4;
}

size_t int4_smem(int n, int r, bool resident, int stages, int64_t chunks, int64_t slots) {
  const size_t hidden = static_cast<size_t>(n) * kChunk * 2;
  return stages * (r * size_t{kStageW} + (resident ? 0 : hidden)) +
         (resident ? chunks * hidden : 0) +
         (static_cast<size_t>(r) * (n < kXchRows ? n : kXchRows) * kXchMost + (slots + 1) * n) * 4 +
         1024 + 512;
}

// Hidden rows of a pass: the accumulators of a chunk's groups are at most 64
// columns wide, so a group of 128 takes up to 64 rows a pass, one of 64 up to
// 32, one of 32 sixteen; more rows read the weight again.  The hidden rows stay
// in shared memory where they leave room for eight stages of codes; where they
// do not, their slices are read again for every tile, and tiles of 256 weight
// rows halve that traffic.
//
// Up to 8 hidden rows against groups of 64 or 128 take int4_rows_kernel, where
// they fit shared memory beside the sums.  Measured at 8 rows x 128256 x 4096, it
// against the other: groups of 128 62 and 77 us, of 64 95 and 107 us, of 32 (an
// accumulator and a load for every word) 166 and 121 us; 16 rows of groups of 128
// 114 and 77 us.
Int4Plan int4_plan(int64_t rows, int64_t vocab, int64_t dim, int group) {
  Int4Plan pl;
  const int64_t blocks = (dim + kChunk - 1) / kChunk;
  pl.n = kRowsN;
  const int64_t sms = sm_count() < kMaxParts ? sm_count() : kMaxParts;
  if (rows <= kRowsN && group >= 64 && rows_smem(blocks, group) <= kSmemLimit) {
    pl.r = 0;
    pl.resident = true;
    pl.stages = 0;
    pl.tile_rows = kRowsTile;
    pl.tiles = (vocab + kRowsTile - 1) / kRowsTile;
    pl.parts = pl.tiles < sms ? pl.tiles : sms;
    return pl;
  }
  const int most = group / 2;
  const int64_t slots = blocks * kChunk / group;
  pl.n = rows > 32 && most >= 64 ? 64 : (rows > 16 && most >= 32 ? 32 : 16);
  for (;; pl.n /= 2) {  // the widest hidden rows leave room for 16 of them only
    pl.resident = int4_smem(pl.n, 1, true, 8, blocks, slots) <= kSmemLimit;
    pl.r = pl.resident ? 1 : 2;
    pl.stages = kMaxStages;
    while (pl.stages > 1 &&
           int4_smem(pl.n, pl.r, pl.resident, pl.stages, blocks, slots) > kSmemLimit)
      --pl.stages;
    if (pl.stages > 1 || pl.n == 16) break;
  }
  // With one row block the warpgroups take turns at the stages.  An even number gives
  // each warpgroup its own: with an odd one it would wait for phases of a stage of
  // which it has not seen the one before, and a parity cannot tell a phase from the
  // next but one.  (At nine stages the warpgroup that is nine chunks ahead of a late load,
  // as far as the buffers let it, took the stage for filled.)
  if (pl.resident) pl.stages -= pl.stages % 2;
  pl.tile_rows = pl.r * kTileV;
  pl.tiles = (vocab + pl.tile_rows - 1) / pl.tile_rows;
  pl.parts = pl.tiles < sms ? pl.tiles : sms;
  return pl;
}

// Workspace: the fp16 rows, the group sums and row scales of whole passes (sized
// for passes of 64, whatever the launch takes), and the statistics' records.
struct Int4Layout {
  size_t hidden, sums, row_scale, records, bytes;
};

Int4Layout int4_layout(int64_t rows, int64_t dim, int64_t vocab, int group, bool stats) {
  auto up = [](size_t x) { return (x + 1023) / 1024 * 1024; };
  const size_t padded = static_cast<size_t>((rows + 63) / 64 * 64);
  const int64_t tiles = (vocab + kTileV - 1) / kTileV;
  Int4Layout l;
  l.hidden = 0;
  l.sums = up(static_cast<size_t>(rows) * dim * 2);
  l.row_scale = l.sums + up(padded * (dim / group) * 4);
  l.records = l.row_scale + up(padded * 4);
  l.bytes = l.records + (stats ? static_cast<size_t>(tiles < kMaxParts ? tiles : kMaxParts) *
                                     static_cast<size_t>(rows) * sizeof(cid_shard_record_t)
                               : 0);
  return l;
}

template <typename T, int N, int S, int R, bool kResident>
int launch_int4(const CUtensorMap& map_w, const CUtensorMap& map_h, const Int4Params& p,
                cudaStream_t stream) {
  const size_t smem =
      int4_smem(N, R, kResident, p.stages, p.chunks, static_cast<int64_t>(p.chunks) * S);
  const cudaError_t e = cudaFuncSetAttribute(int4_head_kernel<T, N, S, R, kResident>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
  if (e != cudaSuccess) return record_cuda_error(e);
  // a programmatic dependent of the kernel that prepares the hidden rows: its set-up
  // and first codes overlap that one's completion, not its run
  return launch_pdl(int4_head_kernel<T, N, S, R, kResident>, dim3(static_cast<unsigned>(p.parts)),
                    dim3(int4_threads(R)), smem, stream, map_w, map_h, p);
}

template <typename T, int N, int S>
int launch_int4(const Int4Plan& pl, const CUtensorMap& map_w, const CUtensorMap& map_h,
                const Int4Params& p, cudaStream_t stream) {
  return pl.resident ? launch_int4<T, N, S, 1, true>(map_w, map_h, p, stream)
                     : launch_int4<T, N, S, 2, false>(map_w, map_h, p, stream);
}

template <typename T, int S, bool kStats>
int launch_rows(const RowsParams& p, size_t smem, cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(int4_rows_kernel<T, S, kStats>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
  if (e != cudaSuccess) return record_cuda_error(e);
  int4_rows_kernel<T, S, kStats>
      <<<static_cast<unsigned>(p.parts), kRowsThreads, smem, stream>>>(p);
  return launch_result();
}

template <typename T, int S>
int launch_rows(const RowsParams& p, size_t smem, cudaStream_t stream) {
  return p.out != nullptr ? launch_rows<T, S, false>(p, smem, stream)
                          : launch_rows<T, S, true>(p, smem, stream);
}

template <typename T>
int dispatch_int4(const void* hidden, int64_t dim, const void* packed, int group, Int4Params p,
                  const Int4Plan& pl, unsigned char* ws, const Int4Layout& l,
                  cudaStream_t stream) {
  p.groups = dim / group;
  p.chunks = static_cast<int>((dim + kChunk - 1) / kChunk);
  p.row_blocks = (p.rows + pl.n - 1) / pl.n;
  p.tiles = pl.tiles;
  p.parts = pl.parts;
  p.stages = pl.stages;
  p.sums = reinterpret_cast<const float*>(ws + l.sums);
  p.row_scale = reinterpret_cast<const float*>(ws + l.row_scale);
  if (pl.r == 0) {
    RowsParams q = {};
    q.packed = static_cast<const uint32_t*>(packed);
    q.scales = static_cast<const uint16_t*>(p.scales);
    q.hidden = static_cast<const uint4*>(hidden);
    q.rows = p.rows;
    q.vocab = p.vocab;
    q.words = static_cast<int>(dim / 8);
    q.groups = static_cast<int>(p.groups);
    q.blocks = static_cast<int>((dim + kChunk - 1) / kChunk);
    q.tiles = pl.tiles;
    q.parts = pl.parts;
    q.out = p.out;
    q.records = p.records;
    q.ids = p.ids;
    q.round_bf16 = p.round_bf16;
    const size_t smem = rows_smem(q.blocks, group);
    return group == 128 ? launch_rows<T, 1>(q, smem, stream) : launch_rows<T, 2>(q, smem, stream);
  }
  int4_prepare_kernel<T><<<static_cast<unsigned>(p.row_blocks * pl.n), kPrepThreads, 0, stream>>>(
      static_cast<const uint4*>(hidden), p.rows, static_cast<int>(dim / 8), group / 8, pl.n,
      reinterpret_cast<uint4*>(ws + l.hidden), reinterpret_cast<float*>(ws + l.sums),
      reinterpret_cast<float*>(ws + l.row_scale));
  int rc = launch_result();
  if (rc != CID_OK) return rc;
  CUtensorMap map_w, map_h;
  // codes copied as 16-bit elements, four columns each
  rc = make_map_sw128(&map_w, CID_DTYPE_F16, packed, dim / 4, p.vocab, dim / 4, kChunk / 4, kTileV,
                      CU_TENSOR_MAP_SWIZZLE_64B);
  if (rc == CID_OK)
    rc = make_map_sw128(&map_h, CID_DTYPE_F16, ws + l.hidden, dim, p.rows, dim, 64, pl.n);
  if (rc != CID_OK) return rc;
  switch (group) {
    case 128:
      return pl.n == 64   ? launch_int4<T, 64, 1>(pl, map_w, map_h, p, stream)
             : pl.n == 32 ? launch_int4<T, 32, 1>(pl, map_w, map_h, p, stream)
                          : launch_int4<T, 16, 1>(pl, map_w, map_h, p, stream);
    case 64:
      return pl.n == 32 ? launch_int4<T, 32, 2>(pl, map_w, map_h, p, stream)
                        : launch_int4<T, 16, 2>(pl, map_w, map_h, p, stream);
    default:
      return launch_int4<T, 16, 4>(pl, map_w, map_h, p, stream);
  }
}

// Widest hidden row of the products: its group sums stay in shared memory.
constexpr int64_t kMaxInt4Dim = 32768;

bool int4_product_ok(int64_t rows, int64_t dim, int64_t vocab, int group) {
  int64_t n = 0;
  return rows >= 0 && rows <= kMaxInt4Rows && int4_weight_ok(vocab, dim, group) &&
         dim <= kMaxInt4Dim && count_ok(rows, dim, &n) && n <= kMaxCount &&
         count_ok(rows, vocab, &n) && n <= kMaxCount;
}

// Checks shared by the two products; rows == 0 is left to the caller.
int check_int4(cid_dtype_t dtype, const void* hidden, int64_t rows, int64_t dim,
               const uint32_t* packed, const void* scales, int group, int64_t vocab,
               const void* workspace, const uint32_t* status) {
  if (dtype != CID_DTYPE_BF16 && dtype != CID_DTYPE_F16) return CID_ERR_UNSUPPORTED_DTYPE;
  if (!int4_product_ok(rows, dim, vocab, group)) return CID_ERR_INVALID_ARGUMENT;
  if (misaligned({{hidden, 16}, {packed, 16}, {scales, 2}, {workspace, 16}, {status, 4}}))
    return CID_ERR_MISALIGNED;
  return CID_OK;
}

int run_int4(cid_dtype_t dtype, const void* hidden, int64_t dim, const void* packed, int group,
             const Int4Params& p, const Int4Plan& pl, void* workspace, const Int4Layout& l,
             void* stream) {
  auto* ws = static_cast<unsigned char*>(workspace);
  return dtype == CID_DTYPE_F16
             ? dispatch_int4<__half>(hidden, dim, packed, group, p, pl, ws, l, as_stream(stream))
             : dispatch_int4<__nv_bfloat16>(hidden, dim, packed, group, p, pl, ws, l,
                                            as_stream(stream));
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
  const unsigned blocks = static_cast<unsigned>((words + kQuantBlock - 1) / kQuantBlock);
  const auto* w = static_cast<const uint4*>(weight);
  if (dtype == CID_DTYPE_F16)
    quantize_kernel<__half><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        w, words, lanes_log2(group_size), packed, static_cast<__half*>(scales));
  else
    quantize_kernel<__nv_bfloat16><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        w, words, lanes_log2(group_size), packed, static_cast<__nv_bfloat16*>(scales));
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
  const unsigned blocks = static_cast<unsigned>((words + kQuantBlock - 1) / kQuantBlock);
  auto* w = static_cast<uint4*>(weight);
  if (dtype == CID_DTYPE_F16)
    dequantize_kernel<__half><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        packed, static_cast<const __half*>(scales), words, lanes_log2(group_size), w);
  else
    dequantize_kernel<__nv_bfloat16><<<blocks, kQuantThreads, 0, as_stream(stream)>>>(
        packed, static_cast<const __nv_bfloat16*>(scales), words, lanes_log2(group_size), w);
  return launch_result();
}

extern "C" size_t cid_lm_head_quantized_workspace_bytes(int64_t rows, int64_t hidden_dim,
                                                        int64_t vocab, int group_size,
                                                        int statistics) {
  if (rows <= 0 || !int4_product_ok(rows, hidden_dim, vocab, group_size)) return 0;
  return int4_layout(rows, hidden_dim, vocab, group_size, statistics != 0).bytes;
}

extern "C" int cid_lm_head_quantized_logits(cid_dtype_t dtype, const void* hidden, int64_t rows,
                                            int64_t hidden_dim, const uint32_t* packed,
                                            const void* scales, int group_size, int64_t vocab,
                                            void* logits, void* workspace,
                                            size_t workspace_bytes, uint32_t* status,
                                            void* stream) {
  const int rc = check_int4(dtype, hidden, rows, hidden_dim, packed, scales, group_size, vocab,
                            workspace, status);
  if (rc != CID_OK) return rc;
  if (misaligned({{logits, 2}})) return CID_ERR_MISALIGNED;
  if (rows == 0) return CID_OK;
  if (any_null({hidden, packed, scales, logits, workspace})) return CID_ERR_INVALID_ARGUMENT;
  const Int4Layout l = int4_layout(rows, hidden_dim, vocab, group_size, false);
  if (workspace_bytes < l.bytes) return CID_ERR_SCRATCH_LIMIT;
  Int4Params p = {};
  p.rows = rows;
  p.vocab = vocab;
  p.scales = scales;
  p.out = logits;
  p.status = status;
  return run_int4(dtype, hidden, hidden_dim, packed, group_size, p,
                  int4_plan(rows, vocab, hidden_dim, group_size), workspace, l, stream);
}

extern "C" int cid_lm_head_quantized_display_statistics(
    cid_dtype_t dtype, const void* hidden, int64_t rows, int64_t hidden_dim,
    const uint32_t* packed, const void* scales, int group_size, int64_t vocab,
    const int64_t* token_ids, int round_bf16, float* confidence, int64_t* predicted,
    float* current_confidence, void* workspace, size_t workspace_bytes, uint32_t* status,
    void* stream) {
  int rc = check_int4(dtype, hidden, rows, hidden_dim, packed, scales, group_size, vocab,
                      workspace, status);
  if (rc != CID_OK) return rc;
  if (misaligned(
          {{token_ids, 8}, {confidence, 4}, {predicted, 8}, {current_confidence, 4}}))
    return CID_ERR_MISALIGNED;
  if (rows == 0) return CID_OK;
  if (any_null({hidden, packed, scales, token_ids, confidence, predicted, current_confidence,
                workspace}))
    return CID_ERR_INVALID_ARGUMENT;
  const Int4Layout l = int4_layout(rows, hidden_dim, vocab, group_size, true);
  if (workspace_bytes < l.bytes) return CID_ERR_SCRATCH_LIMIT;
  auto* records =
      reinterpret_cast<cid_shard_record_t*>(static_cast<unsigned char*>(workspace) + l.records);
  Int4Params p = {};
  p.rows = rows;
  p.vocab = vocab;
  p.scales = scales;
  p.records = records;
  p.ids = token_ids;
  p.status = status;
  p.round_bf16 = round_bf16 ? 1 : 0;
  const Int4Plan pl = int4_plan(rows, vocab, hidden_dim, group_size);
  rc = run_int4(dtype, hidden, hidden_dim, packed, group_size, p, pl, workspace, l, stream);
  if (rc != CID_OK) return rc;
  // merge the parts of every row (ascending column ranges) into its statistics
  int64_t offsets[kMaxParts + 1];
  for (int64_t i = 0; i < pl.parts; ++i)
    offsets[i] = i * pl.tiles / pl.parts * pl.tile_rows;
  offsets[pl.parts] = vocab;
  return cid_display_combine_records(records, static_cast<int>(pl.parts), offsets, token_ids,
                                     rows, confidence, predicted, current_confidence, status,
                                     stream);
}
