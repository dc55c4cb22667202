// Product of two 8-bit (e4m3) operands with a scale for each block of 128, on the 5th-generation tensor cores:
//
//   out[z, m, n] = bias[z, n] + sum over the segments and 128-wide blocks kb of z's contraction
//                  sa[m, kb] * sb[kb, n / 128] * sum_{k in kb} A[m, k] B[k, n]
//
// A's scales belong to 1 x 128 or 128 x 128 blocks, B's to 128 x 128 blocks.  The inner sum runs in tensor memory (four
// MMAs of 32); its 128 x 256 results then go through registers once, where they are scaled and added in fp32.  So a sum in
// the tensor cores' own accumulator stays short however long the contraction is (error against 64 bits of a sum of 120000 products:
// 1.4e-7), and any fp32 scales will do.
//
// Operand layouts, stages and pairs of CTAs are those of gemm_tc.cuh.  What differs:
//   * A stage holds 128 of the contraction axis, one byte each: as many bytes as 64 bf16 values, twice the products.  Four stages
//     (a pair; three for a CTA alone) are as fast as six and leave 64 KB for the output, which goes out by TMA.
//   * The two accumulators of tensor memory alternate from block to block instead of from tile to tile: while the MMAs fill
//     one, the eight epilogue warps read the other and add it to their 128 sums a thread (32 rows x 128 columns a warp).
//     That is 32768 FMAs a block and SM, 256 cycles of the fp32 pipes, and a second reader of tensor memory beside the MMAs: 0.60 us a
//     block, where the MMAs and their copies alone take 0.44 (0.37 in the library's product of unscaled operands).
//   * So blocks that follow one another with the same scales, as most do where A's blocks are 128 x 128 (powers of two, of
//     weights or gradients of one kind), are multiplied into one accumulator, up to kMostJoined of them (1024 products a sum):
//     12 x 4000 x 24576 x 768 in 685 us (2650 TFLOP/s), 925 where no two are equal; 8192^3 404 (2720).
//   * Warps 2 and 3, which have no role there, bring scales, bias and tiles' coordinates to the epilogue through shared memory.
//   * MN-major operands come in boxes of 128(MN) x 128(K): K rows of 128 B, 8-row groups 1024 B apart, boxes 16 KB apart; the
//     32-wide K step of one MMA moves the start address by 4096 B (K-major: by 32 B).
// What bounds it now: joined blocks, shared memory (stages written and read: 64 KB a block and SM) and, with few blocks to a tile,
// the output's way to memory (12 x 4000 x 768 x 24576: 943 us, 740 without the copies); separate ones, the epilogue above, and for
// few blocks its start and output between the tiles (1190 us; scales by row and a bias 1290).
// Tried without gain: MMAs of half the columns, each half of the epilogue on its own two accumulators (925 -> 997 us); sixteen
// epilogue warps of 64 columns (975); reads of 32 columns, packed FMAs, five stages, two stages to an MMA round.
//
// No TMA load uses cluster multicast.  Every wait is bounded as there.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "gemm_tc.cuh"

namespace clt {
namespace f8 {

using tc::kBM;
using tc::kBN;
using tc::kEpiThreads;
using tc::kEpiWarps;
using tc::kFirstEpiWarp;
using tc::kMaxStages;
using tc::kThreads;
using tc::kTmemCols;
constexpr int kBK = 128;         // contraction of a stage = of a scale block
constexpr int kBox = 128 * 128;  // bytes of one box
constexpr int kRegsLean = 88, kRegsEpi = 208;  // 128 * 88 + 256 * 208 = 384 * 168, what the block is launched with
constexpr int kMostJoined = 8;   // blocks whose products may share one sum in tensor memory

template <bool kPair>
struct Tile {
  static constexpr int kCtas = kPair ? 2 : 1;
  static constexpr int kM = kCtas * kBM;
  static constexpr int kBRows = kBN / kCtas;
  static constexpr int kABytes = kBM * kBK;
  static constexpr int kBBytes = kBRows * kBK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = kPair ? 4 : 3;  // (six and four, without room for the output, were no faster)
};
constexpr int kOperandBytes = 144 * 1024;
static_assert(Tile<true>::kStages * Tile<true>::kStageBytes <= kOperandBytes &&
                  Tile<false>::kStages * Tile<false>::kStageBytes <= kOperandBytes,
              "operand stages");
constexpr int kOutBytes = 8 * 1024;  // a warp's output on its way to memory: two boxes of 32 rows x 128 B
// Scales on their way to the epilogue, a window of blocks at a time.  Bit i of `starts`: block i begins a group, blocks with the same
// scales that share one sum in tensor memory; `a` and `b` hold the groups' scales, of the tile's 128 rows (A in 1 x 128: every
// block is a group) or of the whole tile, and of its two halves of columns.
template <bool kByRow>
struct alignas(16) ScaleRing {
  static constexpr int kWindow = kByRow ? 8 : 32, kSlots = kByRow ? 2 : 4;
  float a[kSlots][kByRow ? kWindow * 128 : kWindow];
  float b[kSlots][kWindow][2];
  float bias[kSlots][kBN];  // of tiles, which have a window each at least
  int4 tile[kSlots];  // with a tile's first window: row, column, output slab, blocks (0: there are no more tiles)
  uint32_t starts[kSlots];
  uint32_t far[kSlots][2];  // some scale that a scale warp brought with the window is far_from_one
  uint64_t full[kSlots], empty[kSlots];
};
constexpr int kSmemBytes =
    kOperandBytes + kEpiWarps * kOutBytes + 1024 /*alignment slack*/ + 256 /*barriers*/ + (int)sizeof(ScaleRing<true>);
static_assert(sizeof(tc::Barriers) <= 256 && sizeof(ScaleRing<false>) <= sizeof(ScaleRing<true>) && kSmemBytes <= 232448, "shared memory");
constexpr int kRowsOut = 4;    // rows of the output in flight where they are written value by value
constexpr int kScaleWarps = 2;  // warps 2 and 3

// Scales of one operand: element strides between matrices, between blocks along M (or N) and along K.
struct Scales {
  const float* p;
  long long z, mn, k;
  int shift;  // log2 of the rows of a block: 0 or 7
};

struct Out {
  void* p;
  int dtype;  // 0 fp32, 1 fp16, 2 bf16
  long long ld, z;
  const float* bias;  // [nz, N] or NULL
  long long bias_z;
  int tma;  // rows of every slab start on 16 bytes: copied out by TMA
};

// Waits and arrivals at CTA scope, also where the barrier is the other CTA's: what they order are reads of tensor memory, which
// tcgen05's own fences cover, and no other data passes from CTA to CTA.  At cluster scope (gemm_tc.cuh, once a tile) each arrival
// is a memory fence behind every load in flight and each wait drops the L1 that holds the scales: 8192^3 887 instead of
// 1543 TFLOP/s.
__device__ __forceinline__ bool try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code) {
  if (try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (try_wait(bar, parity)) return true;
    if (*abort_flag != 0) return false;
    if (clock64() - t0 > tc::kWaitCycles) {
      report_status(status, code);
      *abort_flag = 1;
      return false;
    }
  }
}
// Whether the n-th block's products are in tensor memory; uniform over the warp.  All lanes look: one that tells the others costs
// more, each block (8192^3: 463 -> 587 us without the sums).
__device__ __forceinline__ bool block_ready(tc::Barriers* bars, uint32_t n, volatile int* abort_flag, int* status) {
  const bool ok = wait(tc::smem_u32(&bars->tmem_full[n & 1]), (n >> 1) & 1, abort_flag, status, kTimeoutTmemFull);
  if (!__all_sync(0xffffffffu, ok)) return false;
  tc::tc_fence_after();
  return true;
}
// One lane of a converged warp.  A role's warp runs its loop as a whole and only what must not happen 32 times is under this: the
// loop's values then stay in uniform registers, where the MMAs and copies want them (a loop in one lane alone: 2208 instead of
// 2450 TFLOP/s at 12 x 4000 x 24576 x 768, without the sums).
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(one));
  return one != 0;
}
__device__ __forceinline__ void arrive_remote(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

template <bool kPair>
__device__ __forceinline__ void umma_e4m3(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                          uint32_t accumulate) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Instruction descriptor: as tc::instr_desc with both operand formats 0 (e4m3).
__host__ __device__ constexpr uint32_t instr_desc(bool a_mn, bool b_mn, int m) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(kBN >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// Asynchronous read of 16 accumulator columns of this warp's 32 lanes; valid after tmem_ld_wait(r), through which the values pass so
// that nothing that uses them is moved ahead of it.
__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void fma16(float* acc, const uint32_t (&d)[16], float s) {
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = fmaf(__uint_as_float(d[i]), s, acc[i]);
}
__device__ __forceinline__ void mul16(uint32_t (&d)[16], float s) {
#pragma unroll
  for (int i = 0; i < 16; ++i) d[i] = __float_as_uint(__uint_as_float(d[i]) * s);
}
// Scales whose product with another may not be one of fp32's normal numbers: below 2^-63 or from 2^63 on (zeros, infinities and NaN
// among them).
__device__ __forceinline__ bool far_from_one(float s) {
  return (__float_as_uint(s) & 0x7fffffffu) - (64u << 23) >= 126u << 23;
}
// One is then applied after the other where their product is not normal.  A sum d of products is 0 or 2^-18 to 2^28 in magnitude.  Of
// a small product the larger scale comes first (below 2^23: the other is at least 2^-149), of a large one the smaller (above 1), so
// that d times it neither overflows nor loses bits unless the result does.
struct Factors {
  float first, second;
  __device__ __forceinline__ Factors(float a, float b) {
    first = 1.f, second = a * b;
    if (!(fabsf(second) >= 0x1p-126f && fabsf(second) <= 3.402823466e38f) && a != 0.f && b != 0.f) {
      const bool a_first = fabsf(second) < 1.f ? fabsf(a) > fabsf(b) : fabsf(a) < fabsf(b);
      first = a_first ? a : b, second = a_first ? b : a;
    }
  }
};

// ---- stores -------------------------------------------------------------------------------------
template <class T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// 16 bytes of finished sums in the output's type: 4 fp32, 8 16-bit values
template <int kOut>
__device__ __forceinline__ uint4 pack_out(const float* v) {
  if constexpr (kOut == 0)
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  else if constexpr (kOut == 1)
    return make_uint4(pack16<__half>(v[0], v[1]), pack16<__half>(v[2], v[3]), pack16<__half>(v[4], v[5]), pack16<__half>(v[6], v[7]));
  else
    return make_uint4(pack16<__nv_bfloat16>(v[0], v[1]), pack16<__nv_bfloat16>(v[2], v[3]), pack16<__nv_bfloat16>(v[4], v[5]),
                      pack16<__nv_bfloat16>(v[6], v[7]));
}

__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// A warp's 32 rows x 128 columns of finished sums, to the output in the type kOut (as Out::dtype; one instantiation each: with all
// three in one kernel the sums do not stay in registers).  Boxes of 32 rows x 128 B go through two buffers of shared memory
// (128-byte swizzle: conflict-free 16-byte stores, a row per lane) and out by TMA, which clips what lies behind the matrix's
// end; the warp does not wait for its last two.  Rows that do not start on 16 bytes are written from the buffers by the warp.
// (16-byte stores from registers through a small buffer, as in epi::store_rows32, took 2.4 us a tile, in which the tensor cores wait:
// 12 x 4000 x 768 x 24576 1643 instead of 1318 us.)
template <int kOut>
__device__ __forceinline__ void store_warp(const float (&acc)[128], uint8_t* buf, const CUtensorMap* map, const Out& o, int z, int row0,
                                           int col0, int M, int N) {
  constexpr int kSize = kOut == 0 ? 4 : 2, kCols = 128 / kSize, kPer = 16 / kSize;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int c0 = 0; c0 < 128 / kCols; c0 += 2) {
    if (lane == 0) bulk_wait_read();  // the buffers' last copies have been read
    __syncwarp();
#pragma unroll
    for (int c = c0; c < c0 + 2; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        *reinterpret_cast<uint4*>(buf + (c & 1) * 4096 + lane * 128 + ((i ^ (lane & 7)) << 4)) =
            pack_out<kOut>(acc + c * kCols + i * kPer);
    }
    if (o.tma) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
#pragma unroll
        for (int c = c0; c < c0 + 2; ++c) {
          const int n = col0 + c * kCols;
          if (n < N)
            asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map),
                         "r"(tc::smem_u32(buf + (c & 1) * 4096)), "r"(n), "r"(row0), "r"(z)
                         : "memory");
        }
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      }
    } else {
      __syncwarp();
      // a few rows at a time, so that their reads and stores are in flight together (one by one: 25 us of products took 61 to
      // 66, now 25 to 32; more rows spill)
      using U = typename std::conditional<kOut == 0, uint32_t, uint16_t>::type;
      const int rows = min(32, M - row0);
#pragma unroll
      for (int j = 0; j < 2 * kCols; j += 32) {
        const int col = c0 * kCols + j + lane, k = (j + lane) % kCols;
        U* p = (U*)o.p + z * o.z + (long long)row0 * o.ld + col0 + col;
        const uint8_t* box = buf + (j + lane) / kCols * 4096 + k % kPer * kSize;
        if (col0 + col < N) {
#pragma unroll 1
          for (int r0 = 0; r0 < rows; r0 += kRowsOut) {
            U v[kRowsOut];
#pragma unroll
            for (int r = 0; r < kRowsOut; ++r)
              v[r] = *reinterpret_cast<const U*>(box + (r0 + r) * 128 + (((k / kPer) ^ ((r0 + r) & 7)) << 4));
            if (r0 + kRowsOut <= rows) {
#pragma unroll
              for (int r = 0; r < kRowsOut; ++r) p[r * o.ld] = v[r];
            } else {
#pragma unroll
              for (int r = 0; r < kRowsOut; ++r)
                if (r0 + r < rows) p[r * o.ld] = v[r];
            }
            p += kRowsOut * o.ld;
          }
        }
      }
      __syncwarp();
    }
  }
}

template <bool A_MN, bool B_MN, bool kPair, int kOut, bool kByRow>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB,
                const __grid_constant__ CUtensorMap mapOut, GemmGeom g, Scales sa, Scales sb, Out out, int* status) {
  extern __shared__ uint8_t smem_raw[];
  using TL = Tile<kPair>;
  constexpr int kStages = TL::kStages, kStageBytes = TL::kStageBytes, kABytes = TL::kABytes;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* out_smem = smem + kOperandBytes;
  tc::Barriers* bars = reinterpret_cast<tc::Barriers*>(out_smem + kEpiWarps * kOutBytes);
  using Ring = ScaleRing<kByRow>;
  constexpr int kSlots = Ring::kSlots, window = Ring::kWindow;
  Ring* ring = reinterpret_cast<Ring*>(out_smem + kEpiWarps * kOutBytes + 256);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  const int rank = kPair ? (int)(blockIdx.x & 1) : 0;
  const int worker = kPair ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int workers = kPair ? (int)(gridDim.x >> 1) : (int)gridDim.x;
  const int m_tiles = (g.M + TL::kM - 1) / TL::kM;
  const int n_tiles = (g.N + kBN - 1) / kBN;
  const int tiles_per_slab = m_tiles * n_tiles;
  const int total_tiles = tiles_per_slab * g.nz;
  const int kb_per_seg = (g.Kseg + kBK - 1) / kBK;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      tc::mbar_init(tc::smem_u32(&bars->full[i]), 1);
      tc::mbar_init(tc::smem_u32(&bars->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(tc::smem_u32(&bars->tmem_full[i]), 1);
      tc::mbar_init(tc::smem_u32(&bars->tmem_empty[i]), TL::kCtas * kEpiWarps);
    }
    for (int i = 0; i < kSlots; ++i) {
      tc::mbar_init(tc::smem_u32(&ring->full[i]), kScaleWarps);
      // the epilogue and, of the leader and where blocks are joined, the MMA warp
      tc::mbar_init(tc::smem_u32(&ring->empty[i]), kEpiWarps + (rank == 0 && !kByRow ? 1 : 0));
    }
    bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    tc::tmem_alloc<kPair>(tc::smem_u32(&bars->tmem_base), kTmemCols);
    tc::tmem_relinquish<kPair>();
  }
  tc::tc_fence_before();
  if constexpr (kPair)
    tc::cluster_sync();
  else
    __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = bars->tmem_base;

  if (warp < kFirstEpiWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLean));
    if (warp == 0) {
      // ------------------------------ TMA producer ------------------------------
      const bool one = elect_one();
      const uint32_t full0 = tc::smem_u32(&bars->full[0]), empty0 = tc::smem_u32(&bars->empty[0]);
      const uint32_t lead0 = kPair ? tc::cluster_addr(full0, 0) : full0;  // the leader's barriers count the bytes of both
      const uint32_t stage0 = tc::smem_u32(smem);
      int stage = 0;
      uint32_t phase = 0;
      bool alive = true;
      for (int i = 0; alive; ++i) {
        const long long tile_l = tc::tile_of_round(i, worker, workers);
        if (tile_l >= total_tiles) break;
        const int tile = (int)tile_l;
        int z, kb_lo, kb_hi, zo;
        work_item(g, tile / tiles_per_slab, kb_per_seg, z, kb_lo, kb_hi, zo);
        int m0, n0;
        tc::tile_origin(tile % tiles_per_slab, m_tiles, n_tiles, TL::kM, m0, n0);
        m0 += rank * kBM;
        n0 += rank * TL::kBRows;
        int left = kb_hi - kb_lo, kb0 = kb_lo % kb_per_seg;
        for (int j = kb_lo / kb_per_seg; left > 0 && alive; ++j) {
          int za, zb;
          seg_index(g, z, j, za, zb);
          const int kb1 = min(kb_per_seg, kb0 + left);
          left -= kb1 - kb0;
          for (int kb = kb0; kb < kb1; ++kb) {
            // (the vote: lanes that give up a wait at different times leave together)
            alive = __all_sync(0xffffffffu, wait(empty0 + 8 * stage, phase ^ 1, abort_flag, status, kTimeoutEmpty));
            if (!alive) break;
            if (one) {
              const uint32_t full = lead0 + 8 * stage;
              if (rank == 0) tc::mbar_expect_tx(full0 + 8 * stage, TL::kCtas * kStageBytes);
              const uint32_t pa = stage0 + stage * kStageBytes;
              const uint32_t pb = pa + kABytes;
              const int k0 = kb * kBK;
              if (A_MN)
                tc::tma_load_3d<kPair>(pa, &mapA, full, m0, k0, za);
              else
                tc::tma_load_3d<kPair>(pa, &mapA, full, k0, m0, za);
              if (B_MN) {
#pragma unroll
                for (int b = 0; b < TL::kBRows / 128; ++b)
                  tc::tma_load_3d<kPair>(pb + b * kBox, &mapB, full, n0 + 128 * b, k0, zb);
              } else {
                tc::tma_load_3d<kPair>(pb, &mapB, full, k0, n0, zb);
              }
            }
            __syncwarp();
            if (++stage == kStages) stage = 0, phase ^= 1;
          }
          kb0 = 0;
        }
      }
      if constexpr (kPair) {
        // the leader's MMAs read this CTA's stages and its commits arrive here: stay until the last has
        for (int i = 0; i < kStages && alive; ++i) {
          alive = wait(empty0 + 8 * stage, phase ^ 1, abort_flag, status, kTimeoutEmpty);
          if (++stage == kStages) stage = 0, phase ^= 1;
        }
      }
      if (!alive) {
        // let copies that are still in flight land before the CTA's shared memory goes away
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000ll) {
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------ MMA issuer --------------------------------
      if (rank == 0) {
        constexpr uint32_t idesc = instr_desc(A_MN, B_MN, TL::kM);
        const bool one = elect_one();
        const uint32_t full0 = tc::smem_u32(&bars->full[0]), empty0 = tc::smem_u32(&bars->empty[0]);
        const uint32_t acc_full0 = tc::smem_u32(&bars->tmem_full[0]), acc_empty0 = tc::smem_u32(&bars->tmem_empty[0]);
        // descriptors of the first stage; a stage further, or a K step, moves their addresses (in 16-byte units)
        const uint64_t da0 = A_MN ? tc::smem_desc(tc::smem_u32(smem), kBox, 1024) : tc::smem_desc(tc::smem_u32(smem), 16, 1024);
        const uint64_t db0 = B_MN ? tc::smem_desc(tc::smem_u32(smem) + kABytes, kBox, 1024)
                                  : tc::smem_desc(tc::smem_u32(smem) + kABytes, 16, 1024);
        constexpr int kStepA = (A_MN ? 4096 : 32) / 16, kStepB = (B_MN ? 4096 : 32) / 16;
        int stage = 0;
        uint32_t phase = 0;
        uint32_t n = 0, batch = 0;  // groups so far: accumulator n & 1, used for the (n >> 1)-th time; windows so far
        bool alive = true;
        for (int it = 0; alive; ++it) {
          const long long tile_l = tc::tile_of_round(it, worker, workers);
          if (tile_l >= total_tiles) break;
          int z, kb_lo, kb_hi, zo;
          work_item(g, (int)tile_l / tiles_per_slab, kb_per_seg, z, kb_lo, kb_hi, zo);
          for (int left = kb_hi - kb_lo; left > 0 && alive; left -= window, ++batch) {
            const int slot = batch % kSlots, in_window = min(left, window);
            uint32_t starts = 0xffffffffu;
            if constexpr (!kByRow) {
              alive = __all_sync(0xffffffffu, wait(tc::smem_u32(&ring->full[slot]), (batch / kSlots) & 1, abort_flag, status, kTimeoutFull));
              if (!alive) break;
              starts = ring->starts[slot];
            }
            for (int i = 0; i < in_window; ++i) {
              const uint32_t buf = n & 1;
              const bool first = starts >> i & 1, last = i + 1 == in_window || (starts >> (i + 1) & 1);
              const bool ok = (!first || wait(acc_empty0 + 8 * buf, ((n >> 1) & 1) ^ 1, abort_flag, status, kTimeoutTmemEmpty)) &&
                              wait(full0 + 8 * stage, phase, abort_flag, status, kTimeoutFull);
              alive = __all_sync(0xffffffffu, ok);
              if (!alive) break;
              tc::tc_fence_after();
              if (one) {
                const uint32_t tmem_d = tmem_base + buf * kBN;
                const uint64_t da = da0 + (uint32_t)(stage * (kStageBytes / 16)), db = db0 + (uint32_t)(stage * (kStageBytes / 16));
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k)
                  umma_e4m3<kPair>(tmem_d, da + k * kStepA, db + k * kStepB, idesc, k > 0 || !first ? 1u : 0u);
                tc::umma_commit<kPair>(empty0 + 8 * stage);
                if (last) tc::umma_commit<kPair>(acc_full0 + 8 * buf);
              }
              __syncwarp();
              if (++stage == kStages) stage = 0, phase ^= 1;
              if (last) ++n;
            }
            __syncwarp();
            if (lane == 0 && !kByRow) tc::mbar_arrive(tc::smem_u32(&ring->empty[slot]));
          }
          alive = __all_sync(0xffffffffu, alive);
        }
      }
      __syncwarp();
    } else {
      // ------------------------------ scales ------------------------------------
      const int t = threadIdx.x - 64;  // rows t and t + 64 of the CTA's 128
      uint32_t batch = 0;
      bool alive = true;
      for (int it = 0; alive; ++it) {
        const long long tile_l = tc::tile_of_round(it, worker, workers);
        if (tile_l >= total_tiles) break;
        const int tile = (int)tile_l;
        int z, kb_lo, kb_hi, zo, m0, n0;
        work_item(g, tile / tiles_per_slab, kb_per_seg, z, kb_lo, kb_hi, zo);
        tc::tile_origin(tile % tiles_per_slab, m_tiles, n_tiles, TL::kM, m0, n0);
        // rows and columns behind the end take the last ones' scales: their sums are not stored
        const auto row_of = [&](int m) { return sa.p + (long long)(min(m, g.M - 1) >> sa.shift) * sa.mn; };
        const float* b0 = sb.p + (long long)(min(n0, g.N - 1) >> 7) * sb.mn;
        const float* b1 = sb.p + (long long)(min(n0 + 128, g.N - 1) >> 7) * sb.mn;
        // by row: this thread's rows t and t + 64 of the CTA's and a half of the columns, from block `at` on
        const float *pa0 = nullptr, *pa1 = nullptr, *pb = nullptr;
        int seg_left = 0;
        const auto segment = [&](int at) {
          const int j = at / kb_per_seg, kb = at - j * kb_per_seg;
          int za, zb;
          seg_index(g, z, j, za, zb);
          const long long oa = za * sa.z + kb * sa.k;
          pa0 = row_of(m0 + rank * kBM + t) + oa, pa1 = row_of(m0 + rank * kBM + t + 64) + oa;
          pb = (t & 1 ? b1 : b0) + zb * sb.z + kb * sb.k;
          seg_left = kb_per_seg - kb;
        };
        for (int at = kb_lo; at < kb_hi; at += window, ++batch) {
          const int slot = batch % kSlots, n = min(kb_hi - at, window);
          const bool ok =
              wait(tc::smem_u32(&ring->empty[slot]), ((batch / kSlots) & 1) ^ 1, abort_flag, status, kTimeoutTmemEmpty);
          alive = __all_sync(0xffffffffu, ok);
          if (!alive) break;
          if (t == 0 && at == kb_lo) ring->tile[slot] = make_int4(m0 + rank * kBM, n0, zo, kb_hi - kb_lo);
          if (out.bias != nullptr && at == kb_lo) {
            // with the tile's first window; the tile kSlots before took its own before it gave a window back
#pragma unroll
            for (int i = 0; i < kBN; i += 64)
              ring->bias[it % kSlots][i + t] = n0 + i + t < g.N ? __ldg(out.bias + zo * out.bias_z + n0 + i + t) : 0.f;
          }
          if constexpr (kByRow) {
            float va[window], vb[window], vc[window];
#pragma unroll
            for (int i = 0; i < window; ++i) {
              if (i < n) {
                if (seg_left == 0) segment(at + i);
                va[i] = __ldg(pa0), vb[i] = __ldg(pa1);
                vc[i] = t < 2 ? __ldg(pb) : 0.f;
                pa0 += sa.k, pa1 += sa.k, pb += sb.k, --seg_left;
              }
            }
            bool far = false;
#pragma unroll
            for (int i = 0; i < window; ++i) {
              if (i < n) {
                ring->a[slot][i * 128 + t] = va[i], ring->a[slot][i * 128 + t + 64] = vb[i];
                far |= far_from_one(va[i]) || far_from_one(vb[i]);
                if (t < 2) ring->b[slot][i][t] = vc[i], far |= far_from_one(vc[i]);
              }
            }
            far = __any_sync(0xffffffffu, far);
            if (lane == 0) ring->far[slot][warp - 2] = far;
          } else if (warp == 2) {
            // lane i has block at + i: its scales of both CTAs' rows and of both halves of the columns
            float v[4] = {};
            if (lane < n) {
              const int j = (at + lane) / kb_per_seg, kb = at + lane - j * kb_per_seg;
              int za, zb;
              seg_index(g, z, j, za, zb);
              v[0] = __ldg(row_of(m0) + za * sa.z + kb * sa.k);
              v[1] = kPair ? __ldg(row_of(m0 + kBM) + za * sa.z + kb * sa.k) : v[0];
              v[2] = __ldg(b0 + zb * sb.z + kb * sb.k);
              v[3] = __ldg(b1 + zb * sb.z + kb * sb.k);
            }
            bool differs = lane == 0, far = false;
#pragma unroll
            for (int i = 0; i < 4; ++i) far |= lane < n && far_from_one(v[i]);
            far = __any_sync(0xffffffffu, far);
#pragma unroll
            for (int i = 0; i < 4; ++i) differs |= !(v[i] == __shfl_up_sync(0xffffffffu, v[i], 1));
            const uint32_t changes = __ballot_sync(0xffffffffu, differs && lane < n);
            uint32_t starts = 0;
            for (int p = 0; p < n;) {
              starts |= 1u << p;
              const uint32_t later = changes & ~((2u << p) - 1);
              const int next = later != 0 ? __ffs(later) - 1 : n;
              p = min(next, p + kMostJoined);
            }
            if (starts >> lane & 1) {
              const int group = __popc(starts & ((1u << lane) - 1));
              ring->a[slot][group] = rank == 0 ? v[0] : v[1];
              ring->b[slot][group][0] = v[2], ring->b[slot][group][1] = v[3];
            }
            if (lane == 0) ring->starts[slot] = starts, ring->far[slot][0] = far, ring->far[slot][1] = 0;
          }
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(tc::smem_u32(&ring->full[slot]));
        }
      }
      const int slot = batch % kSlots;
      const bool ok =
          alive && wait(tc::smem_u32(&ring->empty[slot]), ((batch / kSlots) & 1) ^ 1, abort_flag, status, kTimeoutTmemEmpty);
      if (__all_sync(0xffffffffu, ok)) {
        if (t == 0) ring->tile[slot] = make_int4(0, 0, 0, 0);
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&ring->full[slot]));
      }
    }
  } else {
    // ------------------------------ epilogue ----------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int ew = warp - kFirstEpiWarp;
    uint8_t* buf8 = out_smem + ew * kOutBytes;
    const auto window_ready = [&](uint32_t batch) {
      const bool ok = wait(tc::smem_u32(&ring->full[batch % kSlots]), (batch / kSlots) & 1, abort_flag, status, kTimeoutTmemFull);
      return (bool)__all_sync(0xffffffffu, ok);
    };
    const int quarter = warp & 3;  // tensor-memory lanes 32*quarter .. +31
    const int half = ew >> 2;      // which 128 columns of the tile
    const uint32_t tbase = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
    uint32_t n = 0, batch = 0;
    bool alive = true;
    // Which tile comes next arrives with its scales: the divisions that it takes are not made here, where the tensor cores would wait.
    for (int it = 0; alive; ++it) {
      if (!window_ready(batch)) break;
      const int4 tile = ring->tile[batch % kSlots];
      if (tile.w == 0) break;
      const int row0 = tile.x + quarter * 32, col0 = tile.y + half * 128, zo = tile.z;
      const bool work = row0 < g.M && col0 < g.N;  // uniform over the warp: something of it is stored
      uint32_t r0[16], r1[16];
      // One read of tensor memory is in flight at any time, across the blocks: the next block's first is issued before this
      // block's last columns are added.
      alive = block_ready(bars, n, abort_flag, status);
      if (alive && work) tmem_ld16_issue(tbase + (n & 1) * kBN, r0);
      float acc[128];
      if (out.bias != nullptr) {
        const float* bias = ring->bias[it % kSlots] + half * 128;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const float4 b = *reinterpret_cast<const float4*>(bias + 4 * i);
          acc[4 * i] = b.x, acc[4 * i + 1] = b.y, acc[4 * i + 2] = b.z, acc[4 * i + 3] = b.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 128; ++i) acc[i] = 0.f;
      }
#pragma unroll 1
      for (int left = tile.w; left > 0 && alive; left -= window, ++batch) {
        const int slot = batch % kSlots;
        if (left < tile.w) alive = window_ready(batch);
        const float* ra = ring->a[slot] + (kByRow ? quarter * 32 + lane : 0);
        const float* rb = &ring->b[slot][0][half];
        const bool far = (ring->far[slot][0] | ring->far[slot][1]) != 0;
        const int groups = kByRow ? min(left, window) : __popc(ring->starts[slot]);
        // Where the scale warps found a scale far from one, one scale is applied after the other (Factors).  That is a loop of its
        // own: 12 x 4000 x 768 x 24576 by rows 1193 us (1174 without such scales being provided for; 1556 where all are such),
        // 1216 with a look at every product inside one loop, 1236 with the flag there.
        const auto blocks = [&](auto kind) {
          constexpr bool split = decltype(kind)::value;
#pragma unroll 1
          for (int i = 0; alive && i < groups; ++i, ++n) {
            float s = ra[kByRow ? i * 128 : i] * rb[i * 2], first = 1.f;
            if constexpr (split) {
              const Factors f(ra[kByRow ? i * 128 : i], rb[i * 2]);
              first = f.first, s = f.second;
            }
            const int buf = n & 1;
            const uint32_t taddr = tbase + buf * kBN;
            if (work) {
#pragma unroll
              for (int c = 0; c < 8; c += 2) {
                tmem_ld_wait(r0);
                tmem_ld16_issue(taddr + 16 * (c + 1), r1);
                if constexpr (split) mul16(r0, first);
                fma16(acc + 16 * c, r0, s);
                tmem_ld_wait(r1);
                if constexpr (split) mul16(r1, first);
                if (c < 6) {
                  tmem_ld16_issue(taddr + 16 * (c + 2), r0);
                  fma16(acc + 16 * (c + 1), r1, s);
                }
              }
            }
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (kPair)
                arrive_remote(tc::cluster_addr(tc::smem_u32(&bars->tmem_empty[buf]), 0));
              else
                tc::mbar_arrive(tc::smem_u32(&bars->tmem_empty[buf]));
            }
            if (i + 1 < groups || left > window) {
              alive = block_ready(bars, n + 1, abort_flag, status);
              if (alive && work) tmem_ld16_issue(tbase + ((n + 1) & 1) * kBN, r0);
            }
            if (work) fma16(acc + 112, r1, s);
          }
        };
        if (far)
          blocks(std::true_type());
        else
          blocks(std::false_type());
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(tc::smem_u32(&ring->empty[slot]));
        if (left <= window && alive && work) store_warp<kOut>(acc, buf8, &mapOut, out, zo, row0, col0, g.M, g.N);
      }
    }
  }

  if (warp >= kFirstEpiWarp && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  tc::tc_fence_before();
  if constexpr (kPair)
    tc::cluster_sync();
  else
    __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after();
    tc::tmem_dealloc<kPair>(tmem_base, kTmemCols);
  }
}

}  // namespace f8
}  // namespace clt
