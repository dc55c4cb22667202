// Product of two 8-bit (e4m3) operands with a scale for each block of 128, on the 5th-generation tensor cores:
//
//   out[z, m, n] = bias[z, n] + sum over the segments and 128-wide blocks kb of z's contraction
//                  sa[m, kb] * sb[kb, n / 128] * sum_{k in kb} A[m, k] B[k, n]
//
// A's scales belong to 1 x 128 or 128 x 128 blocks, B's to 128 x 128 blocks.  The inner sum runs in tensor memory (four
// MMAs of 32); its 128 x 256 results then go through registers once, where they are scaled and added in fp32.  So a sum in
// the tensor cores' own accumulator has 128 terms however long the contraction is, and any fp32 scales will do.
//
// Roles, barriers, operand layouts and pairs of CTAs are those of gemm_tc.cuh.  What differs:
//   * A stage holds 128 of the contraction axis, one byte each: as many bytes as 64 bf16 values, twice the products.
//   * The two accumulators of tensor memory alternate from block to block instead of from tile to tile: while the MMAs fill
//     one, the eight epilogue warps read the other and add it to their 128 sums a thread (32 rows x 128 columns a warp).
//     That is 16384 packed FMAs a block and SM, 256 cycles of the fp32 pipes beside 512 of the tensor cores.
//   * MN-major operands come in boxes of 128(MN) x 128(K): K rows of 128 B, 8-row groups 1024 B apart, boxes 16 KB apart; the
//     32-wide K step of one MMA moves the start address by 4096 B (K-major: by 32 B).
//
// No TMA load uses cluster multicast.  Every wait is bounded as there.
#pragma once

#include <cuda_fp16.h>

#include "gemm_tc.cuh"

namespace clt {
namespace f8 {

using tc::kBM;
using tc::kBN;
using tc::kEpiThreads;
using tc::kEpiWarps;
using tc::kFirstEpiWarp;
using tc::kMaxStages;
using tc::kRegsEpi;
using tc::kRegsLean;
using tc::kThreads;
using tc::kTmemCols;
constexpr int kBK = 128;         // contraction of a stage = of a scale block
constexpr int kBox = 128 * 128;  // bytes of one box

template <bool kPair>
struct Tile {
  static constexpr int kCtas = kPair ? 2 : 1;
  static constexpr int kM = kCtas * kBM;
  static constexpr int kBRows = kBN / kCtas;
  static constexpr int kABytes = kBM * kBK;
  static constexpr int kBBytes = kBRows * kBK;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = kPair ? 6 : 4;
};
constexpr int kOperandBytes = Tile<true>::kStages * Tile<true>::kStageBytes;
static_assert(kOperandBytes == Tile<false>::kStages * Tile<false>::kStageBytes, "both forms fill the same memory");
constexpr int kBiasBytes = kEpiWarps * 128 * 4;  // each warp's own columns
constexpr int kSmemBytes =
    kOperandBytes + 1024 /*alignment slack*/ + 256 /*barriers*/ + kBiasBytes + kEpiWarps * epi::kStageBytes;
static_assert(sizeof(tc::Barriers) <= 256, "barriers");

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
  int aligned;  // rows of every slab start on 16 bytes
};

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

__device__ __forceinline__ void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// Waits for this warp's reads of tensor memory.  The registers are operands so that nothing that uses them is moved ahead.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t d, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(d));
}
// acc += d * s, two at a time
__device__ __forceinline__ void fma16(uint64_t* acc, const uint32_t (&d)[16], uint64_t s2) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[i]) : "l"(pack2(d[2 * i], d[2 * i + 1])), "l"(s2));
}

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

// A warp's 32 x 32 sub-tile of 16-bit values, as epi::store_rows32; rows that are not 16-byte aligned or that end inside the
// sub-tile go out one row to an instruction.
template <class T>
__device__ __forceinline__ void store16(unsigned char* stage, T* base, long long ld, int rows_valid, int cols_valid,
                                        bool aligned, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  uint4* mine = reinterpret_cast<uint4*>(stage + lane * epi::kStageRow);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    mine[i] = make_uint4(pack16<T>(v[8 * i], v[8 * i + 1]), pack16<T>(v[8 * i + 2], v[8 * i + 3]),
                         pack16<T>(v[8 * i + 4], v[8 * i + 5]), pack16<T>(v[8 * i + 6], v[8 * i + 7]));
  __syncwarp();
  if (aligned && cols_valid >= 32) {
    const int piece = lane & 3;
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      const int r = it * 8 + (lane >> 2);
      const uint4 t = *reinterpret_cast<const uint4*>(stage + r * epi::kStageRow + piece * 16);
      if (r < rows_valid) *reinterpret_cast<uint4*>(base + r * ld + piece * 8) = t;
    }
  } else if (lane < cols_valid) {
#pragma unroll 4
    for (int r = 0; r < 32; ++r)
      if (r < rows_valid) base[r * ld + lane] = *reinterpret_cast<const T*>(stage + r * epi::kStageRow + lane * 2);
  }
  __syncwarp();
}

__device__ __forceinline__ void store_chunk(unsigned char* stage, const Out& o, int z, int row0, int n, int M, int N,
                                            const float (&v)[32]) {
  const long long at = z * o.z + (long long)row0 * o.ld + n;
  const int rows = M - row0, cols = N - n;
  if (o.dtype == 0) {
    float* p = (float*)o.p + at;
    if (o.aligned && cols >= 32)
      epi::store_rows32<float>(stage, p, (size_t)o.ld, rows, v);
    else
      epi::store_rows32_scalar(stage, p, (size_t)o.ld, rows, cols, v);
  } else if (o.dtype == 1) {
    store16<__half>(stage, (__half*)o.p + at, o.ld, rows, cols, o.aligned != 0, v);
  } else {
    store16<__nv_bfloat16>(stage, (__nv_bfloat16*)o.p + at, o.ld, rows, cols, o.aligned != 0, v);
  }
}

template <bool A_MN, bool B_MN, bool kPair>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, GemmGeom g,
                Scales sa, Scales sb, Out out, int* status) {
  extern __shared__ uint8_t smem_raw[];
  using TL = Tile<kPair>;
  constexpr int kStages = TL::kStages, kStageBytes = TL::kStageBytes, kABytes = TL::kABytes;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  tc::Barriers* bars = reinterpret_cast<tc::Barriers*>(smem + kOperandBytes);
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
      if (lane == 0) {
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
              if (!tc::mbar_wait(tc::smem_u32(&bars->empty[stage]), phase ^ 1, abort_flag, status, kTimeoutEmpty)) {
                alive = false;
                break;
              }
              const uint32_t own = tc::smem_u32(&bars->full[stage]), full = kPair ? tc::cluster_addr(own, 0) : own;
              if (rank == 0) tc::mbar_expect_tx(own, TL::kCtas * kStageBytes);
              const uint32_t pa = tc::smem_u32(smem + stage * kStageBytes);
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
              if (++stage == kStages) stage = 0, phase ^= 1;
            }
            kb0 = 0;
          }
        }
        if constexpr (kPair) {
          // the leader's MMAs read this CTA's stages and its commits arrive here: stay until the last has
          for (int i = 0; i < kStages && alive; ++i) {
            alive = tc::mbar_wait(tc::smem_u32(&bars->empty[stage]), phase ^ 1, abort_flag, status, kTimeoutEmpty);
            if (++stage == kStages) stage = 0, phase ^= 1;
          }
        }
        if (!alive) {
          // let copies that are still in flight land before the CTA's shared memory goes away
          const long long t0 = clock64();
          while (clock64() - t0 < 2000000ll) {
          }
        }
      }
      __syncwarp();
    } else if (warp == 1) {
      // ------------------------------ MMA issuer --------------------------------
      if (lane == 0 && rank == 0) {
        constexpr uint32_t idesc = instr_desc(A_MN, B_MN, TL::kM);
        int stage = 0;
        uint32_t phase = 0;
        uint32_t n = 0;  // blocks so far: accumulator n & 1, used for the (n >> 1)-th time
        bool alive = true;
        for (int it = 0; alive; ++it) {
          const long long tile_l = tc::tile_of_round(it, worker, workers);
          if (tile_l >= total_tiles) break;
          int z, kb_lo, kb_hi, zo;
          work_item(g, (int)tile_l / tiles_per_slab, kb_per_seg, z, kb_lo, kb_hi, zo);
          for (int kb = kb_lo; kb < kb_hi; ++kb, ++n) {
            const int buf = n & 1;
            if (!tc::mbar_wait(tc::smem_u32(&bars->tmem_empty[buf]), ((n >> 1) & 1) ^ 1, abort_flag, status,
                               kTimeoutTmemEmpty) ||
                !tc::mbar_wait(tc::smem_u32(&bars->full[stage]), phase, abort_flag, status, kTimeoutFull)) {
              alive = false;
              break;
            }
            tc::tc_fence_after();
            const uint32_t pa = tc::smem_u32(smem + stage * kStageBytes);
            const uint32_t pb = pa + kABytes;
            const uint32_t tmem_d = tmem_base + buf * kBN;
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k) {
              const uint64_t da =
                  A_MN ? tc::smem_desc(pa + k * 4096, kBox, 1024) : tc::smem_desc(pa + k * 32, 16, 1024);
              const uint64_t db =
                  B_MN ? tc::smem_desc(pb + k * 4096, kBox, 1024) : tc::smem_desc(pb + k * 32, 16, 1024);
              umma_e4m3<kPair>(tmem_d, da, db, idesc, k > 0 ? 1u : 0u);
            }
            tc::umma_commit<kPair>(tc::smem_u32(&bars->empty[stage]));
            tc::umma_commit<kPair>(tc::smem_u32(&bars->tmem_full[buf]));
            if (++stage == kStages) stage = 0, phase ^= 1;
          }
        }
      }
      __syncwarp();
    }
  } else {
    // ------------------------------ epilogue ----------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsEpi));
    const int ew = warp - kFirstEpiWarp;
    float* bias = reinterpret_cast<float*>(smem + kOperandBytes + 256) + ew * 128;
    unsigned char* stage = smem + kOperandBytes + 256 + kBiasBytes + ew * epi::kStageBytes;
    const int quarter = warp & 3;  // tensor-memory lanes 32*quarter .. +31
    const int half = ew >> 2;      // which 128 columns of the tile
    const uint32_t tbase = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(half * 128);
    uint32_t n = 0;
    bool alive = true;
    for (int it = 0; alive; ++it) {
      const long long tile_l = tc::tile_of_round(it, worker, workers);
      if (tile_l >= total_tiles) break;
      const int tile = (int)tile_l;
      int z, kb_lo, kb_hi, zo;
      work_item(g, tile / tiles_per_slab, kb_per_seg, z, kb_lo, kb_hi, zo);
      int m0, n0;
      tc::tile_origin(tile % tiles_per_slab, m_tiles, n_tiles, TL::kM, m0, n0);
      const int row0 = m0 + rank * kBM + quarter * 32, col0 = n0 + half * 128;
      const bool work = row0 < g.M && col0 < g.N;  // uniform over the warp: something of it is stored
      const long long sa_row = (long long)(min(row0 + lane, g.M - 1) >> sa.shift) * sa.mn;
      const long long sb_col = (long long)(min(col0, g.N - 1) >> 7) * sb.mn;
      if (work && out.bias != nullptr) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int c = col0 + 32 * i + lane;
          bias[32 * i + lane] = c < g.N ? __ldg(out.bias + zo * out.bias_z + c) : 0.f;
        }
        __syncwarp();
      }
      uint64_t acc[64];
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i] = 0;
      int j = kb_lo / kb_per_seg, kb = kb_lo % kb_per_seg;
      const float *pa, *pb;
      float s_next = 0.f;
      const auto segment = [&]() {
        int za, zb;
        seg_index(g, z, j, za, zb);
        pa = sa.p + za * sa.z + sa_row + kb * sa.k;
        pb = sb.p + zb * sb.z + sb_col + kb * sb.k;
      };
      segment();
      if (work) s_next = __ldg(pa) * __ldg(pb);
#pragma unroll 1
      for (int left = kb_hi - kb_lo; left > 0; --left, ++n) {
        const float s = s_next;
        // the next block's scale is on its way while this block is multiplied
        if (left > 1) {
          if (++kb == kb_per_seg) {
            kb = 0, ++j;
            segment();
          } else {
            pa += sa.k, pb += sb.k;
          }
          if (work) s_next = __ldg(pa) * __ldg(pb);
        }
        const int buf = n & 1;
        const bool ok =
            tc::mbar_wait(tc::smem_u32(&bars->tmem_full[buf]), (n >> 1) & 1, abort_flag, status, kTimeoutTmemFull);
        if (!__all_sync(0xffffffffu, ok)) {
          alive = false;
          break;
        }
        tc::tc_fence_after();
        const uint64_t s2 = pack2(__float_as_uint(s), __float_as_uint(s));
        const uint32_t taddr = tbase + buf * kBN;
        uint32_t r0[16], r1[16];
        if (work) {
          tmem_ld16_issue(taddr, r0);
#pragma unroll
          for (int c = 0; c < 8; c += 2) {
            tmem_ld_wait(r0);
            tmem_ld16_issue(taddr + 16 * (c + 1), r1);
            fma16(acc + 8 * c, r0, s2);
            tmem_ld_wait(r1);
            if (c + 2 < 8) {
              tmem_ld16_issue(taddr + 16 * (c + 2), r0);
              fma16(acc + 8 * (c + 1), r1, s2);
            }
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (kPair)
            tc::mbar_arrive_cluster(tc::cluster_addr(tc::smem_u32(&bars->tmem_empty[buf]), 0));
          else
            tc::mbar_arrive(tc::smem_u32(&bars->tmem_empty[buf]));
        }
        if (work) fma16(acc + 56, r1, s2);
      }
      if (!alive || !work) continue;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        if (col0 + 32 * c < g.N) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) unpack2(acc[16 * c + i], v[2 * i], v[2 * i + 1]);
          if (out.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float4 b = *reinterpret_cast<const float4*>(bias + 32 * c + 4 * i);
              v[4 * i] += b.x, v[4 * i + 1] += b.y, v[4 * i + 2] += b.z, v[4 * i + 3] += b.w;
            }
          }
          store_chunk(stage, out, zo, row0, col0 + 32 * c, g.M, g.N, v);
        }
      }
    }
  }

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
