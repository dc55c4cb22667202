// C entry points of the 8-bit contraction: geometry, operand descriptions, parts of long contractions.
#include "../../include/clt_b200.h"
#include "gemm_fp8.cuh"
#include "kernels.h"

using namespace clt;

namespace {

inline long long up(long long a, long long b) { return (a + b - 1) / b; }

// Pairs of CTAs where rounding the rows up to 256 adds at most an eighth.  (They are about as fast a block as single CTAs, and
// take a third less from L2.)
bool pair_rows(int M) { return up(M, 256) * 16 <= up(M, 128) * 9; }
bool use_pair(const GemmGeom& g, int sms) {
  return pair_rows(g.M) && up(g.M, 256) * up(g.N, f8::kBN) * g.nz >= sms / 2;
}

// Cuts the contraction into parts (gemm.cuh) where that is estimated faster; sets g.kb_per_part and returns the number of parts, or
// 0 for whole chains.  Estimates, in us: 0.45 a block of 128 x 256 x 128 (a CTA's, or a pair's of 256 rows; what joined blocks
// take.  Separate ones take 0.60, which the plan does not know: it gets no scales), 1.5 a tile for its
// output and the next one's start; partial sums go to memory and back at 5 TB/s, behind a launch of 4.  Parts are tried that
// fill 1 to 8 rounds of the chip: 257 x 120000 x 768 in 17 parts of 58 blocks, 153 tiles, took 47 us, in 16 of 59, one
// round, 42 (the product by itself; the call 49 on the device with the parts' sum and the gap between the two launches); whole
// chains 500.
int plan_parts(GemmGeom& g, int sms) {
  const int kb_per_seg = (int)up(g.Kseg, f8::kBK);
  const bool pair = pair_rows(g.M);
  const long long tiles = up(g.M, pair ? 256 : 128) * up(g.N, f8::kBN), workers = pair ? sms / 2 : sms;
  long long total = 0, longest = 0;
  for (int z = 0; z < g.nz; ++z) {
    const long long n = (long long)seg_count(g, z) * kb_per_seg;
    total += n;
    longest = n > longest ? n : longest;
  }
  g.kb_per_part = 0;
  if (longest < 8) return 0;
  const double block = 0.45, tile = 1.5;
  // equal chains run in rounds, unequal ones are dealt out longest first
  const double whole = longest * g.nz == total
                           ? up(tiles * g.nz, workers) * (longest * block + tile)
                           : fmax(longest * block + tile, (total * block + g.nz * tile) * tiles / workers);
  double best = 0.95 * whole;
  int best_part = 0;
  for (int rounds = 1; rounds <= 8; ++rounds) {
    const long long room = rounds * workers / tiles;  // parts that these rounds have room for
    if (room <= g.nz) continue;
    GemmGeom h = g;
    long long parts = 0;
    const long long least = up(total, room);
    if (longest * g.nz == total) {
      const long long each = room / g.nz;  // parts of a slab
      if (each < 2) continue;
      h.kb_per_part = (int)(up(longest, each) < 4 ? 4 : up(longest, each));
      parts = g.nz * up(longest, h.kb_per_part);
    } else {
      // (grows by the slabs' last, shorter parts: a few steps)
      for (long long p = least < 4 ? 4 : least; p < longest; p += 1 + p / 64) {
        h.kb_per_part = (int)p;
        parts = 0;
        for (int z = 0; z < g.nz; ++z) parts += part_count(h, z, kb_per_seg);
        if (parts <= room) break;
      }
    }
    if (parts <= g.nz || parts > room || parts > 65535) continue;
    const double us = rounds * (h.kb_per_part * block + tile) + 4.0 + 8.0 * parts * g.M * g.N / 5e6;
    if (us < best) best = us, best_part = h.kb_per_part;
  }
  if (best_part == 0) return 0;
  g.kb_per_part = best_part;
  int parts = 0;
  for (int z = 0; z < g.nz; ++z) parts += part_count(g, z, kb_per_seg);
  return parts;
}

template <class T>
struct FromFloat;
template <>
struct FromFloat<float> {
  __device__ static float get(float v) { return v; }
};
template <>
struct FromFloat<__half> {
  __device__ static __half get(float v) { return __float2half_rn(v); }
};
template <>
struct FromFloat<__nv_bfloat16> {
  __device__ static __nv_bfloat16 get(float v) { return __float2bfloat16_rn(v); }
};

// out[z, m, n] = bias[z, n] + the partial sums of z's parts, in their order.  V consecutive n to a thread (N a multiple of V).
template <class T, int V>
__global__ void __launch_bounds__(128) fp8_sum_parts_kernel(const float* __restrict__ ws, f8::Out out, GemmGeom g, int kb_per_seg) {
  const int z = blockIdx.y;
  const long long slab = (long long)g.M * g.N, i = (blockIdx.x * 128ll + threadIdx.x) * V;
  if (i >= slab) return;
  int first = 0;
  for (int u = 0; u < z; ++u) first += part_count(g, u, kb_per_seg);
  const int parts = part_count(g, z, kb_per_seg);
  const long long m = i / g.N;
  const int n = (int)(i - m * g.N);
  const float* p = ws + first * slab + i;
  float acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = out.bias != nullptr ? __ldg(out.bias + z * out.bias_z + n + k) : 0.f;
#pragma unroll 8
  for (int j = 0; j < parts; ++j) {
    if constexpr (V == 4) {
      const float4 v = __ldcs(reinterpret_cast<const float4*>(p + j * slab));
      acc[0] += v.x, acc[1] += v.y, acc[2] += v.z, acc[3] += v.w;
    } else {
      acc[0] += __ldcs(p + j * slab);
    }
  }
  T* o = (T*)out.p + z * out.z + m * out.ld + n;
#pragma unroll
  for (int k = 0; k < V; ++k) o[k] = FromFloat<T>::get(acc[k]);
}

template <class T>
int sum_parts(const float* ws, const f8::Out& out, const GemmGeom& g, int kb_per_seg, cudaStream_t st) {
  const long long slab = (long long)g.M * g.N;
  if (g.N % 4 == 0)
    fp8_sum_parts_kernel<T, 4><<<dim3((unsigned)up(slab, 512), g.nz), 128, 0, st>>>(ws, out, g, kb_per_seg);
  else
    fp8_sum_parts_kernel<T, 1><<<dim3((unsigned)up(slab, 128), g.nz), 128, 0, st>>>(ws, out, g, kb_per_seg);
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

template <bool A_MN, bool B_MN, bool kPair, int kOut, bool kByRow>
int launch_one(const GemmGeom& g, const tc::TcOperand& a, const tc::TcOperand& b, const f8::Scales& sa, const f8::Scales& sb,
               const f8::Out& out, int* status, int sms, cudaStream_t stream) {
  using TL = f8::Tile<kPair>;
  CUtensorMap mapA, mapB;
  if (int rc = tc::encode_operand_map8(&mapA, a, f8::kBM)) return rc;
  if (int rc = tc::encode_operand_map8(&mapB, b, TL::kBRows)) return rc;
  CUtensorMap mapOut = mapA;  // (not used where rows are not aligned)
  if (out.tma)
    if (int rc = tc::encode_output_map(&mapOut, out.p, out.dtype, g.N, g.M, g.nz, out.ld, out.z)) return rc;
  auto kern = f8::gemm_fp8_kernel<A_MN, B_MN, kPair, kOut, kByRow>;
  static bool attr_set[64];  // per instantiation and device
  int dev = 0;
  CLT_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    CLT_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, f8::kSmemBytes));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const long long total = up(g.M, TL::kM) * up(g.N, f8::kBN) * g.nz, workers = sms / TL::kCtas;
  CLT_CHECK_ARG(total < (1ll << 31), "fp8_matmul: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((total < workers ? total : workers) * TL::kCtas));
  cfg.blockDim = dim3(f8::kThreads);
  cfg.dynamicSmemBytes = f8::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = TL::kCtas, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
  cfg.attrs = &at;
  cfg.numAttrs = kPair ? 1 : 0;
  CLT_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, mapA, mapB, mapOut, g, sa, sb, out, status));
  return 0;
}

template <bool A_MN, bool B_MN, bool kPair, bool kByRow>
int launch(const GemmGeom& g, const tc::TcOperand& a, const tc::TcOperand& b, const f8::Scales& sa, const f8::Scales& sb,
           const f8::Out& out, int* status, int sms, cudaStream_t stream) {
  if (out.dtype == 0) return launch_one<A_MN, B_MN, kPair, 0, kByRow>(g, a, b, sa, sb, out, status, sms, stream);
  if (out.dtype == 1) return launch_one<A_MN, B_MN, kPair, 1, kByRow>(g, a, b, sa, sb, out, status, sms, stream);
  return launch_one<A_MN, B_MN, kPair, 2, kByRow>(g, a, b, sa, sb, out, status, sms, stream);
}

int dispatch(const GemmGeom& g, const tc::TcOperand& a, const tc::TcOperand& b, const f8::Scales& sa, const f8::Scales& sb,
             const f8::Out& out, int* status, int sms, cudaStream_t stream) {
  const bool pair = use_pair(g, sms);
#define CLT_FP8_CASE(AM, BM, ROW)                                                                              \
  if ((a.mn_major != 0) == AM && (b.mn_major != 0) == BM && (sa.shift == 0) == ROW)                            \
    return pair ? launch<AM, BM, true, ROW>(g, a, b, sa, sb, out, status, sms, stream)                         \
                : launch<AM, BM, false, ROW>(g, a, b, sa, sb, out, status, sms, stream);
  CLT_FP8_CASE(false, false, false)
  CLT_FP8_CASE(false, true, false)
  CLT_FP8_CASE(true, false, false)
  CLT_FP8_CASE(true, true, false)
  CLT_FP8_CASE(false, false, true)
  CLT_FP8_CASE(false, true, true)
#undef CLT_FP8_CASE
  CLT_CHECK_ARG(false, "fp8_matmul: operand layout");
}

// The 8-bit copy [Z, R, C] of a pass's operand in one buffer: values, rows of a multiple of 32 (a memory sector), then scales of 128 x 128
// blocks.
struct Copy {
  uint8_t* q;
  float* s;
  int64_t ld, z, sr, sz;  // distances of rows and matrices of the values, of rows and matrices of the scales
  long long bytes;
  Copy(void* buf, long long Z, long long R, long long C) {
    ld = up(C, 32) * 32, z = R * ld, sr = up(C, 128), sz = up(R, 128) * sr;
    q = (uint8_t*)buf;
    s = (float*)(q + Z * z);
    bytes = Z * (z + 4 * sz);
  }
};

bool geom(GemmGeom& g, int mode, int M, int N, int K, int L) {
  if (mode < 0 || mode > 3 || M <= 0 || N <= 0 || K <= 0 || L <= 0 || L > (mode == kBatched ? 65535 : 361)) return false;  // slabs: a grid's y
  g = GemmGeom{mode, M, N, K, L, mode == kDecDW ? L * (L + 1) / 2 : L};
  return true;
}

}  // namespace

extern "C" {

int clt_fp8_matmul_parts(int mode, int M, int N, int K, int L, int num_sms) {
  GemmGeom g;
  if (!geom(g, mode, M, N, K, L)) return 0;
  return plan_parts(g, num_sms > 0 ? num_sms : device_sm_count());
}

int clt_fp8_matmul(int mode, const void* a, int64_t a_ld, int64_t a_z, int a_trans, const float* sa, int64_t sa_z,
                   int64_t sa_mn, int64_t sa_k, int a_rows, const void* b, int64_t b_ld, int64_t b_z, int b_trans,
                   const float* sb, int64_t sb_z, int64_t sb_mn, int64_t sb_k, const float* bias, int64_t bias_z, void* out,
                   int out_dtype, int64_t out_ld, int64_t out_z, float* ws, int64_t ws_floats, int M, int N, int K, int L,
                   int* status, clt_stream_t stream) {
  GemmGeom g;
  CLT_CHECK_ARG(geom(g, mode, M, N, K, L), "fp8_matmul: bad mode %d or dims M=%d N=%d K=%d L=%d", mode, M, N, K, L);
  CLT_CHECK_ARG(a && b && sa && sb && out && status, "fp8_matmul: null pointer");
  CLT_CHECK_ARG(out_dtype >= 0 && out_dtype <= 2, "fp8_matmul: output type %d", out_dtype);
  CLT_CHECK_ARG(a_rows == 128 || (a_rows == 1 && !a_trans),
                "fp8_matmul: blocks of %d rows (1 or 128; a transposed operand needs 128)", a_rows);
  CLT_CHECK_ARG(out_ld >= N, "fp8_matmul: rows of %d values at a distance of %lld", N, (long long)out_ld);
  const int esize = out_dtype == 0 ? 4 : 2, sms = device_sm_count();
  CLT_CHECK_ARG((uintptr_t)out % esize == 0, "fp8_matmul: misaligned output");
  // stacked matrices: [L] each, but the decoder's blocks, which are [pairs]
  const long long pairs = (long long)L * (L + 1) / 2;
  const long long na = L, nb = mode == kDecFwd || mode == kDecDFeat ? pairs : L;
  tc::TcOperand ta{a, a_trans ? 1 : 0, a_trans ? M : K, a_trans ? K : M, a_ld, na, a_z};
  tc::TcOperand tb{b, b_trans ? 0 : 1, b_trans ? K : N, b_trans ? N : K, b_ld, nb, b_z};
  const f8::Scales fa{sa, sa_z, sa_mn, sa_k, a_rows == 1 ? 0 : 7}, fb{sb, sb_z, sb_mn, sb_k, 7};
  f8::Out fo{out, out_dtype, out_ld, out_z, bias, bias_z, 0};
  fo.tma = (uintptr_t)out % 16 == 0 && out_ld * esize % 16 == 0 && (g.nz == 1 || (out_z > 0 && out_z * esize % 16 == 0));
  const long long slab = (long long)M * N;
  if (ws != nullptr) {
    CLT_CHECK_ARG((uintptr_t)ws % 16 == 0, "fp8_matmul: the workspace must be 16-byte aligned");
    GemmGeom gp = g;
    const int parts = plan_parts(gp, sms);
    if (parts > 0 && parts * slab <= ws_floats) {
      gp.nz = parts;
      const f8::Out po{ws, 0, N, slab, nullptr, 0, N % 4 == 0};
      if (int rc = dispatch(gp, ta, tb, fa, fb, po, status, sms, (cudaStream_t)stream)) return rc;
      const int kps = (int)up(K, f8::kBK);
      gp.nz = g.nz;
      if (out_dtype == 0) return sum_parts<float>(ws, fo, gp, kps, (cudaStream_t)stream);
      if (out_dtype == 1) return sum_parts<__half>(ws, fo, gp, kps, (cudaStream_t)stream);
      return sum_parts<__nv_bfloat16>(ws, fo, gp, kps, (cudaStream_t)stream);
    }
  }
  return dispatch(g, ta, tb, fa, fb, fo, status, sms, (cudaStream_t)stream);
}

// ---- whole passes: one entry for the copies and products of a projection or a crosslayer decode --------------------------------
int clt_fp8_copy_units(int Z, int R, int C) {
  if (Z <= 0 || R < 0 || C <= 0) return 0;
  const Copy c(nullptr, Z, R, C);
  const long long n = up(c.bytes, 256);
  return n < (1ll << 31) ? (int)n : 0;
}

int clt_fp8_pass_units(int crosslayer, int backward, int want_dx, int want_dw, int want_db, int B, int L, int K, int N) {
  if (B <= 0 || L <= 0 || K <= 0 || N <= 0 || L > 361) return 0;
  long long ws = 0, bytes = 0;
  const auto parts = [&](int mode, int m, int n, int k) {
    const long long need = 4ll * clt_fp8_matmul_parts(mode, m, n, k, L, 0) * m * n;
    ws = need > ws ? need : ws;
  };
  if (!backward) {
    parts(crosslayer ? kDecFwd : kBatched, B, N, K);
  } else {
    if (want_dx) parts(crosslayer ? kDecDFeat : kBatched, B, K, N);
    if (want_dw) parts(crosslayer ? kDecDW : kBatched, K, N, B);
    bytes = Copy(nullptr, L, B, N).bytes + (want_db ? 4ll * L * up(B, 128) * N + 256 : 0);
  }
  const long long n = up(bytes, 256) + up(ws, 256);
  return n < (1ll << 31) ? (int)n : 0;
}

int clt_fp8_pass_fwd(int crosslayer, const void* x, int dtype, int64_t x_ld, int64_t x_z, const void* W, const uint64_t* blocks,
                     int w_dtype, const float* bias, void* y, void* x_copy, void* w_copy, void* scratch, int64_t scratch_units, int B,
                     int L, int K, int N, int* status, clt_stream_t stream) {
  CLT_CHECK_ARG(x && (crosslayer ? (const void*)blocks : W) && y && x_copy && w_copy, "fp8_pass_fwd: null pointer");
  CLT_CHECK_ARG(B > 0 && L > 0 && L <= 361 && K > 0 && N > 0, "fp8_pass_fwd: bad dims B=%d L=%d K=%d N=%d", B, L, K, N);
  const Copy cx(x_copy, L, B, K), cw(w_copy, crosslayer ? L * (L + 1) / 2 : L, K, N);
  if (int rc = clt_fp8_quantize(x, dtype, x_ld, x_z, cx.q, cx.ld, cx.s, nullptr, L, B, K, 128, stream)) return rc;
  const int rc = crosslayer ? clt_fp8_quantize_blocks(blocks, L, w_dtype, cw.q, cw.ld, cw.s, K, N, stream)
                            : clt_fp8_quantize(W, w_dtype, N, (int64_t)K * N, cw.q, cw.ld, cw.s, nullptr, L, K, N, 128, stream);
  if (rc) return rc;
  return clt_fp8_matmul(crosslayer ? kDecFwd : kBatched, cx.q, cx.ld, cx.z, 0, cx.s, cx.sz, cx.sr, 1, 128, cw.q, cw.ld, cw.z, 0, cw.s,
                        cw.sz, 1, cw.sr, bias, N, y, dtype, (int64_t)L * N, N, (float*)scratch, scratch_units * 64, B, N, K, L, status,
                        stream);
}

int clt_fp8_pass_bwd(int crosslayer, const void* g, int dtype, int64_t g_ld, int64_t g_z, const void* x_copy, const void* w_copy,
                     void* dx, void* dW, int w_dtype, float* db, void* scratch, int64_t scratch_units, int B, int L, int K, int N,
                     int* status, clt_stream_t stream) {
  CLT_CHECK_ARG(g && scratch && (!dx || w_copy) && (!dW || x_copy), "fp8_pass_bwd: null pointer");
  CLT_CHECK_ARG(B > 0 && L > 0 && L <= 361 && K > 0 && N > 0, "fp8_pass_bwd: bad dims B=%d L=%d K=%d N=%d", B, L, K, N);
  CLT_CHECK_ARG((uintptr_t)scratch % 16 == 0 &&
                    scratch_units >= clt_fp8_pass_units(crosslayer, 1, dx != nullptr, dW != nullptr, db != nullptr, B, L, K, N),
                "fp8_pass_bwd: scratch is misaligned or too small (%lld units)", (long long)scratch_units);
  const Copy cg(scratch, L, B, N);
  const int chunks = (int)up(B, 128);
  float* part = db ? (float*)((uint8_t*)scratch + up(cg.bytes, 256) * 256) : nullptr;
  const long long used = up(cg.bytes + (db ? 4ll * L * chunks * N + 256 : 0), 256);
  float* ws = (float*)((uint8_t*)scratch + used * 256);
  const int64_t ws_floats = (scratch_units - used) * 64;
  if (int rc = clt_fp8_quantize(g, dtype, g_ld, g_z, cg.q, cg.ld, cg.s, part, L, B, N, 128, stream)) return rc;
  if (db)
    if (int rc = clt_sum_chunks(part, db, L, chunks, N, stream)) return rc;
  if (dx) {
    const Copy cw(const_cast<void*>(w_copy), crosslayer ? L * (L + 1) / 2 : L, K, N);
    if (int rc = clt_fp8_matmul(crosslayer ? kDecDFeat : kBatched, cg.q, cg.ld, cg.z, 0, cg.s, cg.sz, cg.sr, 1, 128, cw.q, cw.ld, cw.z,
                                1, cw.s, cw.sz, cw.sr, 1, nullptr, 0, dx, dtype, (int64_t)L * K, K, ws, ws_floats, B, K, N, L, status,
                                stream))
      return rc;
  }
  if (dW) {
    const Copy cx(const_cast<void*>(x_copy), L, B, K);
    if (int rc = clt_fp8_matmul(crosslayer ? kDecDW : kBatched, cx.q, cx.ld, cx.z, 1, cx.s, cx.sz, 1, cx.sr, 128, cg.q, cg.ld, cg.z, 0,
                                cg.s, cg.sz, 1, cg.sr, nullptr, 0, dW, w_dtype, N, (int64_t)K * N, ws, ws_floats, K, N, B, L, status,
                                stream))
      return rc;
  }
  return 0;
}

}  // extern "C"
