// Block-scaled 8-bit copies of activations and weights: fp32 / fp16 / bf16 -> e4m3 values with a power-of-two scale for each
// block of 1 x 128 or 128 x 128, and back; and the two-bit checkpoint of the (Jump)ReLU.
//
// The scale of a block is the smallest power of two s (at least 2^-126) with amax / s <= 448, amax over the block's finite values;
// 1 where all are zero.  With a power of two the quotient x / s and the product q * s are exact, so that the only rounding is the
// one to e4m3 (half a step: 2^-4 of the value), whichever way a copy was made, and a copy of a copy is the copy.  e4m3 has no
// infinity: what is not finite becomes NaN, and does not count for the scale.
//
// Where rows start on 16 bytes the kernels are bound by memory: 12 x 4000 x 10000 bf16 to 8 bits 225 us (6.4 TB/s), by rows 245 (5.9),
// back 226 (6.4); a gradient with its column sums, 12 x 4000 x 24576, 573 (6.2); JumpReLU of that size 780 (6.4) and its backward 790
// (6.3), ReLU 765 (6.5) and 723 (6.9).  Other rows cost more instructions, which bound them: 6 x 4000 x 10001 bf16 to 8 bits 180 us,
// by rows 162, back 214, where 10000 columns take 117, 125 and 116; JumpReLU 278 and 249 (166 and 185), ReLU 206 and 201 (163 and 154).
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../../include/clt_b200.h"
#include "common.cuh"
#include "kernels.h"

using namespace clt;

namespace {

// ---- 8 consecutive values ----------------------------------------------------------------------
template <class T>
struct Vec8;
template <>
struct Vec8<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const float* p) {
    a = __ldcs(reinterpret_cast<const float4*>(p)), b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&o)[8]) const {
    o[0] = a.x, o[1] = a.y, o[2] = a.z, o[3] = a.w, o[4] = b.x, o[5] = b.y, o[6] = b.z, o[7] = b.w;
  }
  __device__ __forceinline__ void put(const float (&v)[8]) {
    a = make_float4(v[0], v[1], v[2], v[3]), b = make_float4(v[4], v[5], v[6], v[7]);
  }
  __device__ __forceinline__ void store(float* p) const { st_cs8(p, a, b); }
  // The largest magnitude so far, as bits: they are ordered as the magnitudes are, infinities and NaN behind all numbers.
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    return m;
  }
  static constexpr uint32_t kInf = 0x7f800000u;
  static __device__ __forceinline__ uint32_t join(uint32_t m) { return m; }
  static __device__ __forceinline__ float magnitude(uint32_t bits) { return __uint_as_float(bits); }
};
template <class T>
struct Vec8Half {
  uint4 a;
  __device__ __forceinline__ uint32_t top(uint32_t m) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    return m;
  }
  __device__ __forceinline__ void load(const T* p) { a = __ldcs(reinterpret_cast<const uint4*>(p)); }
  // from any address: the words that hold the values, two bytes more at either end where it is not a word's
  __device__ __forceinline__ void load_words(const T* p) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
    const int shift = ((uintptr_t)p & 2) * 8;
    const uint32_t v[5] = {__ldg(w), __ldg(w + 1), __ldg(w + 2), __ldg(w + 3), shift ? __ldg(w + 4) : 0u};
    a = make_uint4(__funnelshift_r(v[0], v[1], shift), __funnelshift_r(v[1], v[2], shift), __funnelshift_r(v[2], v[3], shift),
                   __funnelshift_r(v[3], v[4], shift));
  }
  __device__ __forceinline__ void store(T* p) const { __stcs(reinterpret_cast<uint4*>(p), a); }
};
template <>
struct Vec8<__nv_bfloat16> : Vec8Half<__nv_bfloat16> {
  __device__ __forceinline__ void get(float (&o)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) o[2 * i] = __uint_as_float(w[i] << 16), o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  __device__ __forceinline__ void put(const float (&v)[8]) {
    a = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
  }
  static constexpr uint32_t kInf = 0x7f80u;
  static __device__ __forceinline__ uint32_t join(uint32_t m) { return max(m & 0xffffu, m >> 16); }
  static __device__ __forceinline__ float magnitude(uint32_t bits) { return __uint_as_float(bits << 16); }
};
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
struct Vec8<__half> : Vec8Half<__half> {
  __device__ __forceinline__ void get(float (&o)[8]) const {
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      o[2 * i] = f.x, o[2 * i + 1] = f.y;
    }
  }
  __device__ __forceinline__ void put(const float (&v)[8]) {
    a = make_uint4(pack_f16x2(v[0], v[1]), pack_f16x2(v[2], v[3]), pack_f16x2(v[4], v[5]), pack_f16x2(v[6], v[7]));
  }
  static constexpr uint32_t kInf = 0x7c00u;
  static __device__ __forceinline__ uint32_t join(uint32_t m) { return max(m & 0xffffu, m >> 16); }
  static __device__ __forceinline__ float magnitude(uint32_t bits) { return __half2float(__ushort_as_half((unsigned short)bits)); }
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void from_f32(float& o, float v) { o = v; }
__device__ __forceinline__ void from_f32(__half& o, float v) { o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }

// `n` of 8 values (the rest 0); `vec`: a 16-byte aligned address and all 8 there
template <class T>
__device__ __forceinline__ Vec8<T> load8(const T* p, int n, bool vec) {
  Vec8<T> r;
  if (vec) {
    r.load(p);
  } else if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      r.load_words(p);
    } else {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
      r.put(v);
    }
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    r.put(v);
  }
  return r;
}
template <class T>
__device__ __forceinline__ void store8(T* p, int n, bool vec, const float (&v)[8]) {
  if (vec) {
    Vec8<T> r;
    r.put(v);
    r.store(p);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) from_f32(p[i], v[i]);
  }
}

// ---- scale and rounding ----------------------------------------------------------------------------
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a <= 3.402823466e38f ? a : 0.f;  // 0 for infinities and NaN
}
// amax = m 2^e with m in [1, 2), and 448 = 1.75 * 2^8: 2^(e-8), or 2^(e-7) where m > 1.75.  (A subnormal amax has e = -127
// here, its scale is the least one either way.)
__device__ __forceinline__ float block_scale(float amax) {
  if (amax == 0.f) return 1.f;
  const uint32_t u = __float_as_uint(amax);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  e = e < -126 ? -126 : e;
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
// 1 / 2^e; exact for every scale (2^-126 .. 2^120)
__device__ __forceinline__ float inverse_scale(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

__device__ __forceinline__ float not_inf(float v) { return fabsf(v) <= 3.402823466e38f ? v : __uint_as_float(0x7fffffffu); }

// `all`: some of the block's values are not finite (the conversion takes infinities for large numbers)
__device__ __forceinline__ uint2 to_e4m3x8(const float (&v)[8], float inv, bool all) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2((all ? not_inf(v[2 * i]) : v[2 * i]) * inv,
                                                (all ? not_inf(v[2 * i + 1]) : v[2 * i + 1]) * inv),
                                    __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

__device__ __forceinline__ uint32_t max8(uint32_t v) {  // over groups of 8 lanes
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ uint32_t max16(uint32_t v) {  // over groups of 16 lanes
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

struct Source {
  const void* x;
  long long ld, z;  // elements
  int R, C;
  int vec;  // rows start on 16 bytes
  __device__ __forceinline__ const void* matrix(int i, int e) const { return (const char*)x + i * z * e; }
};
// The decoder's blocks, tensors of their own: number t holds t + 1 matrices, one after another.
constexpr int kMaxBlocks = 361;  // as many layers as the contraction takes
template <int kMost>
struct BlockList {
  const void* block[kMost];
  long long ld, z;
  int R, C, vec;
  __device__ __forceinline__ const void* matrix(int i, int e) const {
    int t = 0;
    while (i > t) i -= ++t;
    return (const char*)block[t] + i * z * e;
  }
};

// One CTA per 128 x 128 block, 16 lanes x 8 values to a row, 8 rows to a thread: the block is read once, all of it at a time.
// Magnitudes are compared as integers, two 16-bit ones at a time; where a block turns out to hold infinities or NaN they are
// found again without those.
// kSums: sums[z, block of rows, c] = the block's column sums (of what came in), for bias gradients.  They are added up where the
// values are unpacked for rounding, so that 16-bit ones are unpacked once (a gradient of 12 x 4000 x 24576: 650 -> 573 us); fp32
// ones before the barrier, where they cost no registers that the rounding wants (975 -> 964).
template <class T, bool kSums, class S>
__global__ void __launch_bounds__(256) quantize_tile_kernel(const __grid_constant__ S s, uint8_t* __restrict__ q, int q_ld, float* __restrict__ scales,
                                                            float* __restrict__ sums, int row_blocks, int col_blocks) {
  using V = Vec8<T>;
  __shared__ uint32_t part[2][8];
  const int cb = blockIdx.x % col_blocks, rb = blockIdx.x / col_blocks, z = blockIdx.y;
  const int g = threadIdx.x >> 4, c = cb * 128 + (threadIdx.x & 15) * 8;
  const int n = s.C - c;
  const bool vec = s.vec && n >= 8;
  const T* x = (const T*)s.matrix(z, sizeof(T)) + (long long)(rb * 128 + g) * s.ld + c;
  const int rows = s.R - rb * 128 - g;
  V v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = load8<T>(x + (long long)(16 * i) * s.ld, 16 * i < rows ? n : 0, vec && 16 * i < rows);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = v[i].top(top);
  top = max16(V::join(top));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
  if ((threadIdx.x & 31) == 0) part[0][threadIdx.x >> 5] = top;
  constexpr bool kSumsFirst = kSums && sizeof(T) == 4;
  __shared__ float colsum[kSums ? 16 : 1][128];
  float cs[8] = {};
  const auto sums_out = [&] {
#pragma unroll
    for (int k = 0; k < 8; k += 4)
      *reinterpret_cast<float4*>(&colsum[g][(threadIdx.x & 15) * 8 + k]) = make_float4(cs[k], cs[k + 1], cs[k + 2], cs[k + 3]);
  };
  if constexpr (kSumsFirst) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float f[8];
      v[i].get(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) cs[k] += f[k];
    }
    sums_out();
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, part[0][i]);
  const bool all = top >= V::kInf;  // uniform over the CTA
  float amax = V::magnitude(top);
  if (all) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float f[8];
      v[i].get(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) amax = fmaxf(amax, finite_abs(f[k]));
    }
    uint32_t bits = max16(__float_as_uint(amax));
    bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, 16));
    if ((threadIdx.x & 31) == 0) part[1][threadIdx.x >> 5] = bits;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) bits = max(bits, part[1][i]);
    amax = __uint_as_float(bits);
  }
  const float scale = block_scale(amax), inv = inverse_scale(scale);
  if (threadIdx.x == 0) scales[((long long)z * row_blocks + rb) * col_blocks + cb] = scale;
  uint8_t* out = q + ((long long)z * s.R + rb * 128 + g) * q_ld + c;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (16 * i < rows) {
      float f[8];
      v[i].get(f);
      if constexpr (kSums && !kSumsFirst) {
#pragma unroll
        for (int k = 0; k < 8; ++k) cs[k] += f[k];
      }
      if (c < q_ld) *reinterpret_cast<uint2*>(out + (long long)(16 * i) * q_ld) = to_e4m3x8(f, inv, all);
    }
  }
  if constexpr (kSums) {
    if constexpr (!kSumsFirst) {
      sums_out();
      __syncthreads();
    }
    if (threadIdx.x < 128 && cb * 128 + threadIdx.x < s.C) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) t += colsum[i][threadIdx.x];
      sums[((long long)z * row_blocks + rb) * s.C + cb * 128 + threadIdx.x] = t;
    }
  }
}

// 1 x 128 blocks: 8 lanes to a block, each with 8 values of either half.  (16 lanes to a block, 4 blocks one after another in each:
// 290 us for 12 x 4000 x 10000 bf16, this 247; a block's largest and its scale are found for twice as many values at once, and few
// values a thread start more threads' loads.)
template <class T>
__global__ void __launch_bounds__(256) quantize_row_kernel(Source s, uint8_t* __restrict__ q, int q_ld, float* __restrict__ scales,
                                                           int col_blocks, unsigned blocks) {
  using V = Vec8<T>;
  const int lane = threadIdx.x & 7;
  const unsigned block = blockIdx.x * 32 + (threadIdx.x >> 3);
  const bool there = block < blocks;
  const unsigned row = block / col_blocks, z = row / s.R, r = row - z * s.R;
  const int c = (int)(block - row * col_blocks) * 128 + lane * 8, n = there ? s.C - c : 0;
  const T* x = (const T*)s.x + z * s.z + r * s.ld + c;
  V v[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) v[h] = load8<T>(x + 64 * h, n - 64 * h, s.vec && n >= 64 * h + 8);
  const uint32_t top = max8(V::join(v[1].top(v[0].top(0))));
  const bool all = top >= V::kInf;
  float amax = V::magnitude(top), f[2][8];
  v[0].get(f[0]), v[1].get(f[1]);
  if (__any_sync(0xffffffffu, all)) {
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) a = fmaxf(a, finite_abs(f[k >> 3][k & 7]));
    a = __uint_as_float(max8(__float_as_uint(a)));
    if (all) amax = a;
  }
  if (!there) return;
  const float scale = block_scale(amax), inv = inverse_scale(scale);
  if (lane == 0) scales[block] = scale;
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (c + 64 * h < q_ld) *reinterpret_cast<uint2*>(q + (long long)row * q_ld + c + 64 * h) = to_e4m3x8(f[h], inv, all);
}

struct ScaleMap {
  const float* p;
  long long z, r, c;
  int shift;
};

// value * scale is rounded once, to T.  The product has up to 28 bits.  With a power of two it is a number of fp32 (or overflows there
// as in T).  With other scales (a subnormal one counts among them) and 16-bit results it is rounded to odd first: an fp32 with its
// last bit set where anything was lost lies on the same side of every border of T as the product does.
template <class T>
__device__ __forceinline__ bool to_odd_first(float s) { return sizeof(T) == 2 && (__float_as_uint(s) & 0x7fffffu) != 0; }
// Values are 0 or 2^-9 to 448: with a scale of at least 2^-90 what is cut off is a number of fp32, which fmaf finds.  Smaller ones are
// raised before, and the product is lowered, to odd again.  (Infinite scales leave NaN there, and the product as it is.)
__device__ __forceinline__ float to_odd(float v, float s) {
  const bool small = fabsf(s) < 0x1p-90f;
  const float a = small ? s * 0x1p64f : s;
  float p = __fmul_rz(v, a);
  if (fabsf(fmaf(v, a, -p)) > 0.f) p = __uint_as_float(__float_as_uint(p) | 1u);
  if (small) {
    const float f = __fmul_rz(p, 0x1p-64f);
    p = f * 0x1p64f == p ? f : __uint_as_float(__float_as_uint(f) | 1u);
  }
  return p;
}
__device__ __forceinline__ float2 two_values(uint32_t w) {
  return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)w, __NV_E4M3)));
}
// 16 values to a row's next columns, `left` of which are there; `vec`: rows start on 16 bytes
template <class T>
__device__ __forceinline__ void store16(T* o, int left, int vec, const float (&f)[2][8]) {
  if constexpr (sizeof(T) == 2) {
    if (vec && left >= 16 && aligned32(o)) {
      // 32 bytes in one access: two of 16 at a lane distance of 32 touch every sector twice (262 -> 226 us)
      Vec8<T> a, b;
      a.put(f[0]), b.put(f[1]);
      asm volatile("st.global.cs.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(a.a.x), "r"(a.a.y), "r"(a.a.z), "r"(a.a.w),
                   "r"(b.a.x), "r"(b.a.y), "r"(b.a.z), "r"(b.a.w), "l"(o)
                   : "memory");
      return;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) store8<T>(o + 8 * h, left - 8 * h, vec && left >= 8 * h + 8, f[h]);
}
// Out of line, so that powers of two keep their registers and schedule (12 x 4000 x 10000 bf16: 228 us, 250 with this inline; other
// scales 284).
template <class T>
__device__ __noinline__ void store16_to_odd(T* o, int left, int vec, const uint4 w, float s) {
  const uint32_t v[4] = {w.x, w.y, w.z, w.w};
  float f[2][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 t = two_values((v[k >> 1] >> 16 * (k & 1)) & 0xffff);
    f[k >> 2][2 * k & 7] = to_odd(t.x, s), f[k >> 2][(2 * k & 7) + 1] = to_odd(t.y, s);
  }
  store16<T>(o, left, vec, f);
}
// 8 values by two scales, the second from value `first` on
template <class T>
__device__ __noinline__ void store8_to_odd(T* o, uint2 w, float s0, float s1, unsigned first) {
  float f[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 t = two_values(((k < 2 ? w.x : w.y) >> 16 * (k & 1)) & 0xffff);
    f[2 * k] = to_odd(t.x, 2 * k < first ? s0 : s1), f[2 * k + 1] = to_odd(t.y, 2 * k + 1 < first ? s0 : s1);
  }
  store8<T>(o, 8, true, f);
}

// 16 values of a row to a thread.
template <class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint8_t* __restrict__ q, long long q_ld, long long q_z, ScaleMap sc,
                                                         T* __restrict__ out, int R, int C, int groups, long long n, int q_vec,
                                                         int out_vec) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const long long row = i / groups;
  const int c = (int)(i - row * groups) * 16;
  const long long z = row / R, r = row - z * R;
  const uint8_t* p = q + z * q_z + r * q_ld + c;
  const int left = C - c;
  uint32_t w[4] = {0, 0, 0, 0};
  if (q_vec && left >= 16) {
    const uint4 t = __ldcs(reinterpret_cast<const uint4*>(p));
    w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (k < left) w[k >> 2] |= (uint32_t)p[k] << 8 * (k & 3);
  }
  const float s = __ldg(sc.p + z * sc.z + (r >> sc.shift) * sc.r + (c >> 7) * sc.c);
  T* o = out + row * C + c;
  if (to_odd_first<T>(s)) {
    store16_to_odd<T>(o, left, out_vec, make_uint4(w[0], w[1], w[2], w[3]), s);
    return;
  }
  float f[2][8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 t = two_values((w[k >> 1] >> 16 * (k & 1)) & 0xffff);
    f[k >> 2][2 * k & 7] = t.x * s, f[k >> 2][(2 * k & 7) + 1] = t.y * s;
  }
  store16<T>(o, left, out_vec, f);
}

// The same where the result's rows do not start on 16 bytes: 8 values to a thread, counted through all rows, so that every store but
// the last is whole.  words: the copy's rows and their distances are multiples of 4 bytes.
template <class T>
__global__ void __launch_bounds__(256) dequantize_flat_kernel(const uint8_t* __restrict__ q, long long q_ld, long long q_z, ScaleMap sc,
                                                              T* __restrict__ out, int R, unsigned C, long long n, int words) {
  const long long i = (blockIdx.x * 256ll + threadIdx.x) * 8;
  if (i >= n) return;
  long long row = i / C;
  unsigned c = (unsigned)(i - row * C);
  long long z = row / R, r = row - z * R;
  const uint8_t* p = q + z * q_z + r * q_ld + c;
  const float* s = sc.p + z * sc.z + (r >> sc.shift) * sc.r;
  float f[8];
  if (c + 8 <= C) {
    uint32_t w[2] = {0, 0};
    if (words) {
      const uint32_t* v = reinterpret_cast<const uint32_t*>((uintptr_t)p & ~(uintptr_t)3);
      const int shift = ((uintptr_t)p & 3) * 8;
      const uint32_t a = __ldg(v), b = __ldg(v + 1), d = shift ? __ldg(v + 2) : 0u;
      w[0] = __funnelshift_r(a, b, shift), w[1] = __funnelshift_r(b, d, shift);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k >> 2] |= (uint32_t)p[k] << 8 * (k & 3);
    }
    const float s0 = __ldg(s + (c >> 7) * sc.c), s1 = __ldg(s + ((c + 7) >> 7) * sc.c);
    const unsigned left = 128 - (c & 127);  // values of the first block
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 t = two_values((w[k >> 1] >> 16 * (k & 1)) & 0xffff);
      f[2 * k] = t.x * (2 * k < left ? s0 : s1), f[2 * k + 1] = t.y * (2 * k + 1 < left ? s0 : s1);
    }
    // (looked at behind the products: 12 x 4000 x 10001 bf16 439 us, before them 445; with other scales 598)
    if (to_odd_first<T>(__uint_as_float(__float_as_uint(s0) | __float_as_uint(s1))))
      return store8_to_odd<T>(out + i, make_uint2(w[0], w[1]), s0, s1, left);
  } else {  // into the next row
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      f[k] = 0.f;
      if (i + k < n) {
        const __half_raw h = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)*p, __NV_E4M3);
        const float v = __half2float(__half(h)), a = __ldg(s + (c >> 7) * sc.c);
        f[k] = to_odd_first<T>(a) ? to_odd(v, a) : v * a;
        ++p;
        if (++c == C && i + k + 1 < n) {
          c = 0;
          if (++r == R) r = 0, ++z;
          p = q + z * q_z + r * q_ld;
          s = sc.p + z * sc.z + (r >> sc.shift) * sc.r;
        }
      }
    }
  }
  store8<T>(out + i, (int)(n - i < 8 ? n - i : 8), n - i >= 8, f);
}

// Rows of bytes that start anywhere, to rows that start on 16 bytes: 16 of them to a thread, joined of five aligned words (bytes, at
// the matrix's ends).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint8_t* __restrict__ q, long long q_ld, long long q_z,
                                                         uint8_t* __restrict__ out, int pitch, int R, int C, unsigned groups, long long n) {
  const long long i = blockIdx.x * 256ll + threadIdx.x;
  if (i >= n) return;
  const long long row = i / groups;
  const int c = (int)(i - row * groups) * 16;
  const long long z = row / R;
  const uint8_t *begin = q + z * q_z, *end = begin + (R - 1) * q_ld + C, *p = begin + (row - z * R) * q_ld + c;
  const uint8_t* from = (const uint8_t*)((uintptr_t)p & ~(uintptr_t)3);
  uint32_t w[4] = {0, 0, 0, 0};
  if (from >= begin && from + 20 <= end) {
    uint32_t v[5];
#pragma unroll
    for (int k = 0; k < 5; ++k) v[k] = reinterpret_cast<const uint32_t*>(from)[k];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __funnelshift_r(v[k], v[k + 1], 8 * ((uintptr_t)p & 3));
  } else {
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (c + k < C) w[k >> 2] |= (uint32_t)p[k] << 8 * (k & 3);
  }
  *reinterpret_cast<uint4*>(out + row * pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct Bandwidth {
  const float* p;  // on the device, or NULL for
  float value;
  __device__ __forceinline__ float get() const { return p != nullptr ? __ldg(p) : value; }
};

// out[z, c] = sum over the chunks, in their order, of part[z, chunk, c]; times -(theta / bandwidth) where theta is given.
__global__ void __launch_bounds__(256) sum_chunks_kernel(const float* __restrict__ part, float* __restrict__ out, int chunks, int C,
                                                         const float* __restrict__ theta, Bandwidth bandwidth) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C) return;
  const float* p = part + (long long)blockIdx.y * chunks * C + c;
  float acc = 0.f;
#pragma unroll 8
  for (int i = 0; i < chunks; ++i) acc += __ldcs(p + (long long)i * C);
  if (theta != nullptr) acc *= -(theta[c] / bandwidth.get());
  out[(long long)blockIdx.y * C + c] = acc;
}

// ---- (Jump)ReLU with a two-bit checkpoint ---------------------------------------------------------------
// A thread has 8 columns and kRowsAhead rows of them in flight.  A word of the checkpoint is 16 bits for 8 values: the low byte has
// bit i where the gradient passes (x >= 0; ReLU: x > 0), the high byte where theta - bw/2 < x <= theta + bw/2, the window in which the
// threshold gets a gradient.  Both bounds are rounded down, once, which decides the comparisons with an fp32 x as the exact bounds
// would.
constexpr int kRowsAhead = 4;
// the row behind the CTA's last
__device__ __forceinline__ int row_end(int R, int rows) { return (int)min((long long)R, (blockIdx.y + 1ll) * rows); }
struct Window {
  float lo[8], hi[8], theta[8];
};
// 16-bit values are compared two at a time with the bounds in their own type, rounded down once more (820 -> 785 us, 16 rows to a
// thread).
template <class T>
struct Pair;
template <>
struct Pair<__half> {
  using type = __half2;
  static __device__ __forceinline__ type down(float a, float b) { return __halves2half2(__float2half_rd(a), __float2half_rd(b)); }
};
template <>
struct Pair<__nv_bfloat16> {
  using type = __nv_bfloat162;
  static __device__ __forceinline__ type down(float a, float b) { return __halves2bfloat162(__float2bfloat16_rd(a), __float2bfloat16_rd(b)); }
};
template <class T>
struct PackedWindow {
  using P = typename Pair<T>::type;
  P lo[4], hi[4], theta[4];
  __device__ __forceinline__ explicit PackedWindow(const Window& w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo[i] = Pair<T>::down(w.lo[2 * i], w.lo[2 * i + 1]), hi[i] = Pair<T>::down(w.hi[2 * i], w.hi[2 * i + 1]);
      theta[i] = Pair<T>::down(w.theta[2 * i], w.theta[2 * i + 1]);
    }
  }
  // what is not above its threshold becomes 0; the word of the checkpoint
  __device__ __forceinline__ uint32_t apply(uint4& v) const {
    uint32_t x[4] = {v.x, v.y, v.z, v.w}, negative = 0, inside = 0;
    const P zero = Pair<T>::down(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const P p = *reinterpret_cast<const P*>(&x[i]);
      const uint32_t two = 1u << 2 * i | 2u << (2 * i + 16);  // bits 2i and 2i + 1 of the byte, the second in the upper half
      negative |= __hlt2_mask(p, zero) & two;
      inside |= __hgt2_mask(p, lo[i]) & __hle2_mask(p, hi[i]) & two;
      x[i] &= ~__hle2_mask(p, theta[i]);
    }
    v = make_uint4(x[0], x[1], x[2], x[3]);
    return (~(negative | negative >> 16) & 0xffu) | ((inside | inside >> 16) & 0xffu) << 8;
  }
};
// x > theta and x > 0; nothing is above a NaN
__device__ __forceinline__ float threshold(float t) { return t != t ? __uint_as_float(0x7f800000u) : fmaxf(t, 0.f); }
__device__ __forceinline__ void load_window(Window& w, const float* theta, Bandwidth bandwidth, int c, int n) {
  const float bw = bandwidth.get();
  float t[8];
  if (n >= 8 && ((uintptr_t)(theta + c) & 15) == 0) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(theta + c)), b = __ldg(reinterpret_cast<const float4*>(theta + c) + 1);
    t[0] = a.x, t[1] = a.y, t[2] = a.z, t[3] = a.w, t[4] = b.x, t[5] = b.y, t[6] = b.z, t[7] = b.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = k < n ? __ldg(theta + c + k) : 0.f;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    w.theta[k] = threshold(t[k]);
    w.lo[k] = __fmaf_rd(-0.5f, bw, t[k]), w.hi[k] = __fmaf_rd(0.5f, bw, t[k]);
  }
}

// The sums of a CTA's 8 warps over their rows, by column, in the warps' order.
struct WarpSums {
  float of[8][256];
  __device__ __forceinline__ void out(float* part, int c0, int C) const {
    __syncthreads();
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += of[i][threadIdx.x];
    if (c0 + (int)threadIdx.x < C) part[(long long)blockIdx.y * C + c0 + threadIdx.x] = sum;
  }
};

template <class T, bool kJump>
__global__ void __launch_bounds__(256) jump_relu_fwd_kernel(const T* __restrict__ x, long long ld, const float* __restrict__ theta,
                                                            Bandwidth bandwidth, T* __restrict__ y, uint16_t* __restrict__ bits,
                                                            int R, int C, int rows_per_cta) {
  const int words = (C + 7) / 8, w = blockIdx.x * 256 + threadIdx.x;
  if (w >= words) return;
  const int c = w * 8, n = C - c;  // (fp32: the last 8 may be 4)
  const int r0 = blockIdx.y * rows_per_cta, r1 = row_end(R, rows_per_cta);
  Vec8<T> v[kRowsAhead];
  const auto load = [&](int r) {
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) v[i] = load8<T>(x + (r + i) * ld + c, r + i < r1 ? n : 0, n >= 8 && r + i < r1);
  };
  load(r0);
  const auto rows = [&](auto&& apply) {
    for (int r = r0;;) {
#pragma unroll
      for (int i = 0; i < kRowsAhead; ++i)
        if (r + i < r1) bits[(long long)(r + i) * words + w] = (uint16_t)apply(v[i], y + (long long)(r + i) * C + c);
      if ((r += kRowsAhead) >= r1) break;
      load(r);
    }
  };
  if constexpr (kJump && sizeof(T) == 2) {
    Window wide;  // (on its way with the first rows)
    load_window(wide, theta, bandwidth, c, n);
    const PackedWindow<T> win(wide);
    rows([&](Vec8<T>& u, T* to) {
      const uint32_t m = win.apply(u.a);
      u.store(to);
      return m;
    });
  } else {
    Window win;
    if constexpr (kJump) load_window(win, theta, bandwidth, c, n);
    rows([&](Vec8<T>& u, T* to) {
      float f[8];
      u.get(f);
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float t = f[k];
        if constexpr (kJump) {
          if (!(t < 0.f)) m |= 1u << k;
          if (t > win.lo[k] && t <= win.hi[k]) m |= 256u << k;
          f[k] = t <= win.theta[k] ? 0.f : t;  // (at least 0; NaN stays)
        } else {
          if (!(t <= 0.f)) m |= 1u << k;
          f[k] = t <= 0.f ? 0.f : t;
        }
      }
      store8<T>(to, n, n >= 8, f);
      return m;
    });
  }
}

template <class T, bool kJump>
__global__ void __launch_bounds__(256) jump_relu_bwd_kernel(const T* __restrict__ g, long long ld, const uint16_t* __restrict__ bits,
                                                            T* __restrict__ dx, float* __restrict__ part, int R, int C,
                                                            int rows_per_cta, int in_vec, int out_vec) {
  // with a threshold's gradient a warp has 256 columns and the CTA's warps take rows in turn: its sums are made of many rows
  // while a thread walks few of them
  const int words = (C + 7) / 8, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int w = kJump ? blockIdx.x * 32 + lane : blockIdx.x * 256 + threadIdx.x;
  if (!kJump && w >= words) return;
  const int c = w * 8, n = C - c;
  const int r1 = w < words ? row_end(R, rows_per_cta) : 0;
  const int r0 = blockIdx.y * rows_per_cta + (kJump ? warp * kRowsAhead : 0), step = (kJump ? 8 : 1) * kRowsAhead;
  const bool iv = in_vec && n >= 8, ov = out_vec && n >= 8;
  float acc[8] = {};
  for (int r = r0; r < r1; r += step) {
    Vec8<T> v[kRowsAhead];
    uint32_t m[kRowsAhead];
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) {
      v[i] = load8<T>(g + (r + i) * ld + c, r + i < r1 ? n : 0, iv && r + i < r1);
      m[i] = r + i < r1 ? bits[(long long)(r + i) * words + w] : 0u;
    }
#pragma unroll
    for (int i = 0; i < kRowsAhead; ++i) {
      if (r + i < r1) {
        float f[8];
        v[i].get(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (kJump && (m[i] & (256u << k))) acc[k] += f[k];
          if (!(m[i] & (1u << k))) f[k] = 0.f;
        }
        store8<T>(dx + (long long)(r + i) * C + c, n, ov, f);
      }
    }
  }
  if constexpr (kJump) {
    __shared__ WarpSums sums;
#pragma unroll
    for (int k = 0; k < 8; k += 4)
      *reinterpret_cast<float4*>(&sums.of[warp][lane * 8 + k]) = make_float4(acc[k], acc[k + 1], acc[k + 2], acc[k + 3]);
    sums.out(part, blockIdx.x * 256, C);
  }
}

// The same where rows do not start on 16 bytes: a lane's 8 columns are 32 apart, so that a warp's accesses are side by side, and the
// bits of 8 neighbours come from ballots.
template <class T, bool kJump>
__global__ void __launch_bounds__(256) jump_relu_fwd_strided_kernel(const T* __restrict__ x, long long ld,
                                                                    const float* __restrict__ theta, Bandwidth bandwidth,
                                                                    T* __restrict__ y, uint16_t* __restrict__ bits, int R, int C,
                                                                    int rows_per_cta) {
  const int lane = threadIdx.x & 31, c0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 256, words = (C + 7) / 8;
  if (c0 >= C) return;
  float lo[8], hi[8], th[8];
  if constexpr (kJump) {
    const float bw = bandwidth.get();
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int c = c0 + 32 * k + lane;
      const float t = c < C ? __ldg(theta + c) : 0.f;
      th[k] = threshold(t);
      lo[k] = __fmaf_rd(-0.5f, bw, t), hi[k] = __fmaf_rd(0.5f, bw, t);
    }
  }
  const int r0 = blockIdx.y * rows_per_cta, n = row_end(R, rows_per_cta) - r0, left = C - c0 - lane;  // columns from this lane's on
  const T* from = x + (long long)r0 * ld + c0 + lane;
  T* to = y + (long long)r0 * C + c0 + lane;
  uint16_t* word = bits + (long long)r0 * words + c0 / 8 + lane;
  const bool whole = c0 + 256 <= C, has_word = c0 / 8 + lane < words;
  for (int r = 0; r < n; r += 2) {
    float v[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool there = r + i < n;
      if (whole && there) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = to_f32(from[32 * k]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = there && 32 * k < left ? to_f32(from[32 * k]) : 0.f;
      }
      from += ld;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (r + i < n) {
        uint32_t mine = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float t = v[i][k];
          const uint32_t pass = __ballot_sync(0xffffffffu, kJump ? !(t < 0.f) : !(t <= 0.f));
          uint32_t in = 0;
          if constexpr (kJump) in = __ballot_sync(0xffffffffu, t > lo[k] && t <= hi[k]);
          if (lane >> 2 == k) mine = __byte_perm(pass >> 8 * (lane & 3), in >> 8 * (lane & 3), 0x0040);
          v[i][k] = t <= (kJump ? th[k] : 0.f) ? 0.f : t;
        }
        if (whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k) from_f32(to[32 * k], v[i][k]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (32 * k < left) from_f32(to[32 * k], v[i][k]);
        }
        if (has_word) *word = (uint16_t)mine;
      }
      to += C, word += words;
    }
  }
}

template <class T, bool kJump>
__global__ void __launch_bounds__(256) jump_relu_bwd_strided_kernel(const T* __restrict__ g, long long ld,
                                                                    const uint16_t* __restrict__ bits, T* __restrict__ dx,
                                                                    float* __restrict__ part, int R, int C, int rows_per_cta) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = (kJump ? blockIdx.x : blockIdx.x * 8 + warp) * 256, words = (C + 7) / 8;
  if (!kJump && c0 >= C) return;
  // (with a threshold's gradient the warps take rows in turn, as above)
  const int r0 = blockIdx.y * rows_per_cta + (kJump ? 2 * warp : 0), step = kJump ? 16 : 2, left = C - c0 - lane;
  const int n = row_end(R, rows_per_cta) - r0;
  const T* from = g + (long long)r0 * ld + c0 + lane;
  T* to = dx + (long long)r0 * C + c0 + lane;
  const uint16_t* word = bits + (long long)r0 * words + c0 / 8 + lane;
  const bool whole = c0 + 256 <= C, has_word = c0 / 8 + lane < words;
  float acc[8] = {};
  for (int r = 0; r < n; r += step) {
    float v[2][8];
    uint32_t mine[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool there = r + i < n;
      mine[i] = there && has_word ? *word : 0u;
      if (whole && there) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = to_f32(from[32 * k]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = there && 32 * k < left ? to_f32(from[32 * k]) : 0.f;
      }
      from += ld, word += words;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (r + i < n) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint32_t m = __shfl_sync(0xffffffffu, mine[i], 4 * k + (lane >> 3)) >> (lane & 7);
          if (kJump && (m & 256)) acc[k] += v[i][k];
          if (!(m & 1)) v[i][k] = 0.f;
        }
        if (whole) {
#pragma unroll
          for (int k = 0; k < 8; ++k) from_f32(to[32 * k], v[i][k]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (32 * k < left) from_f32(to[32 * k], v[i][k]);
        }
      }
      to += C;
    }
    if constexpr (kJump) from += (step - 2) * ld, word += (step - 2) * words, to += (long long)(step - 2) * C;
  }
  if constexpr (kJump) {
    __shared__ WarpSums sums;
#pragma unroll
    for (int k = 0; k < 8; ++k) sums.of[warp][32 * k + lane] = acc[k];
    sums.out(part, c0, C);
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
long long up(long long a, long long b) { return (a + b - 1) / b; }
int elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

// Rows of a CTA of the (Jump)ReLU kernels that has one of `across` pieces of them: enough CTAs for the chip, within bounds.  Few
// rows, all of them in flight at once, are faster than a walk: 12 x 4000 x 24576 bf16 ReLU in 4 rows 765 us, in 128 848, and 6 x
// 4000 x 10000 fp32 JumpReLU 293 and 336.  Where a thread's thresholds cost more than that: 8 rows for 16-bit values (780; 4: 863),
// 64 for rows that are not aligned.  Where each CTA's sums go to memory and back, 32 to 128, which its 8 warps share.
int rows_per_cta(int R, long long across, int least, int most, int sms) {
  const long long rows = up(R, up(8ll * sms, across)), grid_y = up(R, 65535);
  const long long bounded = rows < least ? least : rows > most ? most : rows;
  return (int)(bounded < grid_y ? grid_y : bounded);
}
int rows_per_sum(int R, int C, int sms) { return rows_per_cta(R, up(C, 256), 32, 128, sms); }

template <class T>
int quantize(const Source& s, uint8_t* q, int q_ld, float* scales, float* sums, int Z, int block_rows, cudaStream_t st) {
  const int cb = (int)up(s.C, 128);
  if (block_rows == 1) {
    const long long blocks = (long long)Z * s.R * cb;
    CLT_CHECK_ARG(blocks < (1ll << 31), "fp8_quantize: too many blocks");
    quantize_row_kernel<T><<<(unsigned)up(blocks, 32), 256, 0, st>>>(s, q, q_ld, scales, cb, (unsigned)blocks);
  } else {
    const long long rb = up(s.R, 128);
    CLT_CHECK_ARG(rb * cb < (1ll << 31) && Z <= 65535, "fp8_quantize: too many blocks");
    const dim3 grid((unsigned)(rb * cb), Z);
    if (sums != nullptr)
      quantize_tile_kernel<T, true, Source><<<grid, 256, 0, st>>>(s, q, q_ld, scales, sums, (int)rb, cb);
    else
      quantize_tile_kernel<T, false, Source><<<grid, 256, 0, st>>>(s, q, q_ld, scales, sums, (int)rb, cb);
  }
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

template <class T, class S>
int quantize_list(const S& s, uint8_t* q, int q_ld, float* scales, int Z, cudaStream_t st) {
  const long long rb = up(s.R, 128), cb = up(s.C, 128);
  CLT_CHECK_ARG(rb * cb < (1ll << 31), "fp8_quantize_blocks: too many blocks");
  quantize_tile_kernel<T, false, S><<<dim3((unsigned)(rb * cb), Z), 256, 0, st>>>(s, q, q_ld, scales, nullptr, (int)rb, (int)cb);
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

template <int kMost>
int quantize_any_list(const uint64_t* blocks, int n, int in_dtype, uint8_t* q, int q_ld, float* scales, int R, int C, cudaStream_t st) {
  const int e = elem_size(in_dtype);
  BlockList<kMost> s{};
  s.ld = C, s.z = (long long)R * C, s.R = R, s.C = C;
  s.vec = (long long)C * e % 16 == 0;
  for (int t = 0; t < n; ++t) {
    s.block[t] = (const void*)(uintptr_t)blocks[t];
    CLT_CHECK_ARG(s.block[t] != nullptr && blocks[t] % e == 0, "fp8_quantize_blocks: block %d is null or misaligned", t);
    s.vec = s.vec && aligned16(s.block[t]);
  }
  const int Z = n * (n + 1) / 2;
  if (in_dtype == 0) return quantize_list<float>(s, q, q_ld, scales, Z, st);
  if (in_dtype == 1) return quantize_list<__half>(s, q, q_ld, scales, Z, st);
  return quantize_list<__nv_bfloat16>(s, q, q_ld, scales, Z, st);
}

template <class T>
int dequantize(const uint8_t* q, long long q_ld, long long q_z, const ScaleMap& sc, T* out, int Z, int R, int C, cudaStream_t st) {
  if (aligned16(out) && (long long)C * sizeof(T) % 16 != 0) {
    const long long n = (long long)Z * R * C, grid = up(n, 2048);
    CLT_CHECK_ARG(grid < (1ll << 31), "fp8_dequantize: too many values");
    dequantize_flat_kernel<T><<<(unsigned)grid, 256, 0, st>>>(q, q_ld, q_z, sc, out, R, (unsigned)C, n,
                                                              (uintptr_t)q % 4 == 0 && q_ld % 4 == 0 && q_z % 4 == 0);
    CLT_CHECK_CUDA(cudaGetLastError());
    return 0;
  }
  const int groups = (int)up(C, 16);
  const long long n = (long long)Z * R * groups, grid = up(n, 256);
  CLT_CHECK_ARG(grid < (1ll << 31), "fp8_dequantize: too many values");
  dequantize_kernel<T><<<(unsigned)grid, 256, 0, st>>>(q, q_ld, q_z, sc, out, R, C, groups, n,
                                                       aligned16(q) && q_ld % 16 == 0 && (Z == 1 || q_z % 16 == 0),
                                                       aligned16(out) && (long long)C * sizeof(T) % 16 == 0);
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

template <class T>
int jump_fwd(const T* x, long long ld, const float* theta, Bandwidth bw, T* y, uint16_t* bits, int R, int C, int sms,
             cudaStream_t st) {
  const bool strided = !aligned16(x) || ld * (long long)sizeof(T) % 16 || !aligned16(y) || C * (long long)sizeof(T) % 16;
  const long long across = up(up(C, 8), 256);
  const int rows = rows_per_cta(R, across, 4, theta == nullptr ? 4 : strided ? 64 : sizeof(T) == 2 ? 8 : 4, sms);
  const dim3 grid((unsigned)across, (unsigned)up(R, rows));
  if (strided) {
    if (theta != nullptr)
      jump_relu_fwd_strided_kernel<T, true><<<grid, 256, 0, st>>>(x, ld, theta, bw, y, bits, R, C, rows);
    else
      jump_relu_fwd_strided_kernel<T, false><<<grid, 256, 0, st>>>(x, ld, theta, bw, y, bits, R, C, rows);
  } else if (theta != nullptr)
    jump_relu_fwd_kernel<T, true><<<grid, 256, 0, st>>>(x, ld, theta, bw, y, bits, R, C, rows);
  else
    jump_relu_fwd_kernel<T, false><<<grid, 256, 0, st>>>(x, ld, theta, bw, y, bits, R, C, rows);
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

template <class T>
int jump_bwd(const T* g, long long ld, const uint16_t* bits, const float* theta, Bandwidth bw, T* dx, float* dtheta, float* ws,
             int R, int C, int sms, cudaStream_t st) {
  const long long across = theta != nullptr ? up(C, 256) : up(up(C, 8), 256);
  const int rows = theta != nullptr ? rows_per_sum(R, C, sms) : rows_per_cta(R, across, 4, 4, sms);
  const dim3 grid((unsigned)across, (unsigned)up(R, rows));
  const int iv = aligned16(g) && ld * (long long)sizeof(T) % 16 == 0, ov = aligned16(dx) && C * (long long)sizeof(T) % 16 == 0;
  const bool strided = !iv || !ov;
  if (theta != nullptr) {
    if (strided)
      jump_relu_bwd_strided_kernel<T, true><<<grid, 256, 0, st>>>(g, ld, bits, dx, ws, R, C, rows);
    else
      jump_relu_bwd_kernel<T, true><<<grid, 256, 0, st>>>(g, ld, bits, dx, ws, R, C, rows, iv, ov);
    sum_chunks_kernel<<<dim3((unsigned)up(C, 256), 1), 256, 0, st>>>(ws, dtheta, (int)grid.y, C, theta, bw);
  } else if (strided) {
    jump_relu_bwd_strided_kernel<T, false><<<grid, 256, 0, st>>>(g, ld, bits, dx, nullptr, R, C, rows);
  } else {
    jump_relu_bwd_kernel<T, false><<<grid, 256, 0, st>>>(g, ld, bits, dx, nullptr, R, C, rows, iv, ov);
  }
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

}  // namespace

extern "C" {

int clt_fp8_quantize(const void* x, int in_dtype, int64_t ld, int64_t z_stride, void* q, int64_t q_ld, float* scales,
                     float* column_sums, int Z, int R, int C, int block_rows, clt_stream_t stream) {
  CLT_CHECK_ARG(x && q && scales, "fp8_quantize: null pointer");
  CLT_CHECK_ARG(Z > 0 && R > 0 && C > 0, "fp8_quantize: bad dims Z=%d R=%d C=%d", Z, R, C);
  CLT_CHECK_ARG(in_dtype >= 0 && in_dtype <= 2, "fp8_quantize: input type %d", in_dtype);
  CLT_CHECK_ARG(block_rows == 1 || block_rows == 128, "fp8_quantize: blocks of %d rows (1 or 128)", block_rows);
  CLT_CHECK_ARG(column_sums == nullptr || block_rows == 128, "fp8_quantize: column sums come with blocks of 128 rows");
  CLT_CHECK_ARG(q_ld >= C && q_ld % 16 == 0 && q_ld < (1ll << 31) && aligned16(q),
                "fp8_quantize: rows of the copy must be 16-byte aligned (distance %lld)", (long long)q_ld);
  const int e = elem_size(in_dtype);
  CLT_CHECK_ARG((uintptr_t)x % e == 0, "fp8_quantize: misaligned input");
  const Source s{x, ld, z_stride, R, C, aligned16(x) && ld * e % 16 == 0 && (Z == 1 || z_stride * e % 16 == 0)};
  cudaStream_t st = (cudaStream_t)stream;
  if (in_dtype == 0) return quantize<float>(s, (uint8_t*)q, (int)q_ld, scales, column_sums, Z, block_rows, st);
  if (in_dtype == 1) return quantize<__half>(s, (uint8_t*)q, (int)q_ld, scales, column_sums, Z, block_rows, st);
  return quantize<__nv_bfloat16>(s, (uint8_t*)q, (int)q_ld, scales, column_sums, Z, block_rows, st);
}

int clt_fp8_quantize_blocks(const uint64_t* blocks, int n, int in_dtype, void* q, int64_t q_ld, float* scales, int R, int C,
                            clt_stream_t stream) {
  CLT_CHECK_ARG(blocks && q && scales, "fp8_quantize_blocks: null pointer");
  CLT_CHECK_ARG(n > 0 && n <= kMaxBlocks && R > 0 && C > 0, "fp8_quantize_blocks: bad dims n=%d (at most %d) R=%d C=%d", n, kMaxBlocks,
                R, C);
  CLT_CHECK_ARG(in_dtype >= 0 && in_dtype <= 2, "fp8_quantize_blocks: input type %d", in_dtype);
  CLT_CHECK_ARG(q_ld >= C && q_ld % 16 == 0 && q_ld < (1ll << 31) && aligned16(q),
                "fp8_quantize_blocks: rows of the copy must be 16-byte aligned (distance %lld)", (long long)q_ld);
  cudaStream_t st = (cudaStream_t)stream;
  return n <= 16 ? quantize_any_list<16>(blocks, n, in_dtype, (uint8_t*)q, (int)q_ld, scales, R, C, st)
                 : quantize_any_list<kMaxBlocks>(blocks, n, in_dtype, (uint8_t*)q, (int)q_ld, scales, R, C, st);
}

int clt_fp8_dequantize(const void* q, int64_t q_ld, int64_t q_z, const float* scales, int64_t s_z, int64_t s_r, int64_t s_c,
                       int block_rows, void* out, int out_dtype, int Z, int R, int C, clt_stream_t stream) {
  CLT_CHECK_ARG(q && scales && out, "fp8_dequantize: null pointer");
  CLT_CHECK_ARG(Z > 0 && R > 0 && C > 0, "fp8_dequantize: bad dims Z=%d R=%d C=%d", Z, R, C);
  CLT_CHECK_ARG(out_dtype >= 0 && out_dtype <= 2, "fp8_dequantize: output type %d", out_dtype);
  CLT_CHECK_ARG(block_rows == 1 || block_rows == 128, "fp8_dequantize: blocks of %d rows (1 or 128)", block_rows);
  CLT_CHECK_ARG((uintptr_t)out % elem_size(out_dtype) == 0, "fp8_dequantize: misaligned output");
  const ScaleMap sc{scales, s_z, s_r, s_c, block_rows == 1 ? 0 : 7};
  cudaStream_t st = (cudaStream_t)stream;
  if (out_dtype == 0) return dequantize<float>((const uint8_t*)q, q_ld, q_z, sc, (float*)out, Z, R, C, st);
  if (out_dtype == 1) return dequantize<__half>((const uint8_t*)q, q_ld, q_z, sc, (__half*)out, Z, R, C, st);
  return dequantize<__nv_bfloat16>((const uint8_t*)q, q_ld, q_z, sc, (__nv_bfloat16*)out, Z, R, C, st);
}

int clt_fp8_align(const void* q, int64_t q_ld, int64_t q_z, void* out, int64_t pitch, int Z, int R, int C, clt_stream_t stream) {
  CLT_CHECK_ARG(q && out, "fp8_align: null pointer");
  CLT_CHECK_ARG(Z > 0 && R > 0 && C > 0 && q_ld >= 0 && q_z >= 0, "fp8_align: bad dims Z=%d R=%d C=%d", Z, R, C);
  CLT_CHECK_ARG(pitch >= C && pitch % 16 == 0 && pitch < (1ll << 31) && aligned16(out),
                "fp8_align: rows of the result must be 16-byte aligned (distance %lld)", (long long)pitch);
  const long long groups = up(C, 16), n = (long long)Z * R * groups, grid = up(n, 256);
  CLT_CHECK_ARG(grid < (1ll << 31), "fp8_align: too many values");
  align_rows_kernel<<<(unsigned)grid, 256, 0, (cudaStream_t)stream>>>((const uint8_t*)q, q_ld, q_z, (uint8_t*)out, (int)pitch, R, C,
                                                                      (unsigned)groups, n);
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

int clt_sum_chunks(const float* part, float* out, int Z, int chunks, int C, clt_stream_t stream) {
  CLT_CHECK_ARG(part && out, "sum_chunks: null pointer");
  CLT_CHECK_ARG(Z > 0 && Z <= 65535 && chunks >= 0 && C > 0, "sum_chunks: bad dims Z=%d chunks=%d C=%d", Z, chunks, C);
  sum_chunks_kernel<<<dim3((unsigned)up(C, 256), Z), 256, 0, (cudaStream_t)stream>>>(part, out, chunks, C, nullptr,
                                                                                          Bandwidth{nullptr, 1.f});
  CLT_CHECK_CUDA(cudaGetLastError());
  return 0;
}

int clt_jump_relu_chunks(int R, int C) { return R > 0 && C > 0 ? (int)up(R, rows_per_sum(R, C, device_sm_count())) : 0; }

int clt_jump_relu_fwd(const void* x, int64_t ld, const float* theta, const float* bandwidth, float bandwidth_value, void* y,
                      void* bits, int dtype, int R, int C, clt_stream_t stream) {
  CLT_CHECK_ARG(x && y && bits, "jump_relu_fwd: null pointer");
  CLT_CHECK_ARG(theta == nullptr || bandwidth != nullptr || bandwidth_value > 0.f, "jump_relu_fwd: bandwidth must be positive");
  CLT_CHECK_ARG(R > 0 && C > 0 && C <= (1 << 30) && ld >= 0, "jump_relu_fwd: bad dims R=%d C=%d", R, C);
  CLT_CHECK_ARG(dtype >= 0 && dtype <= 2 && (uintptr_t)x % elem_size(dtype) == 0 && (uintptr_t)y % elem_size(dtype) == 0,
                "jump_relu_fwd: type %d or misaligned pointer", dtype);
  const int sms = device_sm_count();
  cudaStream_t st = (cudaStream_t)stream;
  uint16_t* b = (uint16_t*)bits;
  const Bandwidth bw{bandwidth, bandwidth_value};
  if (dtype == 0) return jump_fwd<float>((const float*)x, ld, theta, bw, (float*)y, b, R, C, sms, st);
  if (dtype == 1) return jump_fwd<__half>((const __half*)x, ld, theta, bw, (__half*)y, b, R, C, sms, st);
  return jump_fwd<__nv_bfloat16>((const __nv_bfloat16*)x, ld, theta, bw, (__nv_bfloat16*)y, b, R, C, sms, st);
}

int clt_jump_relu_bwd(const void* g, int64_t ld, const void* bits, const float* theta, const float* bandwidth,
                      float bandwidth_value, void* dx, float* dtheta, float* ws, int64_t ws_floats, int dtype, int R, int C,
                      clt_stream_t stream) {
  CLT_CHECK_ARG(g && bits && dx && (theta == nullptr || (dtheta && ws)), "jump_relu_bwd: null pointer");
  CLT_CHECK_ARG(theta == nullptr || bandwidth != nullptr || bandwidth_value > 0.f, "jump_relu_bwd: bandwidth must be positive");
  CLT_CHECK_ARG(R > 0 && C > 0 && C <= (1 << 30) && ld >= 0, "jump_relu_bwd: bad dims R=%d C=%d", R, C);
  CLT_CHECK_ARG(dtype >= 0 && dtype <= 2 && (uintptr_t)g % elem_size(dtype) == 0 && (uintptr_t)dx % elem_size(dtype) == 0,
                "jump_relu_bwd: type %d or misaligned pointer", dtype);
  const int sms = device_sm_count();
  const long long chunks = up(R, rows_per_sum(R, C, sms));
  CLT_CHECK_ARG(theta == nullptr || chunks * C <= ws_floats, "jump_relu_bwd: %lld floats of scratch, %lld needed",
                (long long)ws_floats, chunks * C);
  cudaStream_t st = (cudaStream_t)stream;
  const uint16_t* b = (const uint16_t*)bits;
  const Bandwidth bw{bandwidth, bandwidth_value};
  if (dtype == 0) return jump_bwd<float>((const float*)g, ld, b, theta, bw, (float*)dx, dtheta, ws, R, C, sms, st);
  if (dtype == 1) return jump_bwd<__half>((const __half*)g, ld, b, theta, bw, (__half*)dx, dtheta, ws, R, C, sms, st);
  return jump_bwd<__nv_bfloat16>((const __nv_bfloat16*)g, ld, b, theta, bw, (__nv_bfloat16*)dx, dtheta, ws, R, C, sms, st);
}

}  // extern "C"
