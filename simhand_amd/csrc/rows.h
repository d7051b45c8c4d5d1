// Row-vector helpers of the layer-norm / linear / 8-bit activation kernels: rows of any length at any element alignment, and the block-scaled e4m3 codes.
#pragma once
#include "common.h"

namespace sh {

// 16 bytes at an address that is only element-aligned (a row of odd length): gfx950 serves unaligned global accesses in hardware, the type tells
// the compiler not to assume more
typedef unsigned u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned u32x4_any1 __attribute__((ext_vector_type(4), aligned(1)));

__device__ __forceinline__ uint4 ld16_any(const void* p) {
  const u32x4_any v = *reinterpret_cast<const u32x4_any*>(p);
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void st16_any(void* p, const uint4& v) {
  const u32x4_any o = {v.x, v.y, v.z, v.w};
  *reinterpret_cast<u32x4_any*>(p) = o;
}

// 16-byte chunk <-> fp32 lanes
template <typename T> __device__ __forceinline__ void unpack16(const uint4& v, float (&o)[Vec16<T>::N]) {
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
  if constexpr (Vec16<T>::N == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = h16_lo(w[i]);
      o[2 * i + 1] = h16_hi(w[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __uint_as_float(w[i]);
  }
}
template <typename T> __device__ __forceinline__ uint4 pack16(const float (&o)[Vec16<T>::N]) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (Vec16<T>::N == 8) w[i] = pack_bf16x2(o[2 * i], o[2 * i + 1]);
    else w[i] = __float_as_uint(o[i]);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// the chunk at p of which `left` elements exist (left >= N: all); what is missing reads as zero and is not touched in memory
template <typename T> __device__ __forceinline__ uint4 ld_chunk(const T* p, int left) {
  constexpr int N = Vec16<T>::N;
  if (left >= N) return ld16_any(p);
  unsigned w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
  for (int e = 0; e < N - 1; ++e) {
    if (e < left) {
      if constexpr (N == 8) w[e >> 1] |= (unsigned)p[e] << ((e & 1) * 16);
      else w[e] = __float_as_uint(p[e]);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// v with its first `gone` elements zeroed
template <typename T> __device__ __forceinline__ uint4 drop_first(const uint4& v, int gone) {
  constexpr int N = Vec16<T>::N;
  unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (N == 8) {
      if (gone >= 2 * i + 2) w[i] = 0u;
      else if (gone == 2 * i + 1) w[i] &= 0xffff0000u;
    } else {
      if (gone > i) w[i] = 0u;
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// v's elements moved down by `gone` places, zeros behind them (gone <= 0: v, all of them or more: zeros)
template <typename T> __device__ __forceinline__ uint4 move_down(const uint4& v, int gone) {
  constexpr int N = Vec16<T>::N, D = N / 4;  // elements per dword
  unsigned w[4] = {v.x, v.y, v.z, v.w};
  if (gone >= N) return make_uint4(0u, 0u, 0u, 0u);
  if (gone > 0) {
    if (gone & (2 * D)) { w[0] = w[2]; w[1] = w[3]; w[2] = 0u; w[3] = 0u; }
    if (gone & D) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0u; }
    if (D == 2 && (gone & 1)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = w[i] >> 16 | (i < 3 ? w[i + 1] << 16 : 0u);
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// Elements at .. of a row of len, in two steps: the load (without a branch if the row holds a whole chunk: a ragged last one is read as the row's last N elements), and
// where the values are used tail_of()
template <typename T> __device__ __forceinline__ uint4 ld_tail(const T* row, int at, int len) {
  constexpr int N = Vec16<T>::N;
  if (len < N) return at < len ? ld_chunk<T>(row + at, len - at) : make_uint4(0u, 0u, 0u, 0u);
  return ld16_any(row + (at + N <= len ? at : len - N));
}
template <typename T> __device__ __forceinline__ uint4 tail_of(const uint4& v, int at, int len) {
  return len < Vec16<T>::N ? v : move_down<T>(v, at + Vec16<T>::N - len);
}
// One chunk of a reduction row (the product's K): `k` its first element, `len` the row's length.  The ragged last chunk of a row is read as the row's last N elements with
// those that the chunk before it holds zeroed -- both operands of a product are read like this, so element e of either is the same k, and no element is
// loaded by itself.  Rows shorter than a chunk go element by element.
// In two steps, so that a loop can have the next step's loads in flight: kchunk_at is where to read (no branch), kchunk_gone how much of it to drop.
template <typename T> __device__ __forceinline__ int kchunk_at(int k, int len) { return k + Vec16<T>::N <= len ? k : len - Vec16<T>::N; }
template <typename T> __device__ __forceinline__ int kchunk_gone(int k, int len) { return k + Vec16<T>::N <= len ? 0 : k - (len - Vec16<T>::N); }
template <typename T> __device__ __forceinline__ uint4 ld_kchunk(const T* row, int k, int len) {
  constexpr int N = Vec16<T>::N;
  if (k + N <= len) return ld16_any(row + k);
  if (k >= len) return make_uint4(0u, 0u, 0u, 0u);
  if (len < N) return ld_chunk<T>(row, len);
  return drop_first<T>(ld16_any(row + len - N), k - (len - N));
}
template <typename T> __device__ __forceinline__ void st_chunk(T* p, int left, const uint4& v) {
  constexpr int N = Vec16<T>::N;
  if (left >= N) {
    st16_any(p, v);
    return;
  }
  const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int e = 0; e < N - 1; ++e) {
    if (e < left) {
      if constexpr (N == 8) p[e] = (T)(w[e >> 1] >> ((e & 1) * 16));
      else p[e] = __uint_as_float(w[e]);
    }
  }
}
// fp32 vectors beside a row (gamma, beta, bias): N floats at p, `left` of them existing; missing ones are zero
template <int N> __device__ __forceinline__ void ld_f32(const float* p, int left, float (&o)[N]) {
  typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
  if (left >= N) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const f32x4_any v = *reinterpret_cast<const f32x4_any*>(p + i);
      o[i] = v.x; o[i + 1] = v.y; o[i + 2] = v.z; o[i + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = i < left ? p[i] : 0.f;
  }
}

// ---- 8-bit activations: value = e4m3(code) * 2^(exp - 127), one exp byte (1 .. 247) for 32 consecutive columns of a row ------------------
constexpr int kAct8Block = 32;
__device__ __forceinline__ float act8_scale(unsigned exp) { return __uint_as_float(exp << 23); }
// four codes of one word, by gfx950's scaled conversion (exact: the scale is a power of two)
__device__ __forceinline__ void act8_decode4(unsigned w, float scale, float* o) {
  const auto lo = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, false);
  const auto hi = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, true);
  o[0] = lo[0]; o[1] = lo[1]; o[2] = hi[0]; o[3] = hi[1];
}
// eight codes (two words) -> a 16-byte chunk of the build's 16-bit type, by gfx950's scaled conversion: the scale's exponent is added to the code's, one rounding to nearest even (none
// for bf16).  A quarter of the instructions of decode + pack.
__device__ __forceinline__ uint4 act8_decode8_h16(unsigned lo, unsigned hi, float scale) {
#ifdef SH_H16_FP16
  return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, false)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, scale, true)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, false)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, scale, true)));
#else
  return make_uint4(__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                    __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true)));
#endif
}
// N (4, 8, 16) codes at p, `left` of them existing; missing ones decode to zero
template <int N> __device__ __forceinline__ void act8_ld_codes(const uint8_t* p, int left, unsigned (&w)[N / 4]) {
  if (left >= N) {
    if constexpr (N == 16) {
      const u32x4_any1 v = *reinterpret_cast<const u32x4_any1*>(p);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else if constexpr (N == 8) {
      const u32x2_any v = *reinterpret_cast<const u32x2_any*>(p);
      w[0] = v.x; w[1] = v.y;
    } else {
      typedef unsigned u32_any __attribute__((aligned(1)));
      w[0] = *reinterpret_cast<const u32_any*>(p);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < N / 4; ++i) w[i] = 0u;
#pragma unroll
  for (int e = 0; e < N - 1; ++e)
    if (e < left) w[e >> 2] |= (unsigned)p[e] << ((e & 3) * 8);
}

// xcd-aware order: the hardware puts block b on XCD b % 8; every XCD gets a contiguous range of logical tiles
__device__ __forceinline__ unsigned xcd_order(unsigned bid, unsigned nblk) {
  const unsigned q = nblk >> 3, r = nblk & 7, xcd = bid & 7, j = bid >> 3;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + j;
}

// ---- activations of the linear operator (enum sh_act) and their derivatives, fp32.  NaN stays NaN (also through ReLU). ------------------------
// exp(-z^2 / 2) and the normal distribution function Phi(z) = erfc(-z / sqrt 2) / 2.  erfc(x) = t P(t) exp(-x^2), t = 1 / (1 + x / 2), x >= 0, with P the degree-8
// Chebyshev fit of exp(x^2) erfc(x) / t over t in [1/16, 1] (x <= 30; exp(-x^2) is zero in fp32 long before), in 17 instructions.  Off by at most (8 + z^2) 2^-24 of Phi below zero (4e-7
// near zero, 8e-7 at -3, 7e-6 at -12: z^2 is rounded before exp2, which the product carries over) and by 4e-7 above; exp2's and the reciprocal's last bit come on top.  The library's erff costs
// about three times that, and an epilogue of 256 x 256 of them took as long as the product it follows.  logistic, below, likewise: (3 + 1.2 |z|) 2^-24 of its value.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.35355339059327376f, 1.f));
  float p = -0.05634250491857529f;
  p = fmaf(p, t, 0.2723356783390045f);
  p = fmaf(p, t, -0.4642637073993683f);
  p = fmaf(p, t, 0.2548193037509918f);
  p = fmaf(p, t, -0.01282817404717207f);
  p = fmaf(p, t, 0.1978423148393631f);
  p = fmaf(p, t, 0.2440689206123352f);
  p = fmaf(p, t, 0.2822780907154083f);
  p = fmaf(p, t, 0.28209006786346436f);
  const float q = p * t * e * 0.5f;
  return z < 0.f ? q : 1.f - q;
}
__device__ __forceinline__ float logistic(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == SH_ACT_RELU) return z <= 0.f ? 0.f : z;
  if (act == SH_ACT_GELU) {
    float e;
    return z * normal_cdf(z, e);
  }
  if (act == SH_ACT_SILU) return z * logistic(z);
  return z;
}
// (ReLU: relu_grad below)
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == SH_ACT_GELU) {
    float e;
    const float c = normal_cdf(z, e);
    return fmaf(z * 0.39894228040143268f, e, c);
  }
  if (act == SH_ACT_SILU) {
    const float s = logistic(z);
    return s * fmaf(z, 1.f - s, 1.f);
  }
  return 1.f;
}
// dz = dy relu'(z).  A gate, not a product: what it closes is 0 also where dy is infinite or NaN (as behind the layer norm); a NaN z stays NaN.
__device__ __forceinline__ float relu_grad(float dy, float z) { return z > 0.f ? dy : z <= 0.f ? 0.f : z; }

// ---- column sums: part [nblk][n] -> out [n], folded in 64 bits in the order of the blocks (layernorm.hip) -----------------------------------
int fold_columns(const float* part, int nblk, int n, float* out, hipStream_t s);
}  // namespace sh
