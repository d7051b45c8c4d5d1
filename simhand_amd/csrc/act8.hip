// Activation checkpoints in 8 bits: what a backward pass needs of an activation, kept as e4m3 codes with one power of two for every 32 consecutive
// columns of a row (1.03 bytes a value).  The scale is local -- no amax history, no state, no pass over the tensor before the codes are made -- and a power of two,
// so x 2^-e is exact and the one rounding is the code's own: at most 2^-4 of the value, or 2^-10 2^e where that is more (codes below the grid's normal range).
//
//   A = largest finite |x| of the 32, e = floor(log2 A) - 8, one more where A > 1.75 * 2^floor(log2 A) (so that A 2^-e <= 448, e4m3's largest), e >= -126
//   code = e4m3(x 2^-e) to nearest even; exp byte = e + 127;  x^ = code 2^e, rounded to the tensor's type
//
// Infinities and NaN become NaN (e4m3 has no infinity): an overflow stays visible in the gradient instead of turning into a large number.  |x| beyond
// the last value whose code does not round past the type's range is held there (61440 for fp16, 1.875 * 2^127 else).
// Bound by HBM: 3.03 (fp32: 5.03) bytes per value each way.  401408 x 1024 bf16: pack 214 us, unpack 211 (5.9 TB/s).
#include "rows.h"

namespace sh {

#ifdef SH_H16_FP16
constexpr float kHold16 = 61440.f;
#else
constexpr float kHold16 = 3.1901471898837980e38f;  // 1.875 * 2^127
#endif
constexpr float kHold32 = 3.1901471898837980e38f;

// One thread = 16 consecutive columns of a row, two neighbouring lanes = one block of 32.  units = rows * upr, upr even = 16-column units per row.
template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void act8_pack_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ exps,
                                                        unsigned units, int upr, FastDiv by_upr, int cols) {
  constexpr int N = Vec16<T>::N, L = 16 / N;
  const float hold = N == 8 ? kHold16 : kHold32;
  const unsigned u = blockIdx.x * 256u + threadIdx.x;
  if (u >= units) return;  // units is even: both lanes of a block leave together
  // FLAT (cols a multiple of 32): unit u is simply values 16 u .. 16 u + 15
  const unsigned row = FLAT ? 0u : fdiv(u, by_upr);
  const int c = FLAT ? 0 : (int)(u - row * (unsigned)upr) * 16;
  const long long at = FLAT ? (long long)u * 16 : (long long)row * cols + c;
  const int left = FLAT ? 16 : cols - c;
  float v[16];
#pragma unroll
  for (int i = 0; i < L; ++i) {
    float t[N];
    unpack16<T>(left > i * N ? ld_chunk<T>(x + at + i * N, left - i * N) : make_uint4(0u, 0u, 0u, 0u), t);
#pragma unroll
    for (int e = 0; e < N; ++e) v[i * N + e] = t[e];
  }
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float f = fabsf(v[e]);
    a = fmaxf(a, f <= 3.4028234663852886e38f ? f : 0.f);  // finite ones only
  }
  a = fmaxf(a, __shfl_xor(a, 1));
  const unsigned ab = __float_as_uint(a);
  int e127 = (int)(ab >> 23) - 8 + ((ab & 0x7fffffu) > 0x600000u ? 1 : 0);  // e + 127; a subnormal A ends at the lower bound anyway
  if (e127 < 1) e127 = 1;
  const float inv = __uint_as_float((unsigned)(254 - e127) << 23);
  unsigned w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = v[4 * k + e];
      const float cl = fminf(fmaxf(f, -hold), hold) * inv;
      q[e] = fabsf(f) <= 3.4028234663852886e38f ? cl : __uint_as_float(0x7fc00000u);
    }
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], r, true);
    w[k] = r;
  }
  if (left >= 16) {
    const u32x4_any1 o = {w[0], w[1], w[2], w[3]};
    *reinterpret_cast<u32x4_any1*>(codes + at) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 15; ++e)
      if (e < left) codes[at + e] = (uint8_t)(w[e >> 2] >> ((e & 3) * 8));
  }
  if ((u & 1) == 0) exps[u >> 1] = (uint8_t)e127;
}

template <typename T, bool FLAT>
__global__ __launch_bounds__(256) void act8_unpack_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, T* __restrict__ x,
                                                          unsigned units, int upr, FastDiv by_upr, int cols) {
  constexpr int N = Vec16<T>::N, L = 16 / N;
  const unsigned u = blockIdx.x * 256u + threadIdx.x;
  if (u >= units) return;
  const unsigned row = FLAT ? 0u : fdiv(u, by_upr);
  const int c = FLAT ? 0 : (int)(u - row * (unsigned)upr) * 16;
  const long long at = FLAT ? (long long)u * 16 : (long long)row * cols + c;
  const int left = FLAT ? 16 : cols - c;
  if (left <= 0) return;
  unsigned w[4];
  act8_ld_codes<16>(codes + at, left, w);
  const float sc = act8_scale(exps[u >> 1]);
  float v[16];
#pragma unroll
  for (int k = 0; k < 4; ++k) act8_decode4(w[k], sc, v + 4 * k);
#pragma unroll
  for (int i = 0; i < L; ++i) {
    float t[N];
#pragma unroll
    for (int e = 0; e < N; ++e) t[e] = v[i * N + e];
    if (left > i * N) st_chunk<T>(x + at + i * N, left - i * N, pack16<T>(t));
  }
}

// rows are cut so that a launch's 32-bit unit index stays below 2^31 (64-bit offsets between the launches)
template <typename F> static int act8_launches(int64_t rows, int cols, F&& launch) {
  const int64_t upr = 2 * (((int64_t)cols + kAct8Block - 1) / kAct8Block);
  const int64_t most = ((1ll << 30) / upr) < 1 ? 1 : (1ll << 30) / upr;
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    launch(r, (unsigned)(n * upr), (int)upr);
  }
  return 0;
}

}  // namespace sh

using namespace sh;

extern "C" {

int simhand_act8_pack(const void* x, uint8_t* codes, uint8_t* exps, int64_t rows, int cols, int dtype, sh_stream_t stream) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "act8_pack: dtype %d", dtype);
  SH_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 24), "act8_pack: rows=%lld cols=%d", (long long)rows, cols);
  if (rows == 0) return 0;
  SH_REQUIRE(x && codes && exps, "act8_pack: NULL argument");
  hipStream_t s = (hipStream_t)stream;
  const int64_t eb = dtype == SH_F32 ? 4 : 2, nb = (cols + kAct8Block - 1) / kAct8Block;
  ProfScope ps(SH_PROF_MISC, s, 0, (double)rows * cols * (eb + 1.03125));
  act8_launches(rows, cols, [&](int64_t r, unsigned units, int upr) {
    const unsigned grid = (units + 255) / 256;
    const char* xr = (const char*)x + r * cols * eb;
    uint8_t* cr = codes + r * cols;
    uint8_t* er = exps + r * nb;
    const FastDiv fd = make_fastdiv((unsigned)upr);
#define SH_PACK(T, FLAT) act8_pack_kernel<T, FLAT><<<grid, 256, 0, s>>>((const T*)xr, cr, er, units, upr, fd, cols)
    if (cols % kAct8Block == 0) {
      if (dtype == SH_F32) SH_PACK(float, true);
      else SH_PACK(bf16_t, true);
    } else {
      if (dtype == SH_F32) SH_PACK(float, false);
      else SH_PACK(bf16_t, false);
    }
#undef SH_PACK
  });
  return check_launch("act8_pack");
}

int simhand_act8_unpack(const uint8_t* codes, const uint8_t* exps, void* x, int64_t rows, int cols, int dtype, sh_stream_t stream) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "act8_unpack: dtype %d", dtype);
  SH_REQUIRE(rows >= 0 && cols >= 1 && cols <= (1 << 24), "act8_unpack: rows=%lld cols=%d", (long long)rows, cols);
  if (rows == 0) return 0;
  SH_REQUIRE(codes && exps && x, "act8_unpack: NULL argument");
  hipStream_t s = (hipStream_t)stream;
  const int64_t eb = dtype == SH_F32 ? 4 : 2, nb = (cols + kAct8Block - 1) / kAct8Block;
  ProfScope ps(SH_PROF_MISC, s, 0, (double)rows * cols * (eb + 1.03125));
  act8_launches(rows, cols, [&](int64_t r, unsigned units, int upr) {
    const unsigned grid = (units + 255) / 256;
    char* xr = (char*)x + r * cols * eb;
    const uint8_t* cr = codes + r * cols;
    const uint8_t* er = exps + r * nb;
    const FastDiv fd = make_fastdiv((unsigned)upr);
#define SH_UNPACK(T, FLAT) act8_unpack_kernel<T, FLAT><<<grid, 256, 0, s>>>(cr, er, (T*)xr, units, upr, fd, cols)
    if (cols % kAct8Block == 0) {
      if (dtype == SH_F32) SH_UNPACK(float, true);
      else SH_UNPACK(bf16_t, true);
    } else {
      if (dtype == SH_F32) SH_UNPACK(float, false);
      else SH_UNPACK(bf16_t, false);
    }
#undef SH_UNPACK
  });
  return check_launch("act8_unpack");
}

}  // extern "C"
