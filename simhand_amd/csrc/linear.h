// What the linear operator's kernels share (linear.hip, linear256.hip).
#pragma once
#include "rows.h"

namespace sh {

template <typename T> __device__ __forceinline__ f32x4 mma16(const uint4& a, const uint4& b, f32x4 c) {
  if constexpr (sizeof(T) == 2) {
    return sh_mfma16(a, b, c);
  } else {  // 16 bytes = 4 fp32: MFMA e takes element e of both operands (the same k order on both sides)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
  }
}

struct LinearArgs {
  const void* a;        // [M][K]
  const void* b;        // [N][ldb]
  void* out;            // [M][N]
  void* pre;            // [M][N] or null
  const float* bias;    // [N] or null
  const void* residual; // [M][N] or null
  long long M;
  int N, K, ldb, act;
  unsigned n_tiles;
};

// tile column that row m of MFMA tile ni holds: lane group g of the tiles 2 j, 2 j + 1 ends with columns 32 j + 8 g .. + 7
__device__ __forceinline__ int lin_col(int ni, int m) { return (ni >> 1) * 32 + (m >> 2) * 8 + (ni & 1) * 4 + (m & 3); }

// A wave's finished sums, rows row0 + 16 mi, columns n0 + 32 j .. + 7 of a lane: z = acc + bias, pre <- z, out <- act(z) + residual.  The residual is read for the whole tile before
// the first value is used (chunk after chunk, each waited for: 300000 x 77 -> 256 fp32 with gelu 333 us, like this 293; 231 since its tiles are 64 wide).
template <typename T, int QM, int QN>
__device__ __forceinline__ void linear_store_tile(const LinearArgs& p, long long row0, int n0, const f32x4 (&acc)[QM][QN]) {
  constexpr int VE = Vec16<T>::N, H = 8 / VE;
  uint4 res[QM][QN / 2][H];
  if (p.residual != nullptr) {
#pragma unroll
    for (int mi = 0; mi < QM; ++mi) {
      const long long row = row0 + 16 * mi < p.M ? row0 + 16 * mi : p.M - 1;
#pragma unroll
      for (int j = 0; j < QN / 2; ++j)
#pragma unroll
        for (int h = 0; h < H; ++h) res[mi][j][h] = ld_tail<T>((const T*)p.residual + row * p.N, n0 + 32 * j + h * VE, p.N);
    }
  }
#pragma unroll
  for (int j = 0; j < QN / 2; ++j) {
    const int n = n0 + 32 * j, left = p.N - n;
    if (left <= 0) break;
    float b[8];
    if (p.bias != nullptr) ld_f32<8>(p.bias + n, left, b);
#pragma unroll
    for (int mi = 0; mi < QM; ++mi) {
      const long long row = row0 + 16 * mi;
      if (row >= p.M) break;
      const long long at = row * p.N + n;
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int l = left - h * VE;
        if (l <= 0) break;
        float o[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          const float z = acc[mi][2 * j + (h * VE + e) / 4][(h * VE + e) & 3];
          o[e] = p.bias != nullptr ? z + b[h * VE + e] : z;
        }
        if (p.pre != nullptr) st_chunk<T>((T*)p.pre + at + h * VE, l, pack16<T>(o));
        if (p.act != SH_ACT_NONE) {
#pragma unroll
          for (int e = 0; e < VE; ++e) o[e] = act_value(o[e], p.act);
        }
        if (p.residual != nullptr) {
          float r[VE];
          unpack16<T>(tail_of<T>(res[mi][j][h], n + h * VE, p.N), r);
#pragma unroll
          for (int e = 0; e < VE; ++e) o[e] += r[e];
        }
        st_chunk<T>((T*)p.out + at + h * VE, l, pack16<T>(o));
      }
    }
  }
}

struct WgradArgsL {
  const void* dz;         // [M][N]
  const void* x;          // [M][K] (null: codes)
  const uint8_t* codes;   // [M][K]
  const uint8_t* exps;    // [M][ceil(K / 32)]
  float* part;            // [splits][N][K]
  long long M, per_split; // per_split: a multiple of the k-step
  int N, K;
  unsigned n_tiles, k_tiles;
};

// 256 x 256 tiles, 16-bit operands (linear256.hip, linear_wgrad256.hip)
bool linear256_takes(const LinearArgs& p, int dtype);
int linear256_launch(const LinearArgs& p, hipStream_t s, const char* what);
// rows in registers, K <= 512 (linear_rows.hip)
bool linear_rows_fits(const LinearArgs& p, int dtype);
bool linear_rows_takes(const LinearArgs& p, int dtype);
size_t linear_rows_workspace_bytes(const LinearArgs& p);
int linear_rows_launch(const LinearArgs& p, bool b_padded, void* workspace, hipStream_t s, const char* what);
bool linear_wgrad256_takes(const void* dz, const void* x, const uint8_t* codes, const uint8_t* exps, int64_t rows, int in_dim, int out_dim, int dtype);
void linear_wgrad256_plan(int64_t rows, int in_dim, int out_dim, int* splits, int64_t* per);
int linear_wgrad256_launch(const WgradArgsL& p, int splits, hipStream_t s);

}  // namespace sh
