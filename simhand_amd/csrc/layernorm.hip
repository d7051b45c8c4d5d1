// Layer norm over the last dimension, forward and backward (the BatchNorm of the projection head with statistics per ROW instead of per batch: the
// result of a row depends on no other row, so it is the same on any number of ranks and needs no collective).
//
//   m = sum x / C, v = sum (x - m)^2 / C, r = 1 / sqrt(v + eps), h = (x - m) r, y = h gamma + beta, optionally max(y, 0)
//   backward, u = dy (ReLU: where h gamma + beta > 0), g = u gamma:  dx = r (g - mean(g) - h mean(g h)), dgamma = sum_rows u h, dbeta = sum_rows u
//
// One pass over the data each way: a group of G lanes holds a whole row in registers (NV 16-byte vectors per lane), so the variance is summed about
// the finished mean (no E[x^2] - m^2 cancellation) and nothing is read twice.  Statistics and sums are fp32, the column sums over row blocks are
// folded in 64 bits in a fixed order (bit-reproducible).  Bound by HBM: 2 (3) elements of traffic per element forward (backward).
#include "rows.h"

namespace sh {

// sum over the G lanes that share a row (G = 16 or 64: inside a wave; G = 256: the whole block through LDS), the same bits in every lane
template <int G> __device__ __forceinline__ float group_sum(float v, float* red) {
  constexpr int W = G < 64 ? G : 64;
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if constexpr (G == 256) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the previous use of red is over
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// h gamma + beta in two roundings, in the forward and in the backward pass alike: the ReLU gate that the backward pass recomputes is the forward's
__device__ __forceinline__ float ln_affine(float x, float m, float r, float g, float b, float& h) {
#pragma clang fp contract(off)
  const float d = x - m;
  h = d * r;
  const float t = h * g;
  return t + b;
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             float eps, int relu, T* __restrict__ y, float* __restrict__ mean,
                                                             float* __restrict__ rstd, long long rows, int cols) {
  constexpr int VE = Vec16<T>::N, RB = 256 / G;
  __shared__ float red[4];
  const int t = threadIdx.x % G;
  const long long row = (long long)blockIdx.x * RB + threadIdx.x / G;
  const bool live = row < rows;
  const T* src = x + (live ? row : 0) * cols;
  float v[NV][VE];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * VE;
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (c < cols) q = ld_chunk<T>(src + c, cols - c);
    unpack16<T>(q, v[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VE; ++e) s += v[i][e];
  const float m = group_sum<G>(s, red) / (float)cols;
  float q2 = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * VE;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float d = v[i][e] - m;
      q2 += c + e < cols ? d * d : 0.f;
    }
  }
  const float r = 1.f / sqrtf(group_sum<G>(q2, red) / (float)cols + eps);
  if (!live) return;
  if (t == 0) {
    mean[row] = m;
    rstd[row] = r;
  }
  T* dst = y + row * cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * G + t) * VE;
    if (c >= cols) continue;
    float ga[VE], be[VE], o[VE];
    ld_f32<VE>(gamma + c, cols - c, ga);
    ld_f32<VE>(beta + c, cols - c, be);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      float h;
      o[e] = ln_affine(v[i][e], m, r, ga[e], be[e], h);
      if (relu) o[e] = o[e] <= 0.f ? 0.f : o[e];
    }
    st_chunk<T>(dst + c, cols - c, pack16<T>(o));
  }
}

// A8: x comes as its 8-bit checkpoint (codes + exponents).  part [gridDim.x][2][cols]: sums of u h and u over the block's rows.
template <typename T, int G, int NV, bool A8>
__global__ __launch_bounds__(256) void layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ exps, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, int relu, T* __restrict__ dx,
                                                             float* __restrict__ part, long long rows, int cols) {
  constexpr int VE = Vec16<T>::N, RB = 256 / G;
  __shared__ float red[4];
  __shared__ float fold[2][G == 256 ? 1 : G * NV * VE];
  const int t = threadIdx.x % G, sub = threadIdx.x / G;
  const int eb = (cols + kAct8Block - 1) / kAct8Block;
  float ag[NV][VE], ab[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VE; ++e) ag[i][e] = ab[i][e] = 0.f;
  const float inv = 1.f / (float)cols;
  for (long long row0 = (long long)blockIdx.x * RB; row0 < rows; row0 += (long long)gridDim.x * RB) {
    const long long row = row0 + sub;
    const bool live = row < rows;
    const long long rr = live ? row : 0;
    const float m = mean[rr], r = rstd[rr];
    float h[NV][VE], u[NV][VE];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VE;
      uint4 qd = make_uint4(0u, 0u, 0u, 0u);
      if (c < cols && live) {
        qd = ld_chunk<T>(dy + rr * cols + c, cols - c);
        if constexpr (A8) {
          unsigned w[VE / 4];
          act8_ld_codes<VE>(codes + rr * cols + c, cols - c, w);
          const float sc = act8_scale(exps[rr * eb + c / kAct8Block]);
#pragma unroll
          for (int k = 0; k < VE / 4; ++k) act8_decode4(w[k], sc, &h[i][4 * k]);
        } else {
          unpack16<T>(ld_chunk<T>(x + rr * cols + c, cols - c), h[i]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) h[i][e] = m;
      }
      unpack16<T>(qd, u[i]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VE;
      if (c >= cols || !live) continue;
      float ga[VE], be[VE];
      ld_f32<VE>(gamma + c, cols - c, ga);
      ld_f32<VE>(beta + c, cols - c, be);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (c + e >= cols) continue;
        const float z = ln_affine(h[i][e], m, r, ga[e], be[e], h[i][e]);
        if (relu && !(z > 0.f)) u[i][e] = 0.f;
        ag[i][e] += u[i][e] * h[i][e];
        ab[i][e] += u[i][e];
        u[i][e] *= ga[e];
        s1 += u[i][e];
        s2 += u[i][e] * h[i][e];
      }
    }
    s1 = group_sum<G>(s1, red) * inv;
    s2 = group_sum<G>(s2, red) * inv;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (i * G + t) * VE;
      if (c >= cols) continue;
      float o[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) o[e] = r * (u[i][e] - s1 - h[i][e] * s2);
      st_chunk<T>(dx + row * cols + c, cols - c, pack16<T>(o));
    }
  }
  // the block's column sums: its row groups one after the other (fixed order)
  float* out = part + (long long)blockIdx.x * 2 * cols;
  if constexpr (G == 256) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const int c = (i * G + t) * VE + e;
        if (c < cols) {
          out[c] = ag[i][e];
          out[cols + c] = ab[i][e];
        }
      }
  } else {
    for (int w = 0; w < RB; ++w) {
      if (sub == w) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < VE; ++e) {
            const int c = (i * G + t) * VE + e;
            fold[0][c] = (w == 0 ? 0.f : fold[0][c]) + ag[i][e];
            fold[1][c] = (w == 0 ? 0.f : fold[1][c]) + ab[i][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += 256) {
      out[c] = fold[0][c];
      out[cols + c] = fold[1][c];
    }
  }
}

// [nblk][n] -> [n]: 64 columns x 4 groups of partial rows per block, 64-bit sums
__global__ __launch_bounds__(256) void fold_columns_kernel(const float* __restrict__ part, int nblk, int n, float* __restrict__ out) {
  __shared__ double red[4][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
  double a = 0.0;
  if (c < n)
    for (int b = q; b < nblk; b += 4) a += (double)part[(long long)b * n + c];
  red[q][threadIdx.x & 63] = a;
  __syncthreads();
  if (q == 0 && c < n) out[c] = (float)((red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]));
}
int fold_columns(const float* part, int nblk, int n, float* out, hipStream_t s) {
  fold_columns_kernel<<<ceil_div(n, 64), 256, 0, s>>>(part, nblk, n, out);
  return check_launch("fold_columns");
}

// (G, NV) by the row's 16-byte vectors: the smallest group that holds the row
static int ln_nvec(int cols, int dtype) { return (cols + (dtype == SH_F32 ? 4 : 8) - 1) / (dtype == SH_F32 ? 4 : 8); }
constexpr int kLnMaxVec = 2048;
static int ln_rows_per_block(int nvec) { return nvec <= 16 ? 16 : nvec <= 256 ? 4 : 1; }
// backward blocks: enough to fill the chip twice, few enough that the partial sums stay small beside the rows
static int ln_bwd_blocks(int64_t rows, int nvec) {
  const int64_t need = (rows + ln_rows_per_block(nvec) - 1) / ln_rows_per_block(nvec);
  return (int)(need < 1 ? 1 : need > 1024 ? 1024 : need);
}

#define SH_LN_DISPATCH(CALL)          \
  if (nvec <= 16) { CALL(16, 1); }    \
  else if (nvec <= 64) { CALL(64, 1); }   \
  else if (nvec <= 128) { CALL(64, 2); }  \
  else if (nvec <= 256) { CALL(64, 4); }  \
  else if (nvec <= 512) { CALL(256, 2); } \
  else if (nvec <= 1024) { CALL(256, 4); } \
  else { CALL(256, 8); }

}  // namespace sh

using namespace sh;

extern "C" {

int simhand_layer_norm_fwd(const void* x, const float* gamma, const float* beta, float eps, int relu, void* y, float* mean, float* rstd, int64_t rows,
                           int cols, int dtype, sh_stream_t stream) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "layer_norm_fwd: dtype %d", dtype);
  SH_REQUIRE(rows >= 0 && cols >= 1 && ln_nvec(cols, dtype) <= kLnMaxVec, "layer_norm_fwd: rows=%lld cols=%d (at most %d columns)", (long long)rows, cols,
             kLnMaxVec * (dtype == SH_F32 ? 4 : 8));
  SH_REQUIRE(gamma && beta && (rows == 0 || (x && y && mean && rstd)), "layer_norm_fwd: NULL argument");
  SH_REQUIRE(eps >= 0.f, "layer_norm_fwd: eps < 0");
  if (rows == 0) return 0;
  const int nvec = ln_nvec(cols, dtype);
  const int64_t grid = (rows + ln_rows_per_block(nvec) - 1) / ln_rows_per_block(nvec);
  SH_REQUIRE(grid < (1ll << 31), "layer_norm_fwd: too many rows");
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(SH_PROF_BN, s, 0, 2.0 * rows * cols * (dtype == SH_F32 ? 4 : 2));
#define SH_CALL(G, NV)                                                                                                                           \
  if (dtype == SH_F32)                                                                                                                           \
    layer_norm_fwd_kernel<float, G, NV><<<(unsigned)grid, 256, 0, s>>>((const float*)x, gamma, beta, eps, relu, (float*)y, mean, rstd, rows, cols); \
  else                                                                                                                                           \
    layer_norm_fwd_kernel<bf16_t, G, NV><<<(unsigned)grid, 256, 0, s>>>((const bf16_t*)x, gamma, beta, eps, relu, (bf16_t*)y, mean, rstd, rows, cols)
  SH_LN_DISPATCH(SH_CALL)
#undef SH_CALL
  return check_launch("layer_norm_fwd");
}

size_t simhand_layer_norm_bwd_workspace_bytes(int64_t rows, int cols, int dtype) {
  if (rows < 0 || cols < 1) return 0;
  return (size_t)ln_bwd_blocks(rows, ln_nvec(cols, dtype)) * 2 * cols * sizeof(float);
}

int simhand_layer_norm_bwd(const void* dy, const void* x, const uint8_t* x_codes, const uint8_t* x_exps, const float* gamma, const float* beta,
                           const float* mean, const float* rstd, int relu, void* dx, float* dgamma_dbeta, int64_t rows, int cols, int dtype,
                           void* workspace, size_t workspace_bytes, sh_stream_t stream) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "layer_norm_bwd: dtype %d", dtype);
  SH_REQUIRE(rows >= 0 && cols >= 1 && ln_nvec(cols, dtype) <= kLnMaxVec, "layer_norm_bwd: rows=%lld cols=%d (at most %d columns)", (long long)rows, cols,
             kLnMaxVec * (dtype == SH_F32 ? 4 : 8));
  const bool a8 = x_codes != nullptr;
  SH_REQUIRE(!a8 || (x_exps && !x), "layer_norm_bwd: pass either x or its codes and exponents");
  SH_REQUIRE(gamma && beta && dgamma_dbeta && (rows == 0 || (dy && (x || a8) && mean && rstd && dx)), "layer_norm_bwd: NULL argument");
  const int nvec = ln_nvec(cols, dtype);
  const int grid = ln_bwd_blocks(rows, nvec);
  SH_REQUIRE(workspace && workspace_bytes >= simhand_layer_norm_bwd_workspace_bytes(rows, cols, dtype), "layer_norm_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  const double eb = dtype == SH_F32 ? 4 : 2;
  ProfScope ps(SH_PROF_BN, s, 0, (double)rows * cols * (2 * eb + (a8 ? 1.03125 : eb)));
  float* part = (float*)workspace;
#define SH_ONE(T, G, NV, A8)                                                                                                                    \
  layer_norm_bwd_kernel<T, G, NV, A8><<<grid, 256, 0, s>>>((const T*)dy, (const T*)x, x_codes, x_exps, gamma, beta, mean, rstd, relu, (T*)dx, part, rows, cols)
#define SH_CALL(G, NV)                        \
  if (dtype == SH_F32) {                      \
    if (a8) SH_ONE(float, G, NV, true);       \
    else SH_ONE(float, G, NV, false);         \
  } else {                                    \
    if (a8) SH_ONE(bf16_t, G, NV, true);      \
    else SH_ONE(bf16_t, G, NV, false);        \
  }
  SH_LN_DISPATCH(SH_CALL)
#undef SH_CALL
#undef SH_ONE
  if (check_launch("layer_norm_bwd")) return 1;
  return fold_columns(part, grid, 2 * cols, dgamma_dbeta, s);
}

}  // extern "C"
