// Layer norm over the last dimension, forward and backward (the BatchNorm of the projection head with statistics per ROW instead of per batch: the
// result of a row depends on no other row: bit for bit the same in any batch, on any number of ranks, without a collective).
//
//   m = sum x / C, v = sum (x - m)^2 / C, r = 1 / sqrt(v + eps), h = (x - m) r, y = h gamma + beta, optionally max(y, 0)
//   backward, u = dy (ReLU: where h gamma + beta > 0), g = u gamma:  dx = r (g - mean(g) - h mean(g h)), dgamma = sum_rows u h, dbeta = sum_rows u
//
// One pass over the data each way: a group of G lanes holds a whole row in registers (NV 16-byte vectors per lane), so the variance is summed about
// the finished mean (no E[x^2] - m^2 cancellation) and nothing is read twice.  Statistics and sums are fp32, the column sums over row blocks are
// folded in 64 bits in a fixed order (bit-reproducible).  Bound by HBM: 2 (3) elements of traffic per element forward (backward).
// Measured: forward 100352 x 2048 bf16 154 us (5.3 TB/s; a large copy reaches 4.8), 256 x 512 fp32 3.0 (10 with the call around it); backward 100352 x 2048 bf16 230 (5.4 TB/s), 33001 x 777
// fp16 from codes 35 + 4 for the fold (HBM moves 139 MB at 4.0 TB/s, the vector units are 40 % and the LDS 36 % busy, the waves, three a SIMD, wait two thirds of their time: latency),
// 2048 x 512 fp32 with ReLU 5.8 + 3.2.
#include "rows.h"

namespace sh {

// sums of two values over the G lanes that share a row (G = 16, 32 or 64: inside a wave, on DPP and the row swaps -- no LDS round trips; G = 256: the whole block through
// LDS), the same bits in every lane
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float swap16_add(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap32_add(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
template <int G> __device__ __forceinline__ void group_sum2(float& a, float& b, float (*red)[2]) {
  a = dpp_add<0xB1>(a); b = dpp_add<0xB1>(b);      // lanes 1, 0, 3, 2 of every four
  a = dpp_add<0x4E>(a); b = dpp_add<0x4E>(b);      // 2, 3, 0, 1
  a = dpp_add<0x141>(a); b = dpp_add<0x141>(b);    // mirrored in every eight
  a = dpp_add<0x140>(a); b = dpp_add<0x140>(b);    // mirrored in every sixteen
  if constexpr (G >= 32) { a = swap16_add(a); b = swap16_add(b); }
  if constexpr (G >= 64) { a = swap32_add(a); b = swap32_add(b); }
  if constexpr (G == 256) {
    __syncthreads();  // the previous use of red is over
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6][0] = a;
      red[threadIdx.x >> 6][1] = b;
    }
    __syncthreads();
    a = (red[0][0] + red[1][0]) + (red[2][0] + red[3][0]);
    b = (red[0][1] + red[1][1]) + (red[2][1] + red[3][1]);
  }
}

// h gamma + beta in two roundings, in the forward and in the backward pass alike: the ReLU gate that the backward pass recomputes is the forward's
__device__ __forceinline__ float ln_affine(float x, float m, float r, float g, float b, float& h) {
#pragma clang fp contract(off)
  const float d = x - m;
  h = d * r;
  const float t = h * g;
  return t + b;
}

// Vector i of lane t: columns at .. at + N - 1, of which lo .. hi - 1 count.  RAG = 1 (cols no multiple of the vector): the last vector of a row is moved back to end with the
// row -- one whole load and store, the columns it shares with its neighbour are written twice with the same values and counted once (lo).  RAG = 2: rows shorter than
// a vector go element by element (hi); a variant of its own: inlined into the loops of RAG = 1 its branches make them ten times as long (33001 x 777 from codes 38 us, without 34).
template <int N, int RAG> struct LnVec {
  int at, lo, hi;
  bool on;
  __device__ __forceinline__ LnVec(int c, int cols) : at(c), lo(0), hi(N), on(c < cols) {
    if constexpr (RAG == 1) {
      if (c + N > cols) {
        at = cols - N;
        lo = c - at;
      }
    }
    if constexpr (RAG == 2) hi = cols;
  }
  __device__ __forceinline__ bool counts(int e) const { return RAG == 0 || (RAG == 1 ? e >= lo : e < hi); }
  __device__ __forceinline__ bool exists(int e) const { return RAG != 2 || e < hi; }
  template <typename T> __device__ __forceinline__ uint4 load(const T* row) const {
    if constexpr (RAG == 2) return ld_chunk<T>(row + at, hi);
    return ld16_any(row + at);
  }
  template <typename T> __device__ __forceinline__ void store(T* row, const uint4& v) const {
    if constexpr (RAG == 2) st_chunk<T>(row + at, hi, v);
    else st16_any(row + at, v);
  }
  __device__ __forceinline__ void load_f32(const float* p, float (&o)[N]) const { ld_f32<N>(p + at, RAG == 2 ? hi : N, o); }
};

// KEEP: the ReLU's gate is written too, one byte a vector (a variant of its own: as a branch it cost the others 4 % at 100352 x 2048 bf16)
template <typename T, int G, int NV, int RAG, bool KEEP>
__global__ __launch_bounds__(256) void layer_norm_fwd_kernel(const T* __restrict__ x, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             float eps, int relu, T* __restrict__ y, uint8_t* __restrict__ gate, float* __restrict__ mean,
                                                             float* __restrict__ rstd, long long rows, int cols) {
  constexpr int VE = Vec16<T>::N, RB = 256 / G;
  __shared__ float red[4][2];
  const int t = threadIdx.x % G;
  const long long row = (long long)blockIdx.x * RB + threadIdx.x / G;
  const bool live = row < rows;
  const T* src = x + (live ? row : 0) * cols;
  float v[NV][VE];
  float s = 0.f, unused = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const LnVec<VE, RAG> w((i * G + t) * VE, cols);
    uint4 q = make_uint4(0u, 0u, 0u, 0u);
    if (w.on) q = w.template load<T>(src);
    unpack16<T>(q, v[i]);
#pragma unroll
    for (int e = 0; e < VE; ++e) s += w.counts(e) ? v[i][e] : 0.f;
  }
  group_sum2<G>(s, unused, red);
  const float m = s / (float)cols;
  float q2 = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const LnVec<VE, RAG> w((i * G + t) * VE, cols);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const float d = v[i][e] - m;
      q2 += w.on && w.counts(e) ? d * d : 0.f;
    }
  }
  group_sum2<G>(q2, unused, red);
  const float r = 1.f / sqrtf(q2 / (float)cols + eps);
  if (!live) return;
  if (t == 0) {
    mean[row] = m;
    rstd[row] = r;
  }
  T* dst = y + row * cols;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const LnVec<VE, RAG> w((i * G + t) * VE, cols);
    if (!w.on) continue;
    float ga[VE], be[VE], o[VE];
    w.load_f32(gamma, ga);
    w.load_f32(beta, be);
    unsigned bits = 0u;
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      float h;
      o[e] = ln_affine(v[i][e], m, r, ga[e], be[e], h);
      if constexpr (KEEP) bits |= w.exists(e) && o[e] > 0.f ? 1u << e : 0u;
      if (KEEP || relu) o[e] = o[e] <= 0.f ? 0.f : o[e];
    }
    w.template store<T>(dst, pack16<T>(o));
    if constexpr (KEEP) gate[row * ((cols + VE - 1) / VE) + i * G + t] = (uint8_t)bits;
  }
}

// A8: x comes as its 8-bit checkpoint (codes + exponents).  GATE: 0 no ReLU, 1 its gate recomputed from x, 2 the gate that the forward pass kept (one byte a vector, laid out as
// there): from codes the recomputed sign is wrong wherever the codes' rounding carries a value across zero -- a whole gradient let through or lost, not a rounding of one.
// part [gridDim.x][2][cols]: sums of u h and u over the block's rows.
// A row group walks its rows with the next row's loads in flight; gamma and beta wait in LDS (G < 256), which the column sums reuse at the end.
// blocks of the backward kernel per CU, by the values a lane holds (registers); the grid is as many as run at once
__host__ __device__ constexpr int ln_bwd_occupancy(int nv, bool fp32, bool rag) {
  if (fp32) return nv <= 1 ? 8 : nv <= 2 ? 5 : nv <= 4 ? 3 : 1;
  return nv <= 1 ? 6 : nv <= 2 ? (rag ? 3 : 4) : nv <= 4 ? 2 : 1;
}

template <typename T, int G, int NV, bool A8, int RAG, int GATE>
__global__ __launch_bounds__(256, ln_bwd_occupancy(NV, sizeof(T) == 4, RAG != 0)) void layer_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                             const uint8_t* __restrict__ exps, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, const float* __restrict__ mean,
                                                             const float* __restrict__ rstd, const uint8_t* __restrict__ gate, T* __restrict__ dx,
                                                             float* __restrict__ part, long long rows, int cols) {
  constexpr int VE = Vec16<T>::N, RB = 256 / G, W8 = VE / 4;
  constexpr bool GLOBAL = G == 256;  // wide rows: gamma / beta come from the caches
  __shared__ float red[4][2];
  __shared__ float fold[2][GLOBAL ? 1 : G * NV * VE];
  const int t = threadIdx.x % G, sub = threadIdx.x / G;
  const int eb = (cols + kAct8Block - 1) / kAct8Block;
  float ag[NV][VE], ab[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < VE; ++e) ag[i][e] = ab[i][e] = 0.f;
  if constexpr (!GLOBAL) {
    for (int c = threadIdx.x; c < cols || c < VE; c += 256) {  // (a row shorter than a vector: zeros behind it)
      fold[0][c] = c < cols ? gamma[c] : 0.f;
      fold[1][c] = c < cols ? beta[c] : 0.f;
    }
    __syncthreads();
  }
  const float inv = 1.f / (float)cols;
  // the raw operands of one row
  uint4 qd[NV], qx[A8 ? 1 : NV];
  unsigned qc[A8 ? NV : 1][W8];
  unsigned qe[A8 ? NV : 1];  // exponents of the vector's first and last column
  unsigned qg[GATE == 2 ? NV : 1];
  float qm, qr;
  auto fetch = [&](long long row) __attribute__((always_inline)) {
    const bool live = row < rows;
    const long long rr = live ? row : rows - 1;
    qm = mean[rr];
    qr = rstd[rr];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const LnVec<VE, RAG> w((i * G + t) * VE, cols);
      if (!w.on) continue;
      qd[i] = w.template load<T>(dy + rr * cols);
      if constexpr (GATE == 2) qg[i] = gate[rr * ((cols + VE - 1) / VE) + i * G + t];
      if constexpr (A8) {
        act8_ld_codes<VE>(codes + rr * cols + w.at, RAG == 2 ? w.hi : VE, qc[i]);
        const uint8_t* ex = exps + rr * eb;
        qe[i] = ex[w.at / kAct8Block];
        if constexpr (RAG == 1) qe[i] |= (unsigned)ex[(w.at + VE - 1) / kAct8Block] << 8;
      } else {
        qx[i] = w.template load<T>(x + rr * cols);
      }
    }
  };
  const long long stride = (long long)gridDim.x * RB;
  const long long first = (long long)blockIdx.x * RB;
  if (first < rows) fetch(first + sub);
  for (long long row0 = first; row0 < rows; row0 += stride) {
    const long long row = row0 + sub;
    const bool live = row < rows;
    const float m = qm, r = qr, mr = m * r;
    float h[NV][VE], u[NV][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const LnVec<VE, RAG> w((i * G + t) * VE, cols);
      if (!w.on) continue;
      unpack16<T>(qd[i], u[i]);
      if constexpr (GATE == 2) {
#pragma unroll
        for (int e = 0; e < VE; ++e) u[i][e] = qg[i] >> e & 1u ? u[i][e] : 0.f;
      }
      if constexpr (A8) {
        const float s0 = act8_scale(qe[i] & 0xffu);
#pragma unroll
        for (int k = 0; k < W8; ++k) act8_decode4(qc[i][k], s0, &h[i][4 * k]);
        if constexpr (RAG == 1) {  // a vector that was moved back may span two blocks of 32
          const int edge = kAct8Block - w.at % kAct8Block;
          if (edge < VE) {
            const float s1 = act8_scale(qe[i] >> 8);
            float o[VE];
#pragma unroll
            for (int k = 0; k < W8; ++k) act8_decode4(qc[i][k], s1, o + 4 * k);
#pragma unroll
            for (int e = 0; e < VE; ++e) h[i][e] = e < edge ? h[i][e] : o[e];
          }
        }
      } else {
        unpack16<T>(qx[i], h[i]);
      }
    }
    if (row0 + stride < rows) fetch(row + stride);
    float s1 = 0.f, s2 = 0.f;
    // Three waves a SIMD hide no instruction that need not be there: the gate is a variant of its own (33001 x 777 from codes 38 us, the recomputed one 45), and
    // only a row's ragged last vector -- never in the first half of the lane's vectors -- masks what its neighbour counts.
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const LnVec<VE, RAG> w((i * G + t) * VE, cols);
      if (!w.on || !live) continue;
      float ga[VE], be[VE];
      if constexpr (GLOBAL) {
        w.load_f32(gamma, ga);
        if constexpr (GATE == 1) w.load_f32(beta, be);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          ga[e] = fold[0][w.at + e];
          if constexpr (GATE == 1) be[e] = fold[1][w.at + e];
        }
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if constexpr (GATE == 1) {
          if (!(ln_affine(h[i][e], m, r, ga[e], be[e], h[i][e]) > 0.f)) u[i][e] = 0.f;
        } else {
          h[i][e] = fmaf(h[i][e], r, -mr);  // off by U of |m r| more than (x - m) r, which the mean's own rounding costs already
        }
        const float uc = RAG != 0 && 2 * i >= NV - 1 ? (w.counts(e) ? u[i][e] : 0.f) : u[i][e];
        const float gc = uc * ga[e];
        ag[i][e] += uc * h[i][e];
        ab[i][e] += uc;
        s1 += gc;
        s2 += gc * h[i][e];
        u[i][e] = RAG != 0 && 2 * i >= NV - 1 ? u[i][e] * ga[e] : gc;
      }
    }
    group_sum2<G>(s1, s2, red);
    s1 *= inv * r;
    s2 *= inv * r;
    if (!live) continue;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const LnVec<VE, RAG> w((i * G + t) * VE, cols);
      if (!w.on) continue;
      float o[VE];
#pragma unroll
      for (int e = 0; e < VE; ++e) o[e] = fmaf(r, u[i][e], -fmaf(h[i][e], s2, s1));  // r (g - mean(g) - h mean(g h))
      w.template store<T>(dx + row * cols, pack16<T>(o));
    }
  }
  // the block's column sums: its row groups one after the other (fixed order)
  float* out = part + (long long)blockIdx.x * 2 * cols;
  if constexpr (GLOBAL) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const LnVec<VE, RAG> w((i * G + t) * VE, cols);
#pragma unroll
      for (int e = 0; e < VE; ++e)
        if (w.on && w.counts(e)) {
          out[w.at + e] = ag[i][e];
          out[cols + w.at + e] = ab[i][e];
        }
    }
  } else {
    __syncthreads();  // gamma and beta have been read
    for (int k = 0; k < RB; ++k) {
      if (sub == k) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const LnVec<VE, RAG> w((i * G + t) * VE, cols);
#pragma unroll
          for (int e = 0; e < VE; ++e)
            if (w.on && w.counts(e)) {
              fold[0][w.at + e] = (k == 0 ? 0.f : fold[0][w.at + e]) + ag[i][e];
              fold[1][w.at + e] = (k == 0 ? 0.f : fold[1][w.at + e]) + ab[i][e];
            }
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

// [nblk][n] -> [n]: 32 columns x 32 groups of partial rows per block, 8 loads in flight per thread (the fold is all latency: 4 dependent rounds for 1024 partial rows; four
// groups of 64 columns took 100 us of a 134 us backward pass over 33001 x 777)
__global__ __launch_bounds__(1024) void fold_columns_kernel(const float* __restrict__ part, int nblk, int n, float* __restrict__ out) {
  __shared__ double red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  double a = 0.0;
  if (c < n) {
    int b = ty;
    for (; b + 7 * 32 < nblk; b += 8 * 32) {
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = part[(long long)(b + 32 * i) * n + c];
#pragma unroll
      for (int i = 0; i < 8; ++i) a += (double)v[i];
    }
    for (; b < nblk; b += 32) a += (double)part[(long long)b * n + c];
  }
  red[ty][tx] = a;
  __syncthreads();
  for (int o = 16; o > 0; o >>= 1) {
    if (ty < o) red[ty][tx] += red[ty + o][tx];
    __syncthreads();
  }
  if (ty == 0 && c < n) out[c] = (float)red[0][tx];
}
int fold_columns(const float* part, int nblk, int n, float* out, hipStream_t s) {
  fold_columns_kernel<<<ceil_div(n, 32), 1024, 0, s>>>(part, nblk, n, out);
  return check_launch("fold_columns");
}

// (G, NV) by the row's 16-byte vectors: the smallest group that holds the row
static int ln_nvec(int cols, int dtype) { return (cols + (dtype == SH_F32 ? 4 : 8) - 1) / (dtype == SH_F32 ? 4 : 8); }
static int ln_rag(int cols, int dtype) { return cols % (dtype == SH_F32 ? 4 : 8) == 0 ? 0 : cols >= (dtype == SH_F32 ? 4 : 8) ? 1 : 2; }
constexpr int kLnMaxVec = 2048;
static int ln_rows_per_block(int nvec) { return nvec <= 16 ? 16 : nvec <= 32 ? 8 : nvec <= 256 ? 4 : 1; }
static int ln_nv(int nvec) { return nvec <= 64 ? 1 : nvec <= 128 ? 2 : nvec <= 256 ? 4 : nvec <= 512 ? 2 : nvec <= 1024 ? 4 : 8; }
// backward blocks: one round of what the CUs hold (each then walks its share of the rows with the next row in flight; a second, part-empty round cost a third of the
// pass over 33001 x 777), and no more partial sums than that
static int ln_bwd_blocks(int64_t rows, int cols, int dtype) {
  const int nvec = ln_nvec(cols, dtype);
  if (rows <= 8 * ln_rows_per_block(nvec)) return 1;  // few rows: one block writes the column sums itself, a launch (of the fold) and a workspace less
  const int64_t need = (rows + ln_rows_per_block(nvec) - 1) / ln_rows_per_block(nvec);
  const int64_t most = 256 * ln_bwd_occupancy(ln_nv(nvec), dtype == SH_F32, cols % (dtype == SH_F32 ? 4 : 8) != 0);
  return (int)(need < 1 ? 1 : need > most ? most : need);
}

#define SH_LN_DISPATCH(CALL)          \
  if (nvec <= 16) { CALL(16, 1); }    \
  else if (nvec <= 32) { CALL(32, 1); }   \
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
  return simhand_layer_norm_fwd_ex(x, gamma, beta, eps, relu, y, nullptr, mean, rstd, rows, cols, dtype, stream);
}

int simhand_layer_norm_fwd_ex(const void* x, const float* gamma, const float* beta, float eps, int relu, void* y, uint8_t* gate, float* mean, float* rstd,
                              int64_t rows, int cols, int dtype, sh_stream_t stream) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "layer_norm_fwd: dtype %d", dtype);
  SH_REQUIRE(rows >= 0 && cols >= 1 && ln_nvec(cols, dtype) <= kLnMaxVec, "layer_norm_fwd: rows=%lld cols=%d (at most %d columns)", (long long)rows, cols,
             kLnMaxVec * (dtype == SH_F32 ? 4 : 8));
  SH_REQUIRE(gamma && beta && (rows == 0 || (x && y && mean && rstd)), "layer_norm_fwd: NULL argument");
  SH_REQUIRE(eps >= 0.f, "layer_norm_fwd: eps < 0");
  SH_REQUIRE(!gate || relu, "layer_norm_fwd: a gate without the ReLU");
  if (rows == 0) return 0;
  const int nvec = ln_nvec(cols, dtype);
  const int rpb = ln_rows_per_block(nvec);
  const int64_t most = (1ll << 23) * rpb;  // rows of a launch: its threads are counted in 32 bits
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(SH_PROF_BN, s, 0, 2.0 * rows * cols * (dtype == SH_F32 ? 4 : 2));
  const int rag = ln_rag(cols, dtype);
#define SH_LAUNCH(T, G, NV, RAG, KEEP)                                                                                        \
  layer_norm_fwd_kernel<T, G, NV, RAG, KEEP><<<grid, 256, 0, s>>>((const T*)x + r * cols, gamma, beta, eps, relu, (T*)y + r * cols, \
                                                                  gate + (KEEP ? r * nvec : 0), mean + r, rstd + r, n, cols)
#define SH_ONE(T, G, NV, RAG)                  \
  {                                            \
    if (gate) SH_LAUNCH(T, G, NV, RAG, true);  \
    else SH_LAUNCH(T, G, NV, RAG, false);      \
  }
#define SH_CALL(G, NV)                       \
  if (dtype == SH_F32) {                     \
    if (rag) SH_ONE(float, G, NV, 1)         \
    else SH_ONE(float, G, NV, 0)             \
  } else {                                   \
    if (rag) SH_ONE(bf16_t, G, NV, 1)        \
    else SH_ONE(bf16_t, G, NV, 0)            \
  }
  for (int64_t r = 0; r < rows; r += most) {
    const int64_t n = rows - r < most ? rows - r : most;
    const unsigned grid = (unsigned)((n + rpb - 1) / rpb);
    if (rag == 2) {
      if (dtype == SH_F32) SH_ONE(float, 16, 1, 2)
      else SH_ONE(bf16_t, 16, 1, 2)
    } else {
      SH_LN_DISPATCH(SH_CALL)
    }
  }
#undef SH_CALL
#undef SH_ONE
#undef SH_LAUNCH
  return check_launch("layer_norm_fwd");
}

size_t simhand_layer_norm_bwd_workspace_bytes(int64_t rows, int cols, int dtype) {
  if (rows < 0 || cols < 1) return 0;
  const int blocks = ln_bwd_blocks(rows, cols, dtype);
  return blocks > 1 ? (size_t)blocks * 2 * cols * sizeof(float) : 0;
}

int simhand_layer_norm_bwd(const void* dy, const void* x, const uint8_t* x_codes, const uint8_t* x_exps, const float* gamma, const float* beta,
                           const float* mean, const float* rstd, int relu, void* dx, float* dgamma_dbeta, int64_t rows, int cols, int dtype,
                           void* workspace, size_t workspace_bytes, sh_stream_t stream) {
  return simhand_layer_norm_bwd_ex(dy, x, x_codes, x_exps, gamma, beta, mean, rstd, relu, nullptr, dx, dgamma_dbeta, rows, cols, dtype, workspace, workspace_bytes, stream);
}

int simhand_layer_norm_bwd_ex(const void* dy, const void* x, const uint8_t* x_codes, const uint8_t* x_exps, const float* gamma, const float* beta,
                              const float* mean, const float* rstd, int relu, const uint8_t* gate, void* dx, float* dgamma_dbeta, int64_t rows, int cols,
                              int dtype, void* workspace, size_t workspace_bytes, sh_stream_t stream) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "layer_norm_bwd: dtype %d", dtype);
  SH_REQUIRE(rows >= 0 && cols >= 1 && ln_nvec(cols, dtype) <= kLnMaxVec, "layer_norm_bwd: rows=%lld cols=%d (at most %d columns)", (long long)rows, cols,
             kLnMaxVec * (dtype == SH_F32 ? 4 : 8));
  const bool a8 = x_codes != nullptr;
  SH_REQUIRE(!a8 || (x_exps && !x), "layer_norm_bwd: pass either x or its codes and exponents");
  SH_REQUIRE(!gate || relu, "layer_norm_bwd: a gate without the ReLU");
  SH_REQUIRE(gamma && beta && dgamma_dbeta && (rows == 0 || (dy && (x || a8) && mean && rstd && dx)), "layer_norm_bwd: NULL argument");
  const int nvec = ln_nvec(cols, dtype);
  const int grid = ln_bwd_blocks(rows, cols, dtype);
  SH_REQUIRE(grid == 1 || (workspace && workspace_bytes >= simhand_layer_norm_bwd_workspace_bytes(rows, cols, dtype)), "layer_norm_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  const double eb = dtype == SH_F32 ? 4 : 2;
  ProfScope ps(SH_PROF_BN, s, 0, (double)rows * cols * (2 * eb + (a8 ? 1.03125 : eb)));
  float* part = grid == 1 ? dgamma_dbeta : (float*)workspace;
  const int rag = ln_rag(cols, dtype);
#define SH_LAUNCH(T, G, NV, A8, RAG, GATE)                                                                                                           \
  layer_norm_bwd_kernel<T, G, NV, A8, RAG, GATE><<<grid, 256, 0, s>>>((const T*)dy, (const T*)x, x_codes, x_exps, gamma, beta, mean, rstd, gate, (T*)dx, part, \
                                                                      rows, cols)
#define SH_ONE(T, G, NV, A8, RAG)                 \
  if (gate) SH_LAUNCH(T, G, NV, A8, RAG, 2);      \
  else if (relu) SH_LAUNCH(T, G, NV, A8, RAG, 1); \
  else SH_LAUNCH(T, G, NV, A8, RAG, 0)
#define SH_TYPE(T, G, NV)                       \
  if (a8) {                                     \
    if (rag) { SH_ONE(T, G, NV, true, 1); }     \
    else { SH_ONE(T, G, NV, true, 0); }         \
  } else {                                      \
    if (rag) { SH_ONE(T, G, NV, false, 1); }    \
    else { SH_ONE(T, G, NV, false, 0); }        \
  }
#define SH_CALL(G, NV)                        \
  if (dtype == SH_F32) {                      \
    SH_TYPE(float, G, NV)                     \
  } else {                                    \
    SH_TYPE(bf16_t, G, NV)                    \
  }
#define SH_SHORT(T)                        \
  if (a8) { SH_ONE(T, 16, 1, true, 2); }   \
  else { SH_ONE(T, 16, 1, false, 2); }
  if (rag == 2) {
    if (dtype == SH_F32) { SH_SHORT(float) }
    else { SH_SHORT(bf16_t) }
  } else {
    SH_LN_DISPATCH(SH_CALL)
  }
#undef SH_SHORT
#undef SH_CALL
#undef SH_TYPE
#undef SH_ONE
#undef SH_LAUNCH
  if (check_launch("layer_norm_bwd")) return 1;
  if (grid == 1) return 0;
  return fold_columns(part, grid, 2 * cols, dgamma_dbeta, s);
}

}  // extern "C"
