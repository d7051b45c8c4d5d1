// The linear operator of an MLP / projection head for any sizes:  y = act(x w^T + bias) + residual  and its gradients.
//
//   x [rows][in], w [out][in], y / pre / residual [rows][out] in fp32 or the build's 16-bit type; bias, db, dw fp32; products accumulate in fp32 on the matrix cores
//   (fp32 operands on v_mfma_f32_16x16x4_f32: exact products, no reduced-precision mode), every output is rounded once.
//   act backward: dz = dy act'(pre), db = sum_rows dz (of the unrounded dz);   dx = dz w;   dw = dz^T x, x possibly as its 8-bit checkpoint.
//
// linear_gemm_kernel (forward, and dx with w transposed first; rows at any element address): out [M][N] = a [M][K] b[N][K]^T, tiles of 128 x 128 or 64 x 64, 128 bytes of K a step, both
// operands global -> registers -> LDS with the next step's loads in flight under the MFMAs (a second step in flight and a second buffer: no faster).
// 100000 x 777 -> 333: bf16 113 to 119 us (HBM 2 TB/s, matrix cores 22 % busy: two barriers a step), fp32 532 (336 at the fp32 rate of a large matrix product).  The operands are swapped (b is the MFMA's first one), and b's rows are permuted inside
// the tile, so that a lane ends with 8 consecutive columns of one row: bias, residual, pre-activation and output move as 16-byte vectors.
// linear_wgrad_kernel: dw [N][K] = dz^T x, the reduction runs over rows: tiles of 64 or 128 squared over a range of rows (split), 16-bit operands are read transposed from LDS
// (ds_read_b64_tr_b16); the splits' fp32 partial sums are added in a fixed order by a second launch.  100000 x 777 -> 333: bf16 109 us, fp32 608; 400000 x 64 -> 64 bf16 26;
// from codes 6422528 x 256 -> 64 603 (4.2 TB/s), 1605632 x 512 -> 128 362 (3.5 TB/s); 2048 x 2048 -> 512 fp32 53 (28 at that rate).
#include "linear.h"

namespace sh {

// TILE = 128: each of the 4 waves a 64 x 64 quarter; 64: a 32 x 32 quarter
template <typename T, int TILE>
__global__ __launch_bounds__(256, TILE == 128 ? 2 : 4) void linear_gemm_kernel(LinearArgs p) {
  constexpr int VE = Vec16<T>::N, KE = 128 / sizeof(T);  // elements per 16-byte chunk / per k-step (a tile row is 8 chunks)
  constexpr int Q = TILE / 32, HALF = TILE / 2;          // MFMA tiles per wave and direction, also staging rounds
  __shared__ __attribute__((aligned(16))) char smem[2 * TILE * 128];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int li = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  const unsigned logical = xcd_order(blockIdx.x, gridDim.x);
  const int n0 = (int)(logical % p.n_tiles) * TILE;  // the n-tiles of a row tile are neighbours on one XCD: a is read from HBM once
  const long long m0 = (long long)(logical / p.n_tiles) * TILE;
  // staging: thread = chunk tid & 7 of rows (tid >> 3) + 32 i of either operand; LDS chunk position = chunk ^ (row's key).  Rows past the end repeat the last one (their
  // sums are never stored).
  const int sc = tid & 7, sr = tid >> 3;
  const T* pa[Q];
  const T* pb[Q];
#pragma unroll
  for (int i = 0; i < Q; ++i) {
    const long long m = m0 + sr + 32 * i;
    const int n = n0 + sr + 32 * i;
    pa[i] = (const T*)p.a + (m < p.M ? m : p.M - 1) * p.K;
    pb[i] = (const T*)p.b + (long long)(n < p.N ? n : p.N - 1) * p.ldb;
  }
  uint4 ra[Q], rb[Q];
  auto load = [&](int k0) {
    const int k = k0 + sc * VE;
    if (p.K >= VE) {
      const int at = kchunk_at<T>(k, p.K);
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        ra[i] = ld16_any(pa[i] + at);
        rb[i] = ld16_any(pb[i] + at);
      }
    } else {
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        ra[i] = ld_kchunk<T>(pa[i], k, p.K);
        rb[i] = ld_kchunk<T>(pb[i], k, p.K);
      }
    }
  };
  auto key_b = [](int row) { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); };
  f32x4 acc[Q][Q];
#pragma unroll
  for (int mi = 0; mi < Q; ++mi)
#pragma unroll
    for (int ni = 0; ni < Q; ++ni) acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};
  load(0);
  for (int k0 = 0; k0 < p.K; k0 += KE) {
    __syncthreads();
    if (k0 + KE > p.K && p.K >= VE) {
      const int gone = kchunk_gone<T>(k0 + sc * VE, p.K);
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        ra[i] = drop_first<T>(ra[i], gone);
        rb[i] = drop_first<T>(rb[i], gone);
      }
    }
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      const int row = sr + 32 * i;
      *reinterpret_cast<uint4*>(smem + row * 128 + ((sc ^ ((row >> 1) & 7)) * 16)) = ra[i];
      *reinterpret_cast<uint4*>(smem + TILE * 128 + row * 128 + ((sc ^ key_b(row)) * 16)) = rb[i];
    }
    __syncthreads();
    if (k0 + KE < p.K) load(k0 + KE);
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 fa[Q], fb[Q];
#pragma unroll
      for (int mi = 0; mi < Q; ++mi) {
        const int row = wm * HALF + mi * 16 + li;
        fa[mi] = *reinterpret_cast<const uint4*>(smem + row * 128 + (((kk * 4 + g) ^ ((row >> 1) & 7)) * 16));
      }
#pragma unroll
      for (int ni = 0; ni < Q; ++ni) {
        const int row = wn * HALF + lin_col(ni, li);
        fb[ni] = *reinterpret_cast<const uint4*>(smem + TILE * 128 + row * 128 + (((kk * 4 + g) ^ key_b(row)) * 16));
      }
#pragma unroll
      for (int mi = 0; mi < Q; ++mi)
#pragma unroll
        for (int ni = 0; ni < Q; ++ni) acc[mi][ni] = mma16<T>(fb[ni], fa[mi], acc[mi][ni]);
    }
  }
  linear_store_tile<T, Q, Q>(p, m0 + wm * HALF + li, n0 + wn * HALF + g * 8, acc);
}

// The same product with both operands by LDS-DMA, for rows of whole 16-byte chunks: several k-steps ahead, one barrier per step and nothing staged in registers.  Waves as 2 x 2, each
// QM x QN MFMA tiles: 128 x 128 (80 KB of LDS: activations two steps ahead, weights one), 128 x 64 (72 KB, two steps), 64 x 64 (80 KB, four steps: so small a tile is all
// latency).  One block's epilogue runs under the other's k-loop.  5001 x 1000 -> 333 fp16 12 us, 16 with gelu and the pre-activation; 2048 x 512 -> 2048 fp32 43 (28 at the fp32 rate
// of a large matrix product).  Twice the stages for grids of one block a CU: slower (13.9 us for 11.2); barrier in mid-step with the next fragments read ahead: 12.3.
// BT: b is stored [K][N] (dx = dz w reads w as it is, without a transposed copy): its tile is sub-tiles of 64 columns by K rows, 16-bit operands are read transposed
// (ds_read_b64_tr_b16; the activations' chunks are then read in the halves that match its row order), fp32 ones element by element.
__device__ uint4 g_lin_zero[8];  // read-only zeros

typedef __attribute__((ext_vector_type(4))) short s16x4_t;

template <typename T, int QM, int QN, bool BT>
__global__ __launch_bounds__(256, 2) void linear_dma_kernel(LinearArgs p) {
  constexpr int VE = Vec16<T>::N, KE = 128 / sizeof(T), BM = 32 * QM, BN = 32 * QN;
  constexpr int NA = QM == 2 ? 5 : 3, NB = QN == 4 ? 2 : NA;  // stages
  constexpr int A_BYTES = BM * 128, B_BYTES = BN * 128, B0 = NA * A_BYTES;
  __shared__ __attribute__((aligned(16))) char smem[NA * A_BYTES + NB * B_BYTES];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
  // inline asm: hipcc's wait-count pass would drain every outstanding LDS-DMA in front of each LDS read; the loop counts them itself
  auto dma16 = [](const void* src, unsigned lds_addr) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(src));
  };
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  const unsigned logical = xcd_order(blockIdx.x, gridDim.x);
  const int n0 = (int)(logical % p.n_tiles) * BN;
  const long long m0 = (long long)(logical / p.n_tiles) * BM;
  // instruction i of a wave fills tile rows 32 i + 8 wave .. + 7; lane = row lane >> 3, slot lane & 7; slot s holds chunk s ^ key(row)
  const int slot = lane & 7, lrow = wave * 8 + (lane >> 3);
  auto key_b = [](int row) __attribute__((always_inline)) -> int { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); };
  const int ka = (slot ^ ((lrow >> 1) & 7)) * VE;
  const char* zero = reinterpret_cast<const char*>(g_lin_zero) + slot * 16;
  const char* pa[QM];
#pragma unroll
  for (int i = 0; i < QM; ++i) {
    const long long m = m0 + lrow + 32 * i;
    pa[i] = reinterpret_cast<const char*>((const T*)p.a + (m < p.M ? m : p.M - 1) * p.K + ka);
  }
  // b [N][K]: as a.  b [K][N]: instruction i of a wave = number q = QN wave + i of the tile's; sub-tile q / 8, rows 8 (q % 8) (16 bits) or 4 (q % 8) (fp32) and following; the columns of
  // a row are rotated (16 bits: 32-byte groups by row / 2; fp32: 16-byte slots by 0, 1, 8, 9 for row / 4) so that what a read touches falls on different banks
  auto rot32 = [](int row) __attribute__((always_inline)) -> int { return ((row >> 2) & 1) + ((row >> 3) & 1) * 8; };
  const char* pb[QN];
  int kb[QN];       // the lane's first k of the chunk (b [N][K]) or its row (b [K][N]) inside a step
  bool inside[QN];
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    if constexpr (BT) {
      const int q = QN * wave + i, sub = q >> 3;
      int col;
      if constexpr (sizeof(T) == 2) {
        kb[i] = 8 * (q & 7) + (lane >> 3);
        col = n0 + sub * 64 + ((((slot >> 1) - (kb[i] >> 1)) & 3) * 16) + (slot & 1) * 8;
      } else {
        kb[i] = 4 * (q & 7) + (lane >> 4);
        col = n0 + sub * 64 + (((lane & 15) - rot32(kb[i])) & 15) * 4;
      }
      inside[i] = col < p.N;
      pb[i] = reinterpret_cast<const char*>((const T*)p.b + (long long)kb[i] * p.ldb + (inside[i] ? col : 0));
    } else {
      const int n = n0 + lrow + 32 * i;
      kb[i] = (slot ^ key_b(lrow)) * VE;
      inside[i] = true;
      pb[i] = reinterpret_cast<const char*>((const T*)p.b + (long long)(n < p.N ? n : p.N - 1) * p.ldb + kb[i]);
    }
  }
  const long long b_step = BT ? (long long)KE * p.ldb * (int)sizeof(T) : 128;
  auto issue_a = [&](int kt) __attribute__((always_inline)) {
    const bool ok = kt * KE + ka < p.K;
    const unsigned dst = lds0 + (kt % NA) * A_BYTES + wave * 1024;
#pragma unroll
    for (int i = 0; i < QM; ++i) dma16(ok ? pa[i] + kt * 128 : zero, dst + i * 4096);
  };
  auto issue_b = [&](int kt) __attribute__((always_inline)) {
    const unsigned dst = lds0 + B0 + (kt % NB) * B_BYTES;
#pragma unroll
    for (int i = 0; i < QN; ++i)
      dma16(inside[i] && kt * KE + kb[i] < p.K ? pb[i] + kt * b_step : zero, dst + (BT ? (QN * wave + i) * 1024 : wave * 1024 + i * 4096));
  };
  f32x4 acc[QM][QN];
#pragma unroll
  for (int mi = 0; mi < QM; ++mi)
#pragma unroll
    for (int ni = 0; ni < QN; ++ni) acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int nk = (p.K + KE - 1) / KE;
  const int akey = (li >> 1) & 7, fa0 = (wm * 16 * QM + li) * 128;
  const int rowb = wn * 16 * QN + lin_col(0, li);
  const int fb0 = rowb * 128 + ((g ^ key_b(rowb)) * 16);
  int bt[QN];  // BT: the lane's place in b's tile
#pragma unroll
  for (int ni = 0; ni < QN; ++ni) {
    if constexpr (sizeof(T) == 2) {
      const int row = 4 * g + (li >> 2), c = wn * 16 * QN + (ni >> 1) * 32 + (li & 3) * 8 + (ni & 1) * 4;
      bt[ni] = (c >> 6) * (KE * 128) + row * 128 + ((((c & 63) >> 4) + (row >> 1)) & 3) * 32 + (c & 15) * 2;
    } else {
      const int row = 4 * g, c = wn * 16 * QN + lin_col(ni, li);
      bt[ni] = (c >> 6) * (KE * 256) + row * 256 + ((((c & 63) >> 2) + rot32(row)) & 15) * 16 + (c & 3) * 4;
    }
  }
#pragma unroll
  for (int i = 0; i < NA - 1; ++i) {
    if (i < NB - 1) issue_b(i);
    issue_a(i);
  }
  for (int kt = 0; kt < nk; ++kt) {
    // all but what belongs to the steps behind kt alone has landed (NB = 2: the activations of step kt + 1); every wave is past step kt - 1
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(NB == 2 ? QM : (NA - 2) * (QM + QN)) : "memory");
    issue_b(kt + NB - 1);
    issue_a(kt + NA - 1);
    const char* sa = smem + (kt % NA) * A_BYTES;
    const char* sb = smem + B0 + (kt % NB) * B_BYTES;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 fa[QM], fb[QN];
#pragma unroll
      for (int ni = 0; ni < QN; ++ni) {
        if constexpr (!BT) {
          fb[ni] = *reinterpret_cast<const uint4*>(sb + (kk ? fb0 ^ 64 : fb0) + (lin_col(ni, 0) - lin_col(0, 0)) * 128);
        } else if constexpr (sizeof(T) == 2) {
          typedef s16x4_t __attribute__((address_space(3))) * lds_ptr;
          const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(sb + bt[ni] + kk * 4096)));
          const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(sb + bt[ni] + kk * 4096 + 2048)));
          fb[ni] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          const char* at = sb + bt[ni] + kk * 4096;
          fb[ni] = make_uint4(*reinterpret_cast<const unsigned*>(at), *reinterpret_cast<const unsigned*>(at + 256), *reinterpret_cast<const unsigned*>(at + 512),
                              *reinterpret_cast<const unsigned*>(at + 768));
        }
      }
#pragma unroll
      for (int mi = 0; mi < QM; ++mi) {
        const char* at = sa + fa0 + mi * 2048;
        if constexpr (BT && sizeof(T) == 2) {  // k = 32 kk + 4 g .. + 3 and 16 further: halves of chunks
          const uint2 lo = *reinterpret_cast<const uint2*>(at + (((kk * 4 + (g >> 1)) ^ akey) * 16) + (g & 1) * 8);
          const uint2 hi = *reinterpret_cast<const uint2*>(at + (((kk * 4 + 2 + (g >> 1)) ^ akey) * 16) + (g & 1) * 8);
          fa[mi] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        } else {
          fa[mi] = *reinterpret_cast<const uint4*>(at + (((kk * 4 + g) ^ akey) * 16));
        }
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int mi = 0; mi < QM; ++mi)
#pragma unroll
          for (int ni = 0; ni < QN; ++ni) acc[mi][ni] = mma16<T>(fb[ni], fa[mi], acc[mi][ni]);
      } else {  // element by element over all tiles: consecutive MFMAs do not wait for each other's sums
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int mi = 0; mi < QM; ++mi)
#pragma unroll
            for (int ni = 0; ni < QN; ++ni) {
              const unsigned b4[4] = {fb[ni].x, fb[ni].y, fb[ni].z, fb[ni].w}, a4[4] = {fa[mi].x, fa[mi].y, fa[mi].z, fa[mi].w};
              acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b4[e]), __uint_as_float(a4[e]), acc[mi][ni], 0, 0, 0);
            }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the DMAs past the end have landed before the LDS is given back
  linear_store_tile<T, QM, QN>(p, m0 + wm * 16 * QM + li, n0 + wn * 16 * QN + g * 8, acc);
}

// Few rows: a block of 8 waves makes 16 columns of up to 16 MT rows; every wave takes each eighth 64-byte piece of K, both operands go from memory straight into MFMA
// operands (no LDS: nothing is used twice), and the waves' sums meet in LDS.  What counts here is latency and the number of CUs that read w: 16 columns a block
// put 32 blocks on 512 columns: 8 x 2048 -> 512 fp32 8.3 us, of which the 4 MB of w are one.
template <typename T, int MT>
__global__ __launch_bounds__(512) void linear_skinny_kernel(LinearArgs p) {
  constexpr int VE = Vec16<T>::N, KE = 4 * VE, W = 8;  // elements of a lane group's four chunks
  __shared__ float red[W][MT][16][17];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const long long m0 = (long long)blockIdx.y * (16 * MT);
  const T* pb = (const T*)p.b + (long long)(n0 + li < p.N ? n0 + li : p.N - 1) * p.ldb;
  const T* pa[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const long long m = m0 + 16 * t + li;
    pa[t] = (const T*)p.a + (m < p.M ? m : p.M - 1) * p.K;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
  const int k_first = wave * KE + g * VE;
  constexpr int U = MT >= 4 ? 2 : MT == 2 ? 4 : 8;  // pieces in flight
  int k0 = k_first;
  for (; k0 - g * VE + (U - 1) * W * KE + KE <= p.K; k0 += U * W * KE) {  // U whole pieces
    uint4 b[U], a[U][MT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      b[u] = ld16_any(pb + k0 + u * W * KE);
#pragma unroll
      for (int t = 0; t < MT; ++t) a[u][t] = ld16_any(pa[t] + k0 + u * W * KE);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = mma16<T>(a[u][t], b[u], acc[t]);
  }
  for (; k0 - g * VE < p.K; k0 += W * KE) {
    const uint4 b = ld_kchunk<T>(pb, k0, p.K);
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = mma16<T>(ld_kchunk<T>(pa[t], k0, p.K), b, acc[t]);
  }
  // D[row m = 4 g + r][column n = li]
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wave][t][4 * g + r][li] = acc[t][r];
  __syncthreads();
  for (int i = tid; i < MT * 16 * 16; i += 512) {
    const int n = i & 15, m = (i >> 4) & 15, t = i >> 8;
    const long long row = m0 + 16 * t + m;
    const int col = n0 + n;
    if (row >= p.M || col >= p.N) continue;
    float z = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) z += red[w][t][m][n];
    if (p.bias != nullptr) z += p.bias[col];
    const long long at = row * p.N + col;
    if (p.pre != nullptr) Elem<T>::store((T*)p.pre + at, z);
    z = act_value(z, p.act);
    if (p.residual != nullptr) z += Elem<T>::load((const T*)p.residual + at);
    Elem<T>::store((T*)p.out + at, z);
  }
}

// w [n][k] -> wt [k][ldt], 32 x 32 tiles through LDS; columns n .. ldt - 1 are written as zeros
template <typename T> __global__ __launch_bounds__(256) void linear_transpose_kernel(const T* __restrict__ w, T* __restrict__ wt, int n, int k, int ldt) {
  __shared__ T tile[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = blockIdx.y * 32, k0 = blockIdx.x * 32;
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = n0 + ty + i, c = k0 + tx;
    tile[ty + i][tx] = (r < n && c < k) ? w[(long long)r * k + c] : (T)0;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    const int r = k0 + ty + i, c = n0 + tx;
    if (r < k && c < ldt) wt[(long long)r * ldt + c] = tile[tx][ty + i];
  }
}

// ---- dz = dy act'(pre), db ----------------------------------------------------------------------------------------------------
// One pass, bound by HBM: 100352 x 2048 bf16 with gelu 254 us (4.9 TB/s) and 5 for the fold of the blocks' sums.
// A block covers TX 16-byte vectors of columns (TX = 8 .. 64, the power of two at or above a narrow row's vectors) and 256 / TX rows at a time over its range of rows;
// part [row blocks][cols] = its column sums.  dz may be dy's buffer (no __restrict__ between them): a value is read before the same thread stores it, and what a moved-back vector reads of
// its neighbour's columns is dropped.
template <typename T, int TX>
__global__ __launch_bounds__(256) void linear_act_bwd_kernel(const T* dy, const T* __restrict__ pre, int act, T* dz, float* __restrict__ part,
                                                             long long rows, int cols, long long per_block) {
  constexpr int VE = Vec16<T>::N, TY = 256 / TX;
  __shared__ float red[TY][TX * VE + 1];
  const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
  const int c = (blockIdx.x * TX + tx) * VE;
  const long long r0 = (long long)blockIdx.y * per_block;
  const long long r1 = r0 + per_block < rows ? r0 + per_block : rows;
  float s[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) s[e] = 0.f;
  // a row's ragged last vector is read moved back, as the row's last VE columns; what it shares with its neighbour is neither summed nor stored (dz may be dy)
  const int left = cols - c, gone = left < VE && cols >= VE ? VE - left : 0;
  if (left > 0) {
    for (long long r = r0 + ty; r < r1; r += TY) {
      const long long at = r * cols + c;
      float d[VE];
      unpack16<T>(cols >= VE ? ld16_any(dy + at - gone) : ld_chunk<T>(dy + at, left), d);
      if (act != SH_ACT_NONE) {
        float z[VE];
        unpack16<T>(cols >= VE ? ld16_any(pre + at - gone) : ld_chunk<T>(pre + at, left), z);
        if (act == SH_ACT_RELU) {
#pragma unroll
          for (int e = 0; e < VE; ++e) d[e] = relu_grad(d[e], z[e]);
        } else {
#pragma unroll
          for (int e = 0; e < VE; ++e) d[e] *= act_slope(z[e], act);
        }
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) s[e] += d[e];
      if (dz != nullptr) {
        if (gone == 0) st_chunk<T>(dz + at, left, pack16<T>(d));
        else st_chunk<T>(dz + at, left, move_down<T>(pack16<T>(d), gone));
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VE; ++e)
    if (e >= gone) red[ty][tx * VE + e - gone] = s[e];
  __syncthreads();
  for (int i = threadIdx.x; i < TX * VE; i += 256) {
    const int col = blockIdx.x * TX * VE + i;
    if (col >= cols) continue;
    float a = 0.f;
#pragma unroll
    for (int y = 0; y < TY; ++y) a += red[y][i];
    part[(long long)blockIdx.y * cols + col] = a;
  }
}

// ---- dw = dz^T x ---------------------------------------------------------------------------------------------------------------
// A tile of TILE columns of either operand by KP rows a step, staged global -> registers -> LDS, so any alignment will do: 16-byte loads at element addresses, PF steps ahead (the ragged
// columns behind a row are the next row's -- read, multiplied and never stored; only the tensor's very last chunk goes element by element).  4 waves as 2 x 2.  (Tiles of 256 with 8
// waves: 100000 x 777 -> 333 in 16 bits 143 us for 113, 50000 x 1537 -> 400 122 for 135.)
constexpr int wgrad_rows(bool h, int tile) { return h || tile == 64 ? 32 : 16; }  // of a step

template <typename T, bool A8, int TILE>
__global__ __launch_bounds__(256, TILE == 128 ? 2 : 4) void linear_wgrad_kernel(WgradArgsL p) {
  constexpr bool H = sizeof(T) == 2;
  constexpr int VE = Vec16<T>::N, NT = 256;
  constexpr int QM = TILE / 32, QN = TILE / 32;         // MFMA tiles of a wave
  constexpr int KP = wgrad_rows(H, TILE);               // rows per step
  constexpr int CH = TILE / VE, NCH = KP * CH / NT;     // 16-byte chunks of a tile row; per thread and operand
  constexpr int PF = TILE == 64 && sizeof(T) == 4 ? 2 : 3;  // (3 would not fit its registers)
  static_assert(KP * CH % NT == 0, "a whole number of chunks for every thread");
  // 16 bits: sub-tiles of [KP rows][64 columns] whose 32-byte column groups are rotated by row / 2 (as the LDS-DMA kernel's); fp32: rows padded by 64 bytes
  constexpr int STRIDE = H ? TILE * 2 : TILE * 4 + 64, OPERAND = KP * STRIDE;
  __shared__ __attribute__((aligned(16))) char smem[4 * OPERAND];  // two stages, one barrier per step
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int li = lane & 15, g = lane >> 4, wm = wave >> 1, wn = wave & 1;
  unsigned logical = xcd_order(blockIdx.x, gridDim.x);
  const int k0 = (int)(logical % p.k_tiles) * TILE; logical /= p.k_tiles;
  const int n0 = (int)(logical % p.n_tiles) * TILE;
  const int split = (int)(logical / p.n_tiles);
  const long long r0 = (long long)split * p.per_split;
  const long long r1 = r0 + p.per_split < p.M ? r0 + p.per_split : p.M;
  const int eb = (p.K + kAct8Block - 1) / kAct8Block;
  const long long end_z = p.M * p.N, end_x = p.M * p.K;
  uint4 rd[PF][NCH], rx[A8 ? 1 : PF][NCH];
  unsigned rc[A8 ? PF : 1][NCH][VE / 4], re[A8 ? PF : 1][NCH];
  auto load = [&](long long r, auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int q = tid + NT * i, col = (q % CH) * VE;
      const long long row = r + q / CH;
      const int ln = p.N - (n0 + col), lk = p.K - (k0 + col);
      rd[S][i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < r1 && ln > 0) {
        const long long at = row * p.N + n0 + col;
        rd[S][i] = at + VE <= end_z ? ld16_any((const T*)p.dz + at) : ld_chunk<T>((const T*)p.dz + at, ln);
      }
      if constexpr (A8) {
#pragma unroll
        for (int j = 0; j < VE / 4; ++j) rc[S][i][j] = 0u;
        re[S][i] = 0u;
        if (row < r1 && lk > 0) {
          const long long at = row * p.K + k0 + col;
          act8_ld_codes<VE>(p.codes + at, at + VE <= end_x ? VE : lk, rc[S][i]);
          re[S][i] = p.exps[row * eb + (k0 + col) / kAct8Block];
        }
      } else {
        rx[S][i] = make_uint4(0u, 0u, 0u, 0u);
        if (row < r1 && lk > 0) {
          const long long at = row * p.K + k0 + col;
          rx[S][i] = at + VE <= end_x ? ld16_any((const T*)p.x + at) : ld_chunk<T>((const T*)p.x + at, lk);
        }
      }
    }
  };
  auto place = [](int q) __attribute__((always_inline)) -> int {  // LDS offset of chunk q of an operand's tile
    const int row = q / CH, c = q % CH;
    if constexpr (H) return (c >> 3) * (KP * 128) + row * 128 + ((((c >> 1) & 3) + (row >> 1)) & 3) * 32 + (c & 1) * 16;
    else return row * STRIDE + c * 16;
  };
  auto put = [&](char* stage, auto set) __attribute__((always_inline)) {
    constexpr int S = decltype(set)::value;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int at = place(tid + NT * i);
      *reinterpret_cast<uint4*>(stage + at) = rd[S][i];
      uint4 v;
      if constexpr (A8 && H) {
        v = act8_decode8_h16(rc[S][i][0], rc[S][i][1], act8_scale(re[S][i]));
      } else if constexpr (A8) {
        float f[4];
        act8_decode4(rc[S][i][0], act8_scale(re[S][i]), f);
        v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      } else {
        v = rx[S][i];
      }
      *reinterpret_cast<uint4*>(stage + OPERAND + at) = v;
    }
  };
  f32x4 acc[QM][QN];
#pragma unroll
  for (int mi = 0; mi < QM; ++mi)
#pragma unroll
    for (int ni = 0; ni < QN; ++ni) acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};
  // 16 bits: a transposed read hands lane li rows {4g .. 4g+3, 16+4g ..} of column 16 c16 + li
  const int frow = 4 * g + (li >> 2), fbase = frow * 128 + (li & 3) * 8, frot = frow >> 1;
  auto frag = [&](const char* operand, int c16) __attribute__((always_inline)) -> uint4 {
    typedef s16x4_t __attribute__((address_space(3))) * lds_ptr;
    const char* at = operand + (c16 >> 2) * (KP * 128) + fbase + (((c16 & 3) + frot) & 3) * 32;
    const uint2 lo = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at)));
    const uint2 hi = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 16 * 128)));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  auto multiply = [&](const char* td, const char* tx) __attribute__((always_inline)) {
    if constexpr (H) {
      uint4 fx[QN];
#pragma unroll
      for (int ni = 0; ni < QN; ++ni) fx[ni] = frag(tx, wn * QN + ni);
#pragma unroll
      for (int mi = 0; mi < QM; ++mi) {
        const uint4 fd = frag(td, wm * QM + mi);
#pragma unroll
        for (int ni = 0; ni < QN; ++ni) acc[mi][ni] = mma16<T>(fd, fx[ni], acc[mi][ni]);
      }
    } else {
#pragma unroll
      for (int s4 = 0; s4 < KP / 4; ++s4) {
        float fd[QM], fx[QN];
#pragma unroll
        for (int mi = 0; mi < QM; ++mi) fd[mi] = *reinterpret_cast<const float*>(td + (s4 * 4 + g) * STRIDE + ((wm * QM + mi) * 16 + li) * 4);
#pragma unroll
        for (int ni = 0; ni < QN; ++ni) fx[ni] = *reinterpret_cast<const float*>(tx + (s4 * 4 + g) * STRIDE + ((wn * QN + ni) * 16 + li) * 4);
#pragma unroll
        for (int mi = 0; mi < QM; ++mi)
#pragma unroll
          for (int ni = 0; ni < QN; ++ni) acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x4f32(fd[mi], fx[ni], acc[mi][ni], 0, 0, 0);
      }
    }
  };
  int stage = 0;
  auto step = [&](long long r, auto set) __attribute__((always_inline)) {
    char* at = smem + stage * (2 * OPERAND);
    stage ^= 1;
    put(at, set);
    __syncthreads();
    load(r + PF * KP, set);
    multiply(at, at + OPERAND);
  };
  load(r0, std::integral_constant<int, 0>());
  load(r0 + KP, std::integral_constant<int, 1>());
  if constexpr (PF == 3) load(r0 + 2 * KP, std::integral_constant<int, PF - 1>());
  for (long long r = r0; r < r1; r += PF * KP) {
    step(r, std::integral_constant<int, 0>());
    if (r + KP < r1) step(r + KP, std::integral_constant<int, 1>());
    if constexpr (PF == 3) {
      if (r + 2 * KP < r1) step(r + 2 * KP, std::integral_constant<int, PF - 1>());
    }
  }
  // lane: rows n = n0 + 16 (wm QM + mi) + 4 g + r, column k = k0 + 16 (wn QN + ni) + li
  float* out = p.part + (long long)split * p.N * p.K;
#pragma unroll
  for (int mi = 0; mi < QM; ++mi)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + (wm * QM + mi) * 16 + 4 * g + r;
      if (n >= p.N) continue;
#pragma unroll
      for (int ni = 0; ni < QN; ++ni) {
        const int k = k0 + (wn * QN + ni) * 16 + li;
        if (k < p.K) out[(long long)n * p.K + k] = acc[mi][ni][r];
      }
    }
}

// dw from the splits' partial sums, in a fixed order: GROUPS groups of 64 16-byte columns a block take the splits in turn, 4 loads in flight a thread, and are joined in LDS.  One group
// for few splits, 16 for many (one thread a value walking 512 splits of 64 x 64 took 100 us; 16 groups for the 4 splits of 2048 x 2048 left twelve of them idle: 38 us, not 16).
template <int GROUPS>
__global__ __launch_bounds__(64 * GROUPS) void linear_wgrad_reduce_kernel(const float* __restrict__ part, long long count, int splits, float* __restrict__ dw) {
  __shared__ float4 red[GROUPS][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const long long i = ((long long)blockIdx.x * 64 + tx) * 4;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  const bool whole = i + 4 <= count && (count & 3) == 0;
  if (whole) {
    int s = ty;
    for (; s + 3 * GROUPS < splits; s += 4 * GROUPS) {
      float4 v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = *reinterpret_cast<const float4*>(part + (long long)(s + GROUPS * u) * count + i);
#pragma unroll
      for (int u = 0; u < 4; ++u) { a.x += v[u].x; a.y += v[u].y; a.z += v[u].z; a.w += v[u].w; }
    }
    for (; s < splits; s += GROUPS) {
      const float4 v = *reinterpret_cast<const float4*>(part + (long long)s * count + i);
      a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
    }
  } else if (i < count) {  // dw of an odd number of values: its rows of partial sums start at any element
    const int left = count - i < 4 ? (int)(count - i) : 4;
    for (int s = ty; s < splits; s += GROUPS) {
      float v[4];
      ld_f32<4>(part + (long long)s * count + i, left, v);
      a.x += v[0]; a.y += v[1]; a.z += v[2]; a.w += v[3];
    }
  }
  if constexpr (GROUPS > 1) {
    red[ty][tx] = a;
    __syncthreads();
    for (int o = GROUPS / 2; o > 0; o >>= 1) {
      if (ty < o) {
        const float4 v = red[ty + o][tx];
        float4 w = red[ty][tx];
        w.x += v.x; w.y += v.y; w.z += v.z; w.w += v.w;
        red[ty][tx] = w;
      }
      __syncthreads();
    }
    if (ty > 0) return;
    a = red[0][tx];
  }
  if (whole) {
    *reinterpret_cast<float4*>(dw + i) = a;
  } else {
    const float w[4] = {a.x, a.y, a.z, a.w};
    for (int e = 0; e < 4 && i + e < count; ++e) dw[i + e] = w[e];
  }
}

__global__ __launch_bounds__(256) void rows_zero_kernel(float* p, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0.f;
}

static int linear_bad(const char* what, int64_t rows, int in, int out, int dtype) {
  SH_REQUIRE(dtype == SH_F32 || dtype == SH_BF16, "%s: dtype %d", what, dtype);
  SH_REQUIRE(rows >= 0 && rows < (1ll << 31) && in >= 1 && out >= 1 && in <= (1 << 20) && out <= (1 << 20), "%s: rows=%lld in=%d out=%d", what, (long long)rows, in, out);
  SH_REQUIRE((int64_t)((rows + 127) / 128) * ((in > out ? in : out) / 128 + 1) < (1ll << 31), "%s: rows=%lld in=%d out=%d: too many tiles", what,
             (long long)rows, in, out);
  return 0;
}

// What 32 elements of the reduction of a register-staged tile take (us) with `on_cu` blocks on a CU, measured with one / two / four (16384 x 1023 -> 1023, weight gradient; the product
// agrees): 64 x 64 0.37 / 0.39 / 0.66 in 16 bits and 1.0 / 1.5 / 2.5 in fp32, 128 x 128 0.60 / 0.69 and 2.7 / 4.5.
static double staged_us(bool h, int tile, int on_cu) {
  if (tile == 64) return h ? (on_cu <= 2 ? 0.36 + 0.015 * on_cu : 0.165 * on_cu) : 0.45 + 0.52 * on_cu;
  return h ? 0.51 + 0.09 * on_cu : 0.92 + 1.78 * on_cu;
}
static int staged_on_cu(int tile) { return tile == 64 ? 4 : 2; }  // blocks that fit a CU

// The tile whose rounds over the 256 CUs cost least.  A k-step (128 bytes) of a bm x bn tile brings bm + bn rows into LDS, at the 15 bytes per clock and CU that these kernels reach, and multiplies at 4096
// (fp32: 256) flops per clock, whichever takes longer, and pays its barrier: 5001 x 1000 -> 333 in 16 bits is all operand traffic (64 x 64: 2 rounds of 128 rows, 15 us; 128 x 64:
// one of 192), 2048 x 512 -> 2048 in fp32 all arithmetic.
template <bool BT> static int dma_launch(LinearArgs p, int dtype, hipStream_t s, const char* what) {
  auto cost = [&](int64_t bm, int64_t bn) {
    const int64_t rounds = ((int64_t)ceil_div(p.M, (int)bm) * ceil_div(p.N, (int)bn) + 255) / 256;
    const int64_t fetch = (bm + bn) * 128 / 15, mul = bm * bn * (dtype == SH_F32 ? 64 : 128) / (dtype == SH_F32 ? 256 : 4096);
    return rounds * ((fetch > mul ? fetch : mul) + 300);
  };
  const int64_t c64 = cost(64, 64), c96 = cost(128, 64), c128 = cost(128, 128);
  const int bm = c96 < c64 || c128 < c64 ? 128 : 64, bn = bm == 128 && c128 <= c96 ? 128 : 64;
  p.n_tiles = (unsigned)ceil_div(p.N, bn);
  const unsigned grid = (unsigned)ceil_div(p.M, bm) * p.n_tiles;
#define SH_DMA(T)                                                                  \
  if (bn == 128) linear_dma_kernel<T, 4, 4, BT><<<grid, 256, 0, s>>>(p);           \
  else if (bm == 128) linear_dma_kernel<T, 4, 2, BT><<<grid, 256, 0, s>>>(p);      \
  else linear_dma_kernel<T, 2, 2, BT><<<grid, 256, 0, s>>>(p);
  if (dtype == SH_F32) { SH_DMA(float) }
  else { SH_DMA(bf16_t) }
#undef SH_DMA
  return check_launch(what);
}

// A launch's threads are counted in 32 bits: more than 2^23 tiles (of 64 x 64) go in several launches, each over a range of whole tiles' rows.
template <typename F> static int by_row_ranges(const LinearArgs& p, int dtype, F&& launch) {
  const int64_t tiles = (p.N + 63) / 64, most = ((1ll << 23) / tiles) * 64, eb = dtype == SH_F32 ? 4 : 2;
  for (int64_t r = 0; r < p.M; r += most) {
    LinearArgs q = p;
    q.M = p.M - r < most ? p.M - r : most;
    q.a = (const char*)p.a + r * p.K * eb;
    q.out = (char*)p.out + r * p.N * eb;
    if (p.pre != nullptr) q.pre = (char*)p.pre + r * p.N * eb;
    if (p.residual != nullptr) q.residual = (const char*)p.residual + r * p.N * eb;
    if (launch(q)) return 1;
  }
  return 0;
}

// Which kernel: few rows -> the skinny one (rows <= 64 and so little work that tiles would leave most CUs idle); many -> rows in registers or the 256-wide tiles, as their rules say; whole
// chunks -> the DMA tiles; anything else staged through registers.
static int linear_kernel_of(const LinearArgs& p, int dtype) {
  if (p.M <= 64 && ceil_div(p.N, 64) < 256) return SH_LIN_SKINNY;
  if (linear_rows_takes(p, dtype)) return SH_LIN_ROWS;
  if (linear256_takes(p, dtype)) return SH_LIN_TILES256;
  const int ve = dtype == SH_F32 ? 4 : 8;
  return p.K % ve == 0 && p.ldb % ve == 0 && !(((size_t)p.a | (size_t)p.b) & 15) ? SH_LIN_DMA : SH_LIN_STAGED;
}
static int gemm_launch(const LinearArgs& base, bool b_padded, void* workspace, int dtype, hipStream_t s, const char* what) {
  LinearArgs p = base;
  const int kernel = linear_kernel_of(p, dtype);
  if (kernel == SH_LIN_SKINNY) {
    const int mt = p.M <= 16 ? 1 : p.M <= 32 ? 2 : 4;
    const dim3 grid(ceil_div(p.N, 16), 1);
#define SH_SKINNY(T, MT) linear_skinny_kernel<T, MT><<<grid, 512, 0, s>>>(p)
    if (dtype == SH_F32) {
      if (mt == 1) SH_SKINNY(float, 1);
      else if (mt == 2) SH_SKINNY(float, 2);
      else SH_SKINNY(float, 4);
    } else {
      if (mt == 1) SH_SKINNY(bf16_t, 1);
      else if (mt == 2) SH_SKINNY(bf16_t, 2);
      else SH_SKINNY(bf16_t, 4);
    }
#undef SH_SKINNY
    return check_launch(what);
  }
  if (kernel == SH_LIN_ROWS) return linear_rows_launch(p, b_padded, workspace, s, what);
  if (kernel == SH_LIN_TILES256) return linear256_launch(p, s, what);
  if (kernel == SH_LIN_DMA) return dma_launch<false>(p, dtype, s, what);
  // the tile whose rounds over the CUs cost least, each with its ends (1.2 and 4 us): 128 for 100000 x 777 -> 333 (16 bits 113 us, 64: 173; fp32 532 and 546), 64 for 400000 x 65 -> 63 (43 and
  // 53; fp32 63 and 113) and, for its last round, 5001 x 2047 -> 2047 in fp32 (382 and 515)
  auto cost = [&](int t) {
    const int64_t blocks = (int64_t)ceil_div(p.M, t) * ceil_div(p.N, t), round = 256 * staged_on_cu(t), full = blocks / round, rest = blocks % round;
    const bool h = dtype != SH_F32;
    const double steps = (p.K + 31) / 32;
    return full * staged_us(h, t, staged_on_cu(t)) * steps + (rest ? staged_us(h, t, (int)((rest + 255) / 256)) * steps : 0.) + (full + (rest > 0)) * (t == 64 ? 1.2 : 4.);
  };
  const int tile = cost(128) < cost(64) ? 128 : 64;
  p.n_tiles = (unsigned)ceil_div(p.N, tile);
  const unsigned grid = (unsigned)ceil_div(p.M, tile) * p.n_tiles;
  if (tile == 128) {
    if (dtype == SH_F32) linear_gemm_kernel<float, 128><<<grid, 256, 0, s>>>(p);
    else linear_gemm_kernel<bf16_t, 128><<<grid, 256, 0, s>>>(p);
  } else {
    if (dtype == SH_F32) linear_gemm_kernel<float, 64><<<grid, 256, 0, s>>>(p);
    else linear_gemm_kernel<bf16_t, 64><<<grid, 256, 0, s>>>(p);
  }
  return check_launch(what);
}

static int act_bwd_tx(int cols, int dtype) {
  const int nvec = (cols + (dtype == SH_F32 ? 4 : 8) - 1) / (dtype == SH_F32 ? 4 : 8);
  return nvec <= 8 ? 8 : nvec <= 16 ? 16 : nvec <= 32 ? 32 : 64;
}
static void act_bwd_plan(int64_t rows, int cols, int dtype, int* gx, int* gy, int64_t* per) {
  const int tx = act_bwd_tx(cols, dtype), ty = 256 / tx, ve = dtype == SH_F32 ? 4 : 8;
  *gx = ceil_div(cols, tx * ve);
  int64_t want = (2048 + *gx - 1) / *gx, most = (rows + ty - 1) / ty;
  if (most <= 8) want = 1;  // few rows: one block a strip of columns, whose sums need no fold (a launch and a workspace less)
  if (want > most) want = most;
  if (want < 1) want = 1;
  *per = ((rows + want - 1) / want + ty - 1) / ty * ty;
  if (*per < 1) *per = ty;
  *gy = (int)((rows + *per - 1) / *per);
  if (*gy < 1) *gy = 1;
}

// Tile and splits of the rows: the pair whose estimate is least; the join of the splits reads and writes their sums at 4 TB/s and is a launch more.  It takes 64 without a split for 1000 x
// 1000 -> 1000 in 16 bits (13.7 us; in four 20.8), 64 in 8 splits for 5001 x 1000 -> 333 (21; 128 in 20: 26), 128 in 24 for 100000 x 777 -> 333 (109; 64: 180), and 64 in 4 for 2048 x 2048
// -> 512 in fp32 (53; 128 in 8: 56).
static int linear_wgrad_plan(int64_t rows, int in, int out, int dtype, int* splits, int64_t* per) {
  const bool h = dtype != SH_F32;
  double best = 0.;
  int best_tile = 0;
  for (int tile = 64; tile <= 128; tile *= 2) {
    const int kp = wgrad_rows(h, tile), most = staged_on_cu(tile);
    const int64_t tiles = (int64_t)ceil_div(in, tile) * ceil_div(out, tile), steps = rows > 0 ? (rows + kp - 1) / kp : 1;
    for (int on_cu = 0; on_cu <= most; ++on_cu) {  // as many splits as put on_cu blocks on every CU, of at least 4 steps each; 0: no split
      int64_t sk = on_cu == 0 ? 1 : 256 * on_cu / tiles;
      if (sk > steps / 4) sk = steps / 4;
      if (sk < 1) sk = 1;
      const int64_t each = (steps + sk - 1) / sk, full = (sk * tiles + 255) / 256, rounds = (full + most - 1) / most;
      const double t = staged_us(h, tile, (int)(full < most ? full : most)) * kp / 32;
      const double cost = (double)(rounds * each) * t + (sk > 1 ? 5. + (double)sk * in * out * 2e-6 : 0.);
      if (best_tile == 0 || cost < best) {
        best = cost;
        best_tile = tile;
        *per = each * kp;
        *splits = (int)((steps + each - 1) / each);
      }
    }
  }
  return best_tile;
}

}  // namespace sh

using namespace sh;

extern "C" {

int simhand_test_linear_kernel(int64_t rows, int in_dim, int out_dim, int dtype, int aligned, int residual) {
  const void* at = (const void*)(size_t)(aligned ? 16 : 2);
  const LinearArgs p = {at, at, nullptr, nullptr, nullptr, residual ? at : nullptr, rows, out_dim, in_dim, in_dim, SH_ACT_NONE, 0};
  return linear_kernel_of(p, dtype);
}

size_t simhand_linear_fwd_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype, int aligned) {
  if (rows < 1 || in_dim < 1 || out_dim < 1 || dtype != SH_BF16) return 0;
  // the padded copy of w, wherever the rows-in-registers kernel may be given rows that are no whole 16-byte chunks, by length or by address
  const void* at = (const void*)(size_t)(aligned ? 16 : 2);
  LinearArgs p = {at, at, nullptr, nullptr, nullptr, at, rows, out_dim, in_dim, in_dim, SH_ACT_NONE, 0};
  return linear_rows_fits(p, dtype) ? linear_rows_workspace_bytes(p) : 0;
}

int simhand_linear_fwd(const void* x, const void* w, const float* bias, int act, const void* residual, void* y, void* pre, int64_t rows, int in_dim,
                       int out_dim, int dtype, void* workspace, size_t workspace_bytes, sh_stream_t stream) {
  if (linear_bad("linear_fwd", rows, in_dim, out_dim, dtype)) return 1;
  SH_REQUIRE(act >= SH_ACT_NONE && act <= SH_ACT_SILU, "linear_fwd: act %d", act);
  if (rows == 0) return 0;
  SH_REQUIRE(x && w && y, "linear_fwd: NULL argument");
  const size_t need = simhand_linear_fwd_workspace_bytes(rows, in_dim, out_dim, dtype, !(((size_t)x | (size_t)w | (size_t)residual) & 15));
  SH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && !((size_t)workspace & 15)), "linear_fwd: workspace too small or not at a 16-byte address");
  hipStream_t s = (hipStream_t)stream;
  const double eb = dtype == SH_F32 ? 4 : 2;
  ProfScope ps(SH_PROF_MISC, s, 2.0 * rows * in_dim * out_dim, eb * ((double)rows * in_dim + (double)in_dim * out_dim + (double)rows * out_dim));
  LinearArgs p = {x, w, y, pre, bias, residual, rows, out_dim, in_dim, in_dim, act, 0};
  return by_row_ranges(p, dtype, [&](const LinearArgs& q) { return gemm_launch(q, false, workspace, dtype, s, "linear_fwd"); });
}

size_t simhand_linear_act_bwd_workspace_bytes(int64_t rows, int cols, int dtype) {
  if (rows < 0 || cols < 1) return 0;
  int gx, gy;
  int64_t per;
  act_bwd_plan(rows, cols, dtype, &gx, &gy, &per);
  return gy > 1 ? (size_t)gy * cols * sizeof(float) : 0;
}

int simhand_linear_act_bwd(const void* dy, const void* pre, int act, void* dz, float* db, int64_t rows, int cols, int dtype, void* workspace,
                           size_t workspace_bytes, sh_stream_t stream) {
  if (linear_bad("linear_act_bwd", rows, 1, cols, dtype)) return 1;
  SH_REQUIRE(act >= SH_ACT_NONE && act <= SH_ACT_SILU, "linear_act_bwd: act %d", act);
  SH_REQUIRE(db && (rows == 0 || dy), "linear_act_bwd: NULL argument");
  SH_REQUIRE(rows == 0 || act == SH_ACT_NONE || (pre && dz), "linear_act_bwd: an activation needs pre and dz");
  const size_t need = simhand_linear_act_bwd_workspace_bytes(rows, cols, dtype);
  SH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "linear_act_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  ProfScope ps(SH_PROF_MISC, s, 0, (dtype == SH_F32 ? 4.0 : 2.0) * rows * cols * (act == SH_ACT_NONE ? 1 : 3));
  int gx, gy;
  int64_t per;
  act_bwd_plan(rows, cols, dtype, &gx, &gy, &per);
  float* part = gy == 1 ? db : (float*)workspace;
  const dim3 grid(gx, gy);
#define SH_ACT(T, TX) linear_act_bwd_kernel<T, TX><<<grid, 256, 0, s>>>((const T*)dy, (const T*)pre, act, (T*)dz, part, rows, cols, per)
#define SH_ACT_TX(T)                       \
  switch (act_bwd_tx(cols, dtype)) {       \
    case 8: SH_ACT(T, 8); break;           \
    case 16: SH_ACT(T, 16); break;         \
    case 32: SH_ACT(T, 32); break;         \
    default: SH_ACT(T, 64); break;         \
  }
  if (dtype == SH_F32) { SH_ACT_TX(float) }
  else { SH_ACT_TX(bf16_t) }
#undef SH_ACT_TX
#undef SH_ACT
  if (check_launch("linear_act_bwd")) return 1;
  if (gy == 1) return 0;
  return fold_columns(part, gy, cols, db, s);
}

// dx = dz w with w as it is, unless the product is large enough for the kernels for many rows (whose transposed copy of w is then small change) or w's rows are no whole chunks
static bool dgrad_direct(int64_t rows, int in_dim, int out_dim, int dtype, bool aligned) {
  const int ve = dtype == SH_F32 ? 4 : 8;
  if (in_dim % ve || out_dim % ve || !aligned) return false;
  const void* at = (const void*)(size_t)16;
  LinearArgs wide = {at, at, nullptr, nullptr, nullptr, nullptr, rows, in_dim, out_dim, (out_dim + 7) / 8 * 8, SH_ACT_NONE, 0};
  return !linear256_takes(wide, dtype) && !linear_rows_takes(wide, dtype);
}
size_t simhand_linear_dgrad_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype, int aligned) {
  if (rows < 1 || in_dim < 1 || out_dim < 1 || dgrad_direct(rows, in_dim, out_dim, dtype, aligned != 0)) return 0;
  return (size_t)in_dim * ((out_dim + 7) / 8 * 8) * (dtype == SH_F32 ? 4 : 2);
}
int simhand_linear_dgrad(const void* dz, const void* w, void* dx, int64_t rows, int in_dim, int out_dim, int dtype, void* workspace,
                         size_t workspace_bytes, sh_stream_t stream) {
  if (linear_bad("linear_dgrad", rows, in_dim, out_dim, dtype)) return 1;
  if (rows == 0) return 0;
  SH_REQUIRE(dz && w && dx, "linear_dgrad: NULL argument");
  const bool direct = dgrad_direct(rows, in_dim, out_dim, dtype, !(((size_t)dz | (size_t)w) & 15));
  SH_REQUIRE(direct || (workspace && workspace_bytes >= simhand_linear_dgrad_workspace_bytes(rows, in_dim, out_dim, dtype, 0) && !((size_t)workspace & 15)),
             "linear_dgrad: workspace too small or not at a 16-byte address");
  hipStream_t s = (hipStream_t)stream;
  const double eb = dtype == SH_F32 ? 4 : 2;
  ProfScope ps(SH_PROF_MISC, s, 2.0 * rows * in_dim * out_dim, eb * ((double)rows * in_dim + (double)in_dim * out_dim + (double)rows * out_dim));
  if (direct) {
    LinearArgs p = {dz, w, dx, nullptr, nullptr, nullptr, rows, in_dim, out_dim, in_dim, SH_ACT_NONE, 0};
    return by_row_ranges(p, dtype, [&](const LinearArgs& q) { return dma_launch<true>(q, dtype, s, "linear_dgrad"); });
  }
  const int ldt = (out_dim + 7) / 8 * 8;
  LinearArgs wide = {dz, workspace, dx, nullptr, nullptr, nullptr, rows, in_dim, out_dim, ldt, SH_ACT_NONE, 0};
  const dim3 tg(ceil_div(in_dim, 32), ceil_div(ldt, 32));
  if (dtype == SH_F32) linear_transpose_kernel<float><<<tg, 256, 0, s>>>((const float*)w, (float*)workspace, out_dim, in_dim, ldt);
  else linear_transpose_kernel<bf16_t><<<tg, 256, 0, s>>>((const bf16_t*)w, (bf16_t*)workspace, out_dim, in_dim, ldt);
  if (check_launch("linear_dgrad")) return 1;
  return by_row_ranges(wide, dtype, [&](const LinearArgs& q) { return gemm_launch(q, true, nullptr, dtype, s, "linear_dgrad"); });
}

size_t simhand_linear_wgrad_workspace_bytes(int64_t rows, int in_dim, int out_dim, int dtype) {
  if (rows < 0 || in_dim < 1 || out_dim < 1) return 0;
  // the call's alignment decides between two kernels (below): enough for either
  int splits, wide = 1;
  int64_t per;
  linear_wgrad_plan(rows, in_dim, out_dim, dtype, &splits, &per);
  if (linear_wgrad256_takes(nullptr, nullptr, nullptr, nullptr, rows, in_dim, out_dim, dtype)) linear_wgrad256_plan(rows, in_dim, out_dim, &wide, &per);
  if (wide > splits) splits = wide;
  return splits > 1 ? (size_t)splits * in_dim * out_dim * sizeof(float) : 0;
}

int simhand_linear_wgrad(const void* dz, const void* x, const uint8_t* x_codes, const uint8_t* x_exps, float* dw, int64_t rows, int in_dim, int out_dim,
                         int dtype, void* workspace, size_t workspace_bytes, sh_stream_t stream) {
  if (linear_bad("linear_wgrad", rows, in_dim, out_dim, dtype)) return 1;
  const bool a8 = x_codes != nullptr;
  SH_REQUIRE(!a8 || (x_exps && !x), "linear_wgrad: pass either x or its codes and exponents");
  SH_REQUIRE(dw && (rows == 0 || (dz && (x || a8))), "linear_wgrad: NULL argument");
  const size_t need = simhand_linear_wgrad_workspace_bytes(rows, in_dim, out_dim, dtype);
  SH_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && !((size_t)workspace & 15)), "linear_wgrad: workspace too small or not at a 16-byte address");
  hipStream_t s = (hipStream_t)stream;
  const double eb = dtype == SH_F32 ? 4 : 2;
  ProfScope ps(SH_PROF_MISC, s, 2.0 * rows * in_dim * out_dim, eb * (double)rows * out_dim + (a8 ? 1.03125 : eb) * rows * in_dim + 4.0 * in_dim * out_dim);
  const long long count = (long long)in_dim * out_dim;
  if (rows == 0) {
    rows_zero_kernel<<<(unsigned)((count + 255) / 256), 256, 0, s>>>(dw, count);
    return check_launch("linear_wgrad");
  }
  int splits;
  int64_t per;
  const bool wide = linear_wgrad256_takes(dz, x, x_codes, x_exps, rows, in_dim, out_dim, dtype);
  int tile = 256;  // (the wide kernel's own)
  if (wide) linear_wgrad256_plan(rows, in_dim, out_dim, &splits, &per);
  else tile = linear_wgrad_plan(rows, in_dim, out_dim, dtype, &splits, &per);
  WgradArgsL p = {dz, x, x_codes, x_exps, splits > 1 ? (float*)workspace : dw, rows, per, out_dim, in_dim, (unsigned)ceil_div(out_dim, tile),
                  (unsigned)ceil_div(in_dim, tile)};
  if (wide) {
    if (linear_wgrad256_launch(p, splits, s)) return 1;
  } else {
    const unsigned grid = p.n_tiles * p.k_tiles * (unsigned)splits;
#define SH_WGRAD(T, A8)                                                               \
  if (tile == 128) linear_wgrad_kernel<T, A8, 128><<<grid, 256, 0, s>>>(p);           \
  else linear_wgrad_kernel<T, A8, 64><<<grid, 256, 0, s>>>(p)
    if (dtype == SH_F32) {
      if (a8) { SH_WGRAD(float, true); }
      else { SH_WGRAD(float, false); }
    } else {
      if (a8) { SH_WGRAD(bf16_t, true); }
      else { SH_WGRAD(bf16_t, false); }
    }
#undef SH_WGRAD
    if (check_launch("linear_wgrad")) return 1;
  }
  if (splits > 1) {
    const unsigned blocks = (unsigned)((count + 255) / 256);
    if (splits <= 16) linear_wgrad_reduce_kernel<1><<<blocks, 64, 0, s>>>((const float*)workspace, count, splits, dw);
    else linear_wgrad_reduce_kernel<16><<<blocks, 1024, 0, s>>>((const float*)workspace, count, splits, dw);
    return check_launch("linear_wgrad_reduce");
  }
  return 0;
}

}  // extern "C"
