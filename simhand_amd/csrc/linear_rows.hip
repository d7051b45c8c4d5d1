// out [M][N] = a [M][K] b[N][ldb]^T of 16-bit operands for many rows and a short K (at most 512): the rows stay in registers.
//
// What bounds the 256 x 256 kernel at these sizes is operand traffic: every tile fetches both its operands, 1.6 GB for 100352 x 512 -> 2048, on top of what the epilogue moves -- and the
// epilogue's streams drive the operands out of the 4 MB L2s, behind which 8 TB/s are to be had (30 from the L2s themselves).  Here a wave holds 32 rows of a for the WHOLE of K as MFMA operands (128 registers at K = 512), eight waves 256 rows,
// and only b streams through LDS -- half the traffic.  The work is a list of units (256 rows x 64 columns), dealt out evenly over the CUs in contiguous ranges; b's steps (64 columns x
// 128 of K, 16 KB, four stages, fetched three steps ahead by LDS-DMA) form one sequence across the units, and the residual's tile of the next unit arrives by LDS-DMA as well, so
// nothing in the loop waits for memory but the counted waits below; the stores drain behind them.
// Measured, bf16: 100352 x 512 -> 2048 with a residual 255 us (0.93 GB; HBM moves 1.12 at 4.5 TB/s, the matrix cores are 39 % busy: inside a block they wait while it stores and fetches
// rows), 401408 x 256 -> 1024 282 (1.33 GB at 4.8 TB/s, of which 1.09 are written where 0.82 are due; matrix cores 34 %).  Between runs and beside other work both move by 10 %.
// RAG: rows of a (any K) and of out (any N) at element alignment -- a goes straight to registers, so only b, which is copied into padded rows first, needs whole chunks; the residual is then read in the epilogue, and the waits are not counted past stores that may be missing.
#include "linear.h"

namespace sh {

__device__ uint4 g_lrows_zero[8];  // read-only zeros

constexpr int kRowsMaxN = 4096;  // the bias waits in LDS

template <int KS2, bool RES, bool PRE, bool RAG>
__global__ __launch_bounds__(512, 1) void linear_rows_kernel(LinearArgs p, unsigned units, unsigned per_cu) {
  typedef bf16_t T;
  constexpr int S = 4, D = 3, W_BYTES = 16384, RM = 2, ROWS = 128 * RM, R_BYTES = 16384 * RM, R0 = S * W_BYTES, BIAS0 = R0 + (RES && !RAG ? 2 * R_BYTES : 0);
  constexpr int E_R = RES && !RAG ? 2 * RM : 0, E_ST = (PRE ? 4 : 2) * RM;  // vector-memory operations of a unit: residual DMAs, stores of whole rows
  __shared__ __attribute__((aligned(16))) char smem[BIAS0 + kRowsMaxN * 4];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
  auto dma16 = [](const void* src, unsigned lds_addr) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(src));
  };
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, g = lane >> 4, slot = lane & 7;
  const unsigned cu = xcd_order(blockIdx.x, gridDim.x);
  const unsigned u0 = cu * per_cu, u1 = u0 + per_cu < units ? u0 + per_cu : units;
  if (u0 >= u1) return;
  const unsigned nt = p.n_tiles;  // units per row tile
  float* bias = reinterpret_cast<float*>(smem + BIAS0);
  for (int n = tid; n < (int)nt * 64; n += 512) bias[n] = p.bias != nullptr && n < p.N ? p.bias[n] : 0.f;
  __syncthreads();

  // b: a wave's two DMA instructions of a step fill rows 8 wave .. + 7 (columns of out) of the step's two 64-k halves; slot s of a row holds chunk s ^ key(row)
  auto key_b = [](int row) __attribute__((always_inline)) -> int { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); };
  const int brow = wave * 8 + (lane >> 3), bk = (slot ^ key_b(brow)) * 8;
  const char* zero = reinterpret_cast<const char*>(g_lrows_zero) + slot * 16;
  unsigned wu = u0, wn_ = u0 % nt, w_stage = 0;  // walker over b's steps: unit, its column tile, stage, k
  int wk = 0;
  auto b_row = [&](unsigned tile) __attribute__((always_inline)) {
    const int n = (int)tile * 64 + brow;
    return reinterpret_cast<const char*>((const T*)p.b + (long long)(!RAG || n < p.N ? n : p.N - 1) * p.ldb + bk);
  };
  const char* wrow = b_row(wn_);
  auto dma_w = [&]() __attribute__((always_inline)) {
    const unsigned dst = lds0 + w_stage * W_BYTES + wave * 1024;
    dma16(wu < u1 && wk + bk < p.ldb ? wrow + wk * 2 : zero, dst);
    dma16(wu < u1 && wk + 64 + bk < p.ldb ? wrow + wk * 2 + 128 : zero, dst + 8192);
    w_stage = (w_stage + 1) & (S - 1);
    wk += 128;
    if (wk >= KS2 * 128) {
      wk = 0;
      ++wu;
      wn_ = wn_ + 1 == nt ? 0 : wn_ + 1;
      wrow = b_row(wn_);
    }
  };
  // the residual's tile of unit u: each wave fetches its own 32 rows (8 an instruction); slot s of a row holds chunk s ^ (row & 7)
  auto dma_r = [&](unsigned u) __attribute__((always_inline)) {
    const unsigned uu = u < u1 ? u : u1 - 1;
    const long long m0 = (long long)(uu / nt) * ROWS + wave * (16 * RM) + (lane >> 3);
    const long long col = (long long)(uu % nt) * 64 + (slot ^ (lane >> 3)) * 8;
    const unsigned dst = lds0 + R0 + (u & 1) * R_BYTES + wave * (2048 * RM);
#pragma unroll
    for (int i = 0; i < 2 * RM; ++i) {
      const long long m = m0 + 8 * i < p.M ? m0 + 8 * i : p.M - 1;
      // read once: past the caches where K is long (100352 x 512 -> 2048: 258 -> 246 us, 200704 x 512 -> 1024 263 -> 256; 401408 x 256 -> 1024 382 -> 388)
      if constexpr (KS2 >= 3) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"s"(dst + i * 1024), "v"((const T*)p.residual + m * p.N + col));
      else dma16((const T*)p.residual + m * p.N + col, dst + i * 1024);
    }
  };

  if constexpr (RES && !RAG) dma_r(u0);
#pragma unroll
  for (int i = 0; i < D; ++i) dma_w();
  const int rowb = lin_col(0, li);
  const int fb0 = rowb * 128 + ((g ^ key_b(rowb)) * 16);
  auto read_b = [&](unsigned stage, int phase, uint4 (&fb)[4]) __attribute__((always_inline)) {  // phase = 2 (64-k half) + (32-k half of it)
    const char* at = smem + stage * W_BYTES + (phase >> 1) * 8192 + ((phase & 1) ? fb0 ^ 64 : fb0);
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) fb[ni] = *reinterpret_cast<const uint4*>(at + (lin_col(ni, 0) - lin_col(0, 0)) * 128);
  };
  uint4 fb[2][4];
  // step 0 has landed (steps 1 .. D - 1 may be in flight)
  asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(2 * (D - 1)) : "memory");
  read_b(0, 0, fb[0]);
  unsigned stage = 0, m_have = 0xffffffffu;
  uint4 a[RM][KS2 * 2][2];
  for (unsigned u = u0; u < u1; ++u) {
    const unsigned mt = u / nt;
    const long long mrow = (long long)mt * ROWS + wave * (16 * RM) + li;
    if (mt != m_have) {  // (its loads' wait drains the DMA queue: once per 256 rows)
      m_have = mt;
#pragma unroll
      for (int mi = 0; mi < RM; ++mi) {
        const long long m = mrow + 16 * mi < p.M ? mrow + 16 * mi : p.M - 1;
        const T* row = (const T*)p.a + m * p.K;
#pragma unroll
        for (int ks = 0; ks < KS2 * 2; ++ks)
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            const int k = ks * 64 + kk * 32 + g * 8;
            if constexpr (!RAG) {
              a[mi][ks][kk] = k < p.K ? ld16_any(row + k) : make_uint4(0u, 0u, 0u, 0u);
            } else {  // the ragged last chunk: the row's last 8 elements, moved into place below -- no branch between the loads
              a[mi][ks][kk] = ld16_any(row + (ks < KS2 * 2 - 2 || k + 8 <= p.K ? k : p.K - 8));  // (K > 128 (KS2 - 1): only the last two can end it)
            }
          }
      }
      if constexpr (RAG) {
#pragma unroll
        for (int mi = 0; mi < RM; ++mi)
#pragma unroll
          for (int ks = KS2 * 2 - 2; ks < KS2 * 2; ++ks)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) a[mi][ks][kk] = move_down<T>(a[mi][ks][kk], ks * 64 + kk * 32 + g * 8 + 8 - p.K);
      }
    }
    const bool full = !RAG && (long long)mt * ROWS + (wave + 1) * (16 * RM) <= p.M;
    const bool steady = full && u >= u0 + 2;  // the two units before this one made all their stores
    f32x4 acc[RM][4];
#pragma unroll
    for (int mi = 0; mi < RM; ++mi)
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < KS2; ++j) {
#pragma unroll
      for (int ph = 0; ph < 4; ++ph) {
        if (ph == 2) {
          // In mid-step: step s + 1 has landed, everybody is past step s - 1.  Behind the DMAs of step s + 1 (issued two steps ago) stand those of step s + 2, and of the two steps
          // in between: the residual's, where a unit began, and a unit's stores, where it ended.
          constexpr int kWait[5] = {0, 2 + 2 * E_R + 2 * E_ST, 2 + E_R + E_ST, 0, 0};
          constexpr int X = KS2 == 1 ? kWait[1] : KS2 == 2 ? kWait[2] : 0;
          if constexpr (KS2 <= 2) {
            if (steady) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(X) : "memory");
            else asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
          } else {
            // j = 0: the stores; j = 1: stores and residual; j = 2: the residual; later: neither
            if (steady && j == 0) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 + E_ST) : "memory");
            else if (steady && j == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 + E_R + E_ST) : "memory");
            else if (j == 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 + E_R) : "memory");
            else asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
          }
          dma_w();
          if constexpr (RES && !RAG) {
            if (j == 0) dma_r(u + 1);
          }
        }
        if (ph < 3) read_b(stage, ph + 1, fb[(ph + 1) & 1]);
        else read_b((stage + 1) & (S - 1), 0, fb[0]);
#pragma unroll
        for (int mi = 0; mi < RM; ++mi)
#pragma unroll
          for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = sh_mfma16(fb[ph & 1][ni], a[mi][2 * j + (ph >> 1)][ph & 1], acc[mi][ni]);
      }
      stage = (stage + 1) & (S - 1);
    }
    // ---- the unit's 16 RM x 64 values of this wave: lane = row mrow + 16 mi, columns n + 32 h (8 each)
    asm volatile("" ::: "memory");
    if constexpr (RES && !RAG) {
      // behind this unit's residual (fetched at the start of the unit before): 2 KS2 - 1 steps of b, the next residual, the last unit's stores
      if (steady) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * (2 * KS2 - 1) + E_R + E_ST) : "memory");
      else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * KS2 - 2) : "memory");
    }
    const int n = (int)(u - mt * nt) * 64 + g * 8;
    const long long row_bytes = (long long)p.N * 2;
    const long long at0 = mrow * row_bytes + n * 2;
    const bool aligned = ((size_t)p.out & 15) == 0;
    auto finish = [&](auto act) __attribute__((always_inline)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int left = RAG ? p.N - (n + 32 * h) : 8;
        if (RAG && left <= 0) continue;
        float b8[8];
        ld_f32<8>(bias + n + 32 * h, 8, b8);  // (the bias's place in LDS is padded with zeros)
#pragma unroll
        for (int mi = 0; mi < RM; ++mi) {
          float z[8];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            z[r] = acc[mi][2 * h][r] + b8[r];
            z[4 + r] = acc[mi][2 * h + 1][r] + b8[4 + r];
          }
          const bool in = mrow + 16 * mi < p.M;
          const long long at = at0 + 16 * mi * row_bytes + 64 * h;
          if (PRE && in) {
            if constexpr (RAG) st_chunk<T>((T*)((char*)p.pre + at), left, pack16<T>(z));
            else st16_any((char*)p.pre + at, pack16<T>(z));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) z[e] = act_value(z[e], decltype(act)::value);
          if constexpr (RES) {
            float r8[8];
            uint4 q = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (!RAG) q = *reinterpret_cast<const uint4*>(smem + R0 + (u & 1) * R_BYTES + wave * (2048 * RM) + (16 * mi + li) * 128 + (((h * 4 + g) ^ (li & 7)) * 16));
            else if (in) q = ld_chunk<T>((const T*)((const char*)p.residual + at), left);
            unpack16<T>(q, r8);
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] += r8[e];
          }
          if (!in) continue;
          // without a residual the stores go past the caches (401408 x 256 -> 1024: 302 -> 280 us, 300032 x 384 -> 512 165 -> 145; but 600064 x 256 -> 320 171 -> 193); with one that costs a fifth (381 -> 463)
          if constexpr (RAG) {
            st_chunk<T>((T*)((char*)p.out + at), left, pack16<T>(z));
          } else {
            if (RES || !aligned) st16_any((char*)p.out + at, pack16<T>(z));
            else st16<true>((char*)p.out + at, pack16<T>(z));
          }
        }
      }
    };
    if (p.act == SH_ACT_NONE) finish(std::integral_constant<int, SH_ACT_NONE>());
    else if (p.act == SH_ACT_RELU) finish(std::integral_constant<int, SH_ACT_RELU>());
    else if (p.act == SH_ACT_GELU) finish(std::integral_constant<int, SH_ACT_GELU>());
    else finish(std::integral_constant<int, SH_ACT_SILU>());
    asm volatile("" ::: "memory");
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the DMAs past the end have landed before the LDS is given back
}

static bool rows_whole(const LinearArgs& p) {
  return p.K % 8 == 0 && p.N % 64 == 0 && p.ldb % 8 == 0 && !(((size_t)p.a | (size_t)p.b | (size_t)p.residual) & 15);
}
// What the kernel can take: K in registers, at least four units a CU.  (Ragged columns alone are the LDS-DMA tiles' business.)
bool linear_rows_fits(const LinearArgs& p, int dtype) {
  if (dtype != SH_BF16 || p.K > 512 || p.N > kRowsMaxN || p.K < 32 || (int64_t)ceil_div(p.M, 256) * ceil_div(p.N, 64) < 1024) return false;
  return rows_whole(p) || p.K % 8 != 0 || (((size_t)p.a) & 15) != 0;
}
// ... and where it pays; us of this kernel and of what takes the call otherwise (the tiles of linear256.hip and linear.hip), over N from 50 to 2048 by K from 32 to 512, rows for 2e8 values.
// Whole chunks and 64-column units: with a residual (100352 x 512 -> 2048: 257 and 331, 1605632 x 128 -> 512: 734 and 765, 568064 x 32 -> 320: 164 and 258; within 10 % either way at N = 64);
// without one for K and N from 256 (401408 x 256 -> 1024: 280 and 326, 347136 x 256 -> 320: 92 and 112; but 1605632 x 128 -> 512: 452 and 435, 446208 x 256 -> 192: 94 and 87).
// Rows that are no whole chunks, which the other kernels stage through registers: without a residual from three units a row tile (300000 x 77 -> 192: 47 and 55, 100000 x 333 -> 777: 109 and
// 152; but 622848 x 129 -> 192: 204 and 184); with one, read in the epilogue row by row, where K is long enough to pay for that (with gelu, 100000 x 333 -> 777: 207 and 270, 314880 x 505
// -> 130: 185 and 284, 443392 x 201 -> 250: 262 and 305; but 361472 x 33 -> 520: 333 and 258, 200000 x 129 -> 130: 92 and 61, 503552 x 333 -> 64: 138 and 131).
bool linear_rows_takes(const LinearArgs& p, int dtype) {
  if (!linear_rows_fits(p, dtype)) return false;
  if (rows_whole(p)) return p.residual != nullptr || (p.K >= 256 && p.N >= 256);
  return p.residual != nullptr ? p.K >= 192 && p.N >= 128 : p.N >= 192;
}
size_t linear_rows_workspace_bytes(const LinearArgs& p) { return rows_whole(p) ? 0 : (size_t)p.N * ((p.K + 7) / 8 * 8) * 2; }

// b [N][ldb] -> rows of kp elements, zeros behind K
__global__ __launch_bounds__(256) void linear_pad_kernel(const bf16_t* __restrict__ b, bf16_t* __restrict__ out, int n, int k, int ldb, int kp) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const int row = (int)(i / (kp / 8)), c = (int)(i % (kp / 8)) * 8;
  if (row < n) *reinterpret_cast<uint4*>(out + (long long)row * kp + c) = ld_chunk<bf16_t>(b + (long long)row * ldb + c, k - c);
}

// workspace: linear_rows_workspace_bytes() (unless b's rows are already padded with zeros to a multiple of 8 at 16-byte addresses: b_padded)
int linear_rows_launch(const LinearArgs& base, bool b_padded, void* workspace, hipStream_t s, const char* what) {
  LinearArgs p = base;
  const bool rag = !rows_whole(base);
  // K <= 128: ragged rows without a residual and whole ones with it are all that linear_rows_takes lets through
  SH_REQUIRE(p.K > 128 || rag == (p.residual == nullptr), "%s: rows in registers: K = %d", what, p.K);
  if (rag && !b_padded) {
    const int kp = (p.K + 7) / 8 * 8;
    linear_pad_kernel<<<(unsigned)(((int64_t)p.N * (kp / 8) + 255) / 256), 256, 0, s>>>((const bf16_t*)p.b, (bf16_t*)workspace, p.N, p.K, p.ldb, kp);
    if (check_launch(what)) return 1;
    p.b = workspace;
    p.ldb = kp;
  }
  p.n_tiles = (unsigned)ceil_div(p.N, 64);
  const unsigned units = (unsigned)ceil_div(p.M, 256) * p.n_tiles, per_cu = (units + 255) / 256;
#define SH_ROWS(KS2, RES, PRE, RAG) linear_rows_kernel<KS2, RES, PRE, RAG><<<256, 512, 0, s>>>(p, units, per_cu)
#define SH_ROWS_K(RES, PRE)                                                                      \
  if (rag) {                                                                                     \
    switch ((p.K + 127) / 128) {                                                                 \
      case 1: if constexpr (!RES) SH_ROWS(1, RES, PRE, true); break;                          \
      case 2: SH_ROWS(2, RES, PRE, true); break;                                              \
      case 3: SH_ROWS(3, RES, PRE, true); break;                                              \
      default: SH_ROWS(4, RES, PRE, true); break;                                             \
    }                                                                                            \
  } else {                                                                                       \
    switch ((p.K + 127) / 128) {                                                                 \
      case 1: if constexpr (RES) SH_ROWS(1, RES, PRE, false); break;                          \
      case 2: SH_ROWS(2, RES, PRE, false); break;                                             \
      case 3: SH_ROWS(3, RES, PRE, false); break;                                             \
      default: SH_ROWS(4, RES, PRE, false); break;                                            \
    }                                                                                            \
  }
  if (p.residual != nullptr) {
    if (p.pre != nullptr) { SH_ROWS_K(true, true) }
    else { SH_ROWS_K(true, false) }
  } else {
    if (p.pre != nullptr) { SH_ROWS_K(false, true) }
    else { SH_ROWS_K(false, false) }
  }
#undef SH_ROWS_K
#undef SH_ROWS
  return check_launch(what);
}

}  // namespace sh
