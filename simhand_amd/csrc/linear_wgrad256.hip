// dw [N][K] = dz^T x of 16-bit operands in 256 x 256 tiles over a range of rows, x as it is or as its 8-bit checkpoint (linear_wgrad).
//
// The reduction runs over rows, so both operands are read transposed from LDS (ds_read_b64_tr_b16).  One block of 8 waves per CU, as 2 (n) x 4 (k) of 128 x 64 each; a step =
// 32 rows; every operand tile is four sub-tiles of [32 rows][64 columns] whose 32-byte column groups are rotated by row / 2, which keeps the transposed reads off
// each other's banks.  The operands arrive by LDS-DMA several steps ahead, one barrier per step.
// A8: the codes (8 KB a step instead of 16) and their exponents arrive by LDS-DMA too; every thread decodes the 16 codes it fetched itself -- no barrier in between -- into the
// 16-bit sub-tile of the NEXT step while the matrix cores work on this one.  What the layer reads of x halves, and the product is memory-bound: the decoding hides.
// Measured, 401408 x 1024 -> 256 bf16 (1.03 GB, 210 GFLOP): 207 to 213 us (HBM 5.3 TB/s), from codes 201 to 209 (0.63 GB; 133 us at the rate of
// a large matrix product, itself 63 % of the dense peak; the matrix cores are 46 % busy either way), and 12 us for the join of the splits.
#include "linear.h"

namespace sh {

__device__ uint4 g_w256_zero[8];  // read-only zeros

typedef __attribute__((ext_vector_type(4))) short s16x4_w;

template <bool A8>
__global__ __launch_bounds__(512, 1) void linear_wgrad256_kernel(WgradArgsL p) {
  typedef bf16_t T;
  constexpr int KP = 32, SUB = KP * 128, HALF = 4 * SUB;    // rows per step, bytes of a sub-tile / of one operand's tile
  constexpr int NS = 5, D = NS - 1;                         // stages; steps the DMAs run ahead
  constexpr int RAW = KP * 256, RAWE = KP * 8;              // codes and exponents of a step
  constexpr int XS = A8 ? 2 : NS;                           // stages of the 16-bit x tile
  constexpr int X0 = NS * HALF, R0 = X0 + XS * HALF, E0 = R0 + (A8 ? NS * RAW : 0), BYTES = E0 + (A8 ? NS * RAWE : 0);
  static_assert(BYTES <= 160 * 1024, "LDS of a CU");
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
  auto dma16 = [](const void* src, unsigned lds_addr) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(src));
  };
  auto dma4 = [](const void* src, unsigned lds_addr) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_addr), "v"(src));
  };
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, g = lane >> 4, wm = wave >> 2, wn = wave & 3;
  unsigned logical = xcd_order(blockIdx.x, gridDim.x);
  const int k0 = (int)(logical % p.k_tiles) * 256; logical /= p.k_tiles;
  const int n0 = (int)(logical % p.n_tiles) * 256;
  const int split = (int)(logical / p.n_tiles);
  const long long r0 = (long long)split * p.per_split;
  const long long r1 = r0 + p.per_split < p.M ? r0 + p.per_split : p.M;
  const int rows = r0 < r1 ? (int)(r1 - r0) : 0;
  const int nk = (rows + KP - 1) / KP;

  // a DMA instruction fills 8 rows of a sub-tile: lane l = row l >> 3, 16-byte slot l & 7; the slot's columns carry the row's rotation
  const int slot = lane & 7, r8 = lane >> 3;
  const char* zero = reinterpret_cast<const char*>(g_w256_zero) + slot * 16;
  constexpr int NI = A8 ? 2 : 4;  // DMA instructions of dz / x sub-tiles per wave and step
  const int sub = A8 ? wave >> 1 : wave & 3, part0 = A8 ? (wave & 1) * 2 : 0;
  const bool is_dz = A8 || wave < 4;
  const int width = is_dz ? p.N : p.K, base = is_dz ? n0 : k0;
  const T* src0 = is_dz ? (const T*)p.dz : (const T*)p.x;
  const long long step_bytes = (long long)KP * width * 2;
  const char* ptr[NI];
  bool inside[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int row = 8 * (part0 + i) + r8;
    const int col = base + sub * 64 + ((((slot >> 1) - (row >> 1)) & 3) * 16) + (slot & 1) * 8;
    inside[i] = col < width;
    ptr[i] = reinterpret_cast<const char*>(src0 + (r0 + row) * width + (inside[i] ? col : 0));
  }
  // A8: lane = row 4 wave + (lane >> 4) of the step, codes k0 + 16 (lane & 15) .. + 15; exponents of the wave's four rows: lanes 0 .. 7, half a row's 8 bytes each (all 32 rows by
  // every wave would be 256 cache lines a step, three times what the operands take)
  const int crow = 4 * wave + (lane >> 4), ccol = 16 * li;
  const long long eb = (p.K + kAct8Block - 1) / kAct8Block;
  const bool cin = A8 && k0 + ccol < p.K, ein = A8 && k0 / 32 + 4 * (lane & 1) < eb;
  const uint8_t* cptr = A8 ? p.codes + (r0 + crow) * p.K + (cin ? k0 + ccol : 0) : nullptr;
  const uint8_t* eptr = A8 ? p.exps + (r0 + 4 * wave + (lane >> 1)) * eb + (ein ? k0 / 32 + 4 * (lane & 1) : 0) : nullptr;
  unsigned fill = 0;  // stage the next DMAs go to
  auto dma_step = [&](int c) __attribute__((always_inline)) {
    const int left = rows - c * KP;  // rows of step c (<= 0: none, zeros)
    const unsigned dst = lds0 + (is_dz ? 0 : X0) + fill * HALF + sub * SUB + part0 * 1024;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      dma16(inside[i] && 8 * (part0 + i) + r8 < left ? ptr[i] : zero, dst + i * 1024);
      ptr[i] += step_bytes;
    }
    if constexpr (A8) {
      dma16(cin && crow < left ? (const void*)cptr : (const void*)zero, lds0 + R0 + fill * RAW + wave * 1024);
      if (lane < 8) dma4(ein && 4 * wave + (lane >> 1) < left ? (const void*)eptr : (const void*)zero, lds0 + E0 + fill * RAWE + wave * 32);
      cptr += (long long)KP * p.K;
      eptr += KP * eb;
    }
    fill = fill == NS - 1 ? 0 : fill + 1;
  };
  // the thread's own 16 codes of the step in stage `from`: fetched from LDS, then decoded into their 32 bytes of the 16-bit tile `to`.  The halves of a 32-byte group change places in
  // the odd sub-tiles: eight neighbouring lanes then write 128 different bytes of the banks.
  uint4 cq;
  unsigned ce;
  auto codes_get = [&](unsigned from) __attribute__((always_inline)) {
    cq = *reinterpret_cast<const uint4*>(smem + R0 + from * RAW + wave * 1024 + lane * 16);
    ce = *reinterpret_cast<const uint8_t*>(smem + E0 + from * RAWE + crow * 8 + (li >> 1));
  };
  const int put_at = X0 + (li >> 2) * SUB + crow * 128 + (((li & 3) + (crow >> 1)) & 3) * 32 + ((li >> 2) & 1) * 16;
  auto codes_put = [&](unsigned to) __attribute__((always_inline)) {
    const float sc = act8_scale(ce);
    char* at = smem + to * HALF;
    *reinterpret_cast<uint4*>(at + put_at) = act8_decode8_h16(cq.x, cq.y, sc);
    *reinterpret_cast<uint4*>(at + (put_at ^ 16)) = act8_decode8_h16(cq.z, cq.w, sc);
  };

  f32x4 acc[8][4];
#pragma unroll
  for (int mi = 0; mi < 8; ++mi)
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < D; ++c) dma_step(c);

  typedef s16x4_w __attribute__((address_space(3))) * lds_ptr;
  auto tr2 = [](const char* a) __attribute__((always_inline)) -> uint4 {
    const s16x4_w lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(a));
    const s16x4_w hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(a + 16 * 128));
    const uint2 l = __builtin_bit_cast(uint2, lo), h = __builtin_bit_cast(uint2, hi);
    return make_uint4(l.x, l.y, h.x, h.y);
  };
  // lane's rows of a step: 4g + (li >> 2) and + 16 (same rotation); its 8 bytes of the 32-byte column group: (li & 3) * 8
  const int frow = 4 * g + (li >> 2);
  int offs[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) offs[q] = frow * 128 + (((q + (frow >> 1)) & 3) * 32) + (li & 3) * 8;

  const int xhalf = A8 ? (wn & 1) * 16 : 0;
  // The barrier stands in the MIDDLE of a step: it says that step j + 1 has landed (and, A8, is decoded) while half of step j's MFMAs are still to come, and under those the
  // first fragments of step j + 1 are read.  With the barrier at the top all eight waves read fragments at once and the matrix cores waited for them: 44 % busy.
  uint4 fa[4], fb[2][4];
  auto read_a = [&](unsigned stage, int mi) __attribute__((always_inline)) {
    fa[mi & 3] = tr2(smem + stage * HALF + (wm * 2 + (mi >> 2)) * SUB + offs[mi & 3]);
  };
  auto x_tile = [&](int j, unsigned stage) __attribute__((always_inline)) { return smem + X0 + (A8 ? (unsigned)(j & 1) : stage) * HALF + wn * SUB; };
  if constexpr (A8) {  // the first step's x tile (its codes are this thread's own)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * (D - 1)) : "memory");
    codes_get(0);
    codes_put(0);
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 * (D - 1)) : "memory");
#pragma unroll
  for (int ni = 0; ni < 4; ++ni) fb[0][ni] = tr2(x_tile(0, 0) + (offs[ni] ^ xhalf));
  read_a(0, 0);
  read_a(0, 1);
  unsigned use = 0;  // stage of step j
  auto step = [&](int j, auto parity) __attribute__((always_inline)) {
    constexpr int P = decltype(parity)::value;
    const unsigned nxt = use == NS - 1 ? 0 : use + 1;
    if constexpr (A8) {  // step j + 1 has landed as far as this wave's own DMAs go: steps j + 2 .. j + D - 1 may be in flight
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(4 * (D - 2)) : "memory");
      codes_get(nxt);
    }
#pragma unroll
    for (int mi = 0; mi < 8; ++mi) {
      if (mi < 6) read_a(use, mi + 2);
      if (mi == 5) {
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) fb[P ^ 1][ni] = tr2(x_tile(j + 1, nxt) + (offs[ni] ^ xhalf));
      }
      if (mi >= 6) read_a(nxt, mi - 6);
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = sh_mfma16(fa[mi & 3], fb[P][ni], acc[mi][ni]);
      if constexpr (A8) {
        if (mi == 1) codes_put((unsigned)((j + 1) & 1));  // read last in the second half of step j - 2
      }
      if (mi == 3) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 * (D - 2)) : "memory");
        dma_step(j + D);  // into the stage of step j - 1, which every wave has read
      }
    }
    use = nxt;
  };
  for (int j = 0; j < nk; j += 2) {
    step(j, std::integral_constant<int, 0>());
    if (j + 1 < nk) step(j + 1, std::integral_constant<int, 1>());
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");

  // lane: rows n0 + 128 wm + 16 mi + 4 g + r, column k0 + 64 wn + 16 ni + li
  float* out = p.part + (long long)split * p.N * p.K;
#pragma unroll
  for (int mi = 0; mi < 8; ++mi)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + wm * 128 + mi * 16 + 4 * g + r;
      if (n >= p.N) continue;
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) {
        const int k = k0 + wn * 64 + ni * 16 + li;
        if (k < p.K) out[(long long)n * p.K + k] = acc[mi][ni][r];
      }
    }
}

// 16-byte chunks at 16-byte addresses, both sides wide enough for the tile, rows for at least 16 steps a block; codes: exponents at 4-byte addresses (K a multiple of 128)
bool linear_wgrad256_takes(const void* dz, const void* x, const uint8_t* codes, const uint8_t* exps, int64_t rows, int in_dim, int out_dim, int dtype) {
  if (dtype != SH_BF16 || out_dim % 8 || in_dim % 8 || out_dim < 192 || in_dim < 192 || rows < 4096) return false;
  if ((size_t)dz & 15) return false;
  return codes ? in_dim % 128 == 0 && !((size_t)codes & 15) && !((size_t)exps & 3) : !((size_t)x & 15);
}
// as many splits as fill the CUs once
void linear_wgrad256_plan(int64_t rows, int in_dim, int out_dim, int* splits, int64_t* per) {
  const int64_t tiles = (int64_t)ceil_div(in_dim, 256) * ceil_div(out_dim, 256), steps = (rows + 31) / 32;
  int64_t sk = 256 / tiles;
  if (sk > (steps + 15) / 16) sk = (steps + 15) / 16;
  if (sk < 1) sk = 1;
  const int64_t each = (steps + sk - 1) / sk;
  *per = each * 32;
  *splits = (int)((steps + each - 1) / each);
}
int linear_wgrad256_launch(const WgradArgsL& base, int splits, hipStream_t s) {
  WgradArgsL p = base;
  p.n_tiles = (unsigned)ceil_div(p.N, 256);
  p.k_tiles = (unsigned)ceil_div(p.K, 256);
  const unsigned grid = p.n_tiles * p.k_tiles * (unsigned)splits;
  if (p.codes) linear_wgrad256_kernel<true><<<grid, 512, 0, s>>>(p);
  else linear_wgrad256_kernel<false><<<grid, 512, 0, s>>>(p);
  return check_launch("linear_wgrad");
}

}  // namespace sh
