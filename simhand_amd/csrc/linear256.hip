// out [M][N] = a [M][K] b[N][K]^T of 16-bit operands in 256 x 256 tiles, for many rows (linear_fwd, and the input gradient).
//
// One block of 8 waves per CU keeps its operands in the CU's 160 KB of LDS -- activations in three stages of a 64-element k-step (they come from HBM: fetched two
// steps ahead), weights in two (L2: one step ahead) -- filled by LDS-DMA, 128 bytes of operand traffic per MFMA.  A block works through a LIST of tiles and its k-steps
// form one sequence across them: the first steps of the next tile are already on their way while the finished one is scaled, activated, added to its residual and stored, and
// the stores drain under the next tile's MFMAs.  These layers are short in K (256 .. 512 for the wide outputs: 4 .. 8 steps) and bound by memory, so a kernel that fills
// and drains its pipeline for every tile pays for both ends each time.
// Measured, bf16: 1605632 x 128 -> 512 436 us (2.1 GB: 4.7 TB/s), 1605632 x 64 -> 256 199 us (1.03 GB: 5.2 TB/s); 100352 x 512 -> 2048 with a residual 331 us, where its operand traffic
// binds (the rows-in-registers kernel takes that one: 257).
#include "linear.h"

namespace sh {

__device__ uint4 g_l256_zero[8];  // read-only zeros: the DMAs past the last row, column or step fetch these

__global__ __launch_bounds__(512, 1) void linear256_kernel(LinearArgs p, unsigned tiles, unsigned per_xcd) {
  typedef bf16_t T;
  constexpr int A_BYTES = 256 * 128, B_BASE = 3 * A_BYTES;
  __shared__ __attribute__((aligned(16))) char smem[5 * A_BYTES];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) char*)smem;
  // inline asm: hipcc's wait-count pass would drain every outstanding LDS-DMA in front of each LDS read; the loop counts them itself.  Nothing is returned in registers.
  auto dma16 = [](const void* src, unsigned lds_addr) __attribute__((always_inline)) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(src));
  };
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int li = lane & 15, g = lane >> 4, wm = wave >> 2, wn = wave & 3;
  // the block's tiles: XCD x (blocks x, x + 8, ..) owns tiles [x per_xcd, (x + 1) per_xcd), its CUs take them in turn -- at any time the XCD's L2 serves the n-tiles of few
  // row tiles and the whole of b
  const unsigned xcd = blockIdx.x & 7, cus = gridDim.x >> 3;
  const unsigned t_end = (xcd + 1) * per_xcd < tiles ? (xcd + 1) * per_xcd : tiles;
  unsigned tile = xcd * per_xcd + (blockIdx.x >> 3);
  if (tile >= t_end) return;
  const int nk = (p.K + 63) / 64;

  // DMA map: instruction i of a wave fills tile rows 64 i + 8 wave .. + 7 (128 B each); lane l = row l >> 3, 16-byte slot l & 7.  The swizzle is applied to the source: slot s
  // of a row holds chunk s ^ key(row).
  const int slot = lane & 7, lrow = wave * 8 + (lane >> 3);
  auto key_b = [](int row) __attribute__((always_inline)) -> int { return ((row >> 1) & 1) | (((row >> 3) & 3) << 1); };
  const int ka = (slot ^ ((lrow >> 1) & 7)) * 8, kb = (slot ^ key_b(lrow)) * 8;  // first element of the lane's chunk inside the k-step
  const char* zero = reinterpret_cast<const char*>(g_l256_zero) + slot * 16;
  const unsigned dst_row = (unsigned)wave * 1024u;
  // two walkers over the sequence of k-steps (tile, k): a two steps ahead of the MFMAs, b one
  struct Walk { unsigned tile; int k; unsigned stage; };
  Walk wa = {tile, 0, 0}, wb = {tile, 0, 0};
  const char* pa[4];
  const char* pb[4];
  auto rows_a = [&]() __attribute__((always_inline)) {
    const long long m0 = (long long)(wa.tile / p.n_tiles) * 256 + lrow;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long m = m0 + 64 * i;
      pa[i] = reinterpret_cast<const char*>((const T*)p.a + (m < p.M ? m : p.M - 1) * p.K + ka);
    }
  };
  auto rows_b = [&]() __attribute__((always_inline)) {
    const int n0 = (int)(wb.tile % p.n_tiles) * 256 + lrow;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int n = n0 + 64 * i;
      pb[i] = reinterpret_cast<const char*>((const T*)p.b + (long long)(n < p.N ? n : p.N - 1) * p.ldb + kb);
    }
  };
  auto dma_a = [&](int i) __attribute__((always_inline)) {
    const bool ok = wa.tile < t_end && wa.k + ka < p.K;
    dma16(ok ? pa[i] + wa.k * 2 : zero, lds0 + wa.stage * A_BYTES + dst_row + i * 8192);
  };
  auto dma_b = [&](int i) __attribute__((always_inline)) {
    const bool ok = wb.tile < t_end && wb.k + kb < p.K;
    dma16(ok ? pb[i] + wb.k * 2 : zero, lds0 + B_BASE + wb.stage * A_BYTES + dst_row + i * 8192);
  };
  auto next_a = [&]() __attribute__((always_inline)) {
    wa.stage = wa.stage == 2 ? 0 : wa.stage + 1;
    wa.k += 64;
    if (wa.k >= p.K) {
      wa.k = 0;
      wa.tile += cus;
      if (wa.tile < t_end) rows_a();
    }
  };
  auto next_b = [&]() __attribute__((always_inline)) {
    wb.stage ^= 1;
    wb.k += 64;
    if (wb.k >= p.K) {
      wb.k = 0;
      wb.tile += cus;
      if (wb.tile < t_end) rows_b();
    }
  };
  rows_a();
  rows_b();
#pragma unroll
  for (int i = 0; i < 4; ++i) dma_a(i);
  next_a();
#pragma unroll
  for (int i = 0; i < 4; ++i) dma_b(i);
  next_b();
#pragma unroll
  for (int i = 0; i < 4; ++i) dma_a(i);
  next_a();

  const int fo = (g ^ ((li >> 1) & 7)) * 16;
  const int fa0 = (wm * 128 + li) * 128;
  const int rowb = wn * 64 + lin_col(0, li);
  const int fb0 = rowb * 128 + ((g ^ key_b(rowb)) * 16);
  unsigned sa = 0, sb = 0;
  bool loose = false;  // the tile before this one was a whole one: at least 16 stores stand behind its DMAs
  for (; tile < t_end; tile += cus) {
    f32x4 acc[8][4];
#pragma unroll
    for (int mi = 0; mi < 8; ++mi)
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) acc[mi][ni] = (f32x4){0.f, 0.f, 0.f, 0.f};
    for (int kt = 0; kt < nk; ++kt) {
      // In flight, oldest first: this step's b (4 instructions), the next step's a (4), then whatever the epilogue issued.  All but the last 4 (+ 16 stores) have landed ->
      // this step's operands are in LDS; the barrier makes them everybody's, and says that the step before has been read.
      if (kt == 0 && loose) asm volatile("s_waitcnt vmcnt(20) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const char* st = smem + sa * A_BYTES;
      const char* stb = smem + B_BASE + sb * A_BYTES;
      sa = sa == 2 ? 0 : sa + 1;
      sb ^= 1;
      uint4 fb[2][4], fa[2][2];
#pragma unroll
      for (int ni = 0; ni < 4; ++ni) fb[0][ni] = *reinterpret_cast<const uint4*>(stb + fb0 + (lin_col(ni, 0) - lin_col(0, 0)) * 128);
      fa[0][0] = *reinterpret_cast<const uint4*>(st + fa0 + fo);
      fa[0][1] = *reinterpret_cast<const uint4*>(st + fa0 + 16 * 128 + fo);
#pragma unroll
      for (int grp = 0; grp < 8; ++grp) {
        const int kk = grp >> 2, q = grp & 3;
        if (grp < 7) {  // the next group's fragments are read under this group's MFMAs
          const int nkk = (grp + 1) >> 2, nq = (grp + 1) & 3;
          const int f = nkk == 0 ? fo : (fo ^ 64);
          if (grp == 3) {
#pragma unroll
            for (int ni = 0; ni < 4; ++ni) fb[1][ni] = *reinterpret_cast<const uint4*>(stb + (fb0 ^ 64) + (lin_col(ni, 0) - lin_col(0, 0)) * 128);
          }
          fa[(grp + 1) & 1][0] = *reinterpret_cast<const uint4*>(st + fa0 + (2 * nq) * 16 * 128 + f);
          fa[(grp + 1) & 1][1] = *reinterpret_cast<const uint4*>(st + fa0 + (2 * nq + 1) * 16 * 128 + f);
        }
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) acc[2 * q][ni] = sh_mfma16(fb[kk][ni], fa[grp & 1][0], acc[2 * q][ni]);
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) acc[2 * q + 1][ni] = sh_mfma16(fb[kk][ni], fa[grp & 1][1], acc[2 * q + 1][ni]);
        // one DMA instruction per group, the next step's b first
        if (grp < 4) dma_b(grp);
        else dma_a(grp - 4);
      }
      next_b();
      next_a();
    }
    asm volatile("" ::: "memory");  // the epilogue's memory operations stay behind the loop's DMAs (the count of `loose` relies on it)
    // lane: row m0 + 16 mi, columns n, n + 32 (8 each)
    const long long tm = (long long)(tile / p.n_tiles) * 256;
    const int tn = (int)(tile % p.n_tiles) * 256;
    const long long m0 = tm + wm * 128 + li;
    const int n = tn + wn * 64 + g * 8;
    loose = tm + 256 <= p.M && tn + 256 <= p.N;
    float bias[2][8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[j][e] = 0.f;
      if (p.bias != nullptr && n + 32 * j < p.N) ld_f32<8>(p.bias + n + 32 * j, 8, bias[j]);
    }
    const long long row_bytes = (long long)p.N * 2;
    const long long at0 = m0 * row_bytes + n * 2;
    auto finish = [&](auto has_res, auto has_pre, auto act) __attribute__((always_inline)) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // two row groups at a time: their residual vectors are requested together
        uint4 res[2][2];
        if constexpr (decltype(has_res)::value) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 2; ++j)
              if (m0 + 32 * q + 16 * h < p.M && n + 32 * j < p.N)
                res[h][j] = ld16_any((const char*)p.residual + at0 + (32 * q + 16 * h) * row_bytes + 64 * j);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int mi = 2 * q + h;
            if (m0 + 16 * mi >= p.M || n + 32 * j >= p.N) continue;
            const long long at = at0 + 16 * mi * row_bytes + 64 * j;
            float z[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              z[r] = acc[mi][2 * j][r] + bias[j][r];
              z[4 + r] = acc[mi][2 * j + 1][r] + bias[j][4 + r];
            }
            if constexpr (decltype(has_pre)::value) st16_any((char*)p.pre + at, pack16<T>(z));
#pragma unroll
            for (int e = 0; e < 8; ++e) z[e] = act_value(z[e], decltype(act)::value);
            if constexpr (decltype(has_res)::value) {
              float r[8];
              unpack16<T>(res[h][j], r);
#pragma unroll
              for (int e = 0; e < 8; ++e) z[e] += r[e];
            }
            st16_any((char*)p.out + at, pack16<T>(z));
          }
        asm volatile("" ::: "memory");
      }
    };
    auto by_act = [&](auto has_res, auto has_pre) __attribute__((always_inline)) {
      if (p.act == SH_ACT_NONE) finish(has_res, has_pre, std::integral_constant<int, SH_ACT_NONE>());
      else if (p.act == SH_ACT_RELU) finish(has_res, has_pre, std::integral_constant<int, SH_ACT_RELU>());
      else if (p.act == SH_ACT_GELU) finish(has_res, has_pre, std::integral_constant<int, SH_ACT_GELU>());
      else finish(has_res, has_pre, std::integral_constant<int, SH_ACT_SILU>());
    };
    if (p.residual != nullptr) {
      if (p.pre != nullptr) by_act(std::true_type(), std::true_type());
      else by_act(std::true_type(), std::false_type());
    } else {
      if (p.pre != nullptr) by_act(std::false_type(), std::true_type());
      else by_act(std::false_type(), std::false_type());
    }
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // the DMAs past the end have landed before the LDS is given back
}

// Rows of 16-byte chunks at 16-byte addresses (the DMA's unit), and enough tiles for the chip.
bool linear256_takes(const LinearArgs& p, int dtype) {
  if (dtype != SH_BF16 || p.K % 8 || p.N % 8 || p.ldb % 8 || p.N < 128) return false;
  if (((size_t)p.a | (size_t)p.b) & 15) return false;
  return (int64_t)ceil_div(p.M, 256) * ceil_div(p.N, 256) >= 192;
}
int linear256_launch(const LinearArgs& base, hipStream_t s, const char* what) {
  LinearArgs p = base;
  p.n_tiles = (unsigned)ceil_div(p.N, 256);
  const unsigned tiles = (unsigned)ceil_div(p.M, 256) * p.n_tiles;
  const unsigned per_xcd = (tiles + 7) / 8;
  linear256_kernel<<<256, 512, 0, s>>>(p, tiles, per_xcd);
  return check_launch(what);
}

}  // namespace sh
