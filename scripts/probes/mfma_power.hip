// Probe: sustained MFMA rate AND energy per FLOP on RANDOM vs ZERO register operands, bf16 16x16x32 vs 32x32x16 vs the scaled e4m3 16x16x128
// (the chip clocks to its power budget: which shape buys more FLOP per joule?).  2 waves per SIMD, operands in registers, no memory traffic.
// Round 6: the 32x32x16 loop of round 5 had 4 accumulators per wave, each used twice per iteration -- issue-bound on a
// dependent chain even on zeros, so its column said nothing about the instruction.  Now 8 INDEPENDENT 32x32 accumulators per wave (128 acc registers,
// 16 waves' worth of independent MFMAs per SIMD with 2 waves), one MFMA each per iteration; 16x16x32 keeps its 16 independent accumulators.  A host
// thread samples the amdgpu hwmon power node while each shape runs ~1.5 s at the cap; pJ/FLOP = mean socket power / rate (idle power NOT subtracted).
// build: hipcc --offload-arch=gfx950 -O3 -Xclang -target-feature -Xclang -packed-fp32-ops -o scripts/probes/mfma_power scripts/probes/mfma_power.hip -lpthread ; run on the GPU box.
#include <hip/hip_runtime.h>
#include <dirent.h>
#include <limits.h>
#include <cctype>
#include <atomic>
#include <chrono>
#include <cstdio>
#include <cstdlib>
#include <string>
#include <thread>
#include <vector>
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) int i32x8;

template <int SHAPE>
__global__ __launch_bounds__(512, 1) void k(const uint4* in, float* out, int iters) {
  const int tid = threadIdx.x;
  uint4 a[4], b[4];
  for (int i = 0; i < 4; ++i) { a[i] = in[(tid * 8 + i) & 4095]; b[i] = in[(tid * 8 + 4 + i) & 4095]; }
  float s = 0.f;
  if (SHAPE == 16) {
    f32x4 acc[16];
    for (int i = 0; i < 16; ++i) acc[i] = (f32x4){0, 0, 0, 0};
    for (int it = 0; it < iters; ++it) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a[i & 3]), __builtin_bit_cast(bf16x8, b[(i >> 2) & 3]), acc[i], 0, 0, 0);
    }
    for (int i = 0; i < 16; ++i) s += acc[i][0] + acc[i][1] + acc[i][2] + acc[i][3];
  } else if (SHAPE == 128) {  // v_mfma_scale_f32_16x16x128_f8f6f4 on e4m3 bytes, unit scales: the fp8 configuration's instruction (65 536 FLOP each)
    f32x4 acc[16];
    for (int i = 0; i < 16; ++i) acc[i] = (f32x4){0, 0, 0, 0};
    i32x8 a8[2], b8[2];
    for (int i = 0; i < 4; ++i) {  // no e4m3 NaN bytes (0x7f / 0xff): clear the exponent's low bit, keep sign and the rest random
      a[i].x &= 0xF7F7F7F7u; a[i].y &= 0xF7F7F7F7u; a[i].z &= 0xF7F7F7F7u; a[i].w &= 0xF7F7F7F7u;
      b[i].x &= 0xF7F7F7F7u; b[i].y &= 0xF7F7F7F7u; b[i].z &= 0xF7F7F7F7u; b[i].w &= 0xF7F7F7F7u;
    }
    for (int i = 0; i < 2; ++i) {
      a8[i] = (i32x8){(int)a[2 * i].x, (int)a[2 * i].y, (int)a[2 * i].z, (int)a[2 * i].w, (int)a[2 * i + 1].x, (int)a[2 * i + 1].y, (int)a[2 * i + 1].z, (int)a[2 * i + 1].w};
      b8[i] = (i32x8){(int)b[2 * i].x, (int)b[2 * i].y, (int)b[2 * i].z, (int)b[2 * i].w, (int)b[2 * i + 1].x, (int)b[2 * i + 1].y, (int)b[2 * i + 1].z, (int)b[2 * i + 1].w};
    }
    for (int it = 0; it < iters; ++it) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        acc[i] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8[i & 1], b8[(i >> 1) & 1], acc[i], 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
    }
    for (int i = 0; i < 16; ++i) s += acc[i][0] + acc[i][1] + acc[i][2] + acc[i][3];
  } else {  // 32x32x16 bf16: 8 independent accumulators, one MFMA each per iteration (32 768 FLOP each: the same FLOPs per iteration as 16 x 16x16x32)
    f32x16 acc[8];
    for (int i = 0; i < 8; ++i) for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
    for (int it = 0; it < iters; ++it) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a[i & 3]), __builtin_bit_cast(bf16x8, b[(i >> 1) & 3]), acc[i], 0, 0, 0);
    }
    for (int i = 0; i < 8; ++i) for (int j = 0; j < 16; ++j) s += acc[i][j];
  }
  out[blockIdx.x * 512 + tid] = s;
}

// ---- amdgpu hwmon sampling (socket power in uW, gfx clock in Hz) ----
static std::string find_hwmon() {  // the hwmon directory of the card whose PCI address is HIP device 0's (a box can hold more cards than it shows)
  char bus[64] = {0};
  if (hipDeviceGetPCIBusId(bus, sizeof(bus), 0) != hipSuccess) bus[0] = 0;
  for (char* q = bus; *q; ++q) *q = (char)tolower(*q);
  for (int c = 0; c < 128; ++c) {
    const std::string dev = "/sys/class/drm/card" + std::to_string(c) + "/device";
    char real[512];
    if (!realpath(dev.c_str(), real)) continue;
    std::string rp = real;
    for (auto& ch : rp) ch = (char)tolower(ch);
    if (bus[0] && rp.find(bus) == std::string::npos) continue;
    std::string base = dev + "/hwmon";
    DIR* d = opendir(base.c_str());
    if (!d) continue;
    while (dirent* e = readdir(d)) {
      std::string n = e->d_name;
      if (n.rfind("hwmon", 0) == 0) {
        std::string p = base + "/" + n;
        FILE* f = fopen((p + "/power1_average").c_str(), "r");
        if (!f) f = fopen((p + "/power1_input").c_str(), "r");
        if (f) { fclose(f); closedir(d); return p; }
      }
    }
    closedir(d);
  }
  return "";
}
static double read_num(const std::string& p) {
  FILE* f = fopen(p.c_str(), "r");
  if (!f) return -1;
  double v = -1;
  if (fscanf(f, "%lf", &v) != 1) v = -1;
  fclose(f);
  return v;
}

int main() {
  const int nblk = 256 * 8, iters = 4000;
  uint4* in; float* out;
  hipMalloc(&in, 4096 * 16); hipMalloc(&out, nblk * 512 * 4);
  std::vector<unsigned> h(4096 * 4);
  hipEvent_t e0, e1; hipEventCreate(&e0); hipEventCreate(&e1);
  const std::string hw = find_hwmon();
  printf("hwmon: %s\n", hw.empty() ? "(none: power columns empty)" : hw.c_str());
  printf("| operands | MFMA | ms / 20 launches | TFLOP/s | socket W | sclk MHz | pJ / FLOP |\n|---|---|---|---|---|---|---|\n");
  for (int mode = 0; mode < 2; ++mode) {
    for (auto& v : h) {  // bf16 pairs: random values ~ N(0,1)-ish magnitudes (random sign / exponent near 0 / mantissa), or zeros
      unsigned lo = 0x3f00u + (rand() & 0xff) + ((rand() & 1) << 15) , hi = 0x3f00u + (rand() & 0xff) + ((rand() & 1) << 15);
      v = mode == 0 ? (lo | (hi << 16)) : 0u;
    }
    hipMemcpy(in, h.data(), 4096 * 16, hipMemcpyHostToDevice);
    for (int shape : {16, 32, 128, 16, 32, 128}) {
      auto launch20 = [&]() {
        for (int l = 0; l < 20; ++l) {
          if (shape == 16) k<16><<<nblk, 512>>>(in, out, iters); else if (shape == 32) k<32><<<nblk, 512>>>(in, out, iters); else k<128><<<nblk, 512>>>(in, out, iters);
        }
      };
      launch20(); hipDeviceSynchronize();  // warm: the clock settles at the cap
      std::atomic<bool> stop{false};
      double pw_sum = 0, ck_sum = 0; long pw_n = 0;
      std::thread smp([&]() {
        if (hw.empty()) return;
        std::string pp = hw + "/power1_average";
        if (read_num(pp) < 0) pp = hw + "/power1_input";
        while (!stop.load()) {
          double p = read_num(pp), c = read_num(hw + "/freq1_input");
          if (p > 0) { pw_sum += p * 1e-6; ck_sum += c > 0 ? c * 1e-6 : 0; ++pw_n; }
          std::this_thread::sleep_for(std::chrono::milliseconds(5));
        }
      });
      const int reps = 8;  // ~1.3-2.5 s per row
      hipEventRecord(e0);
      for (int r = 0; r < reps; ++r) launch20();
      hipEventRecord(e1); hipEventSynchronize(e1);
      stop = true; smp.join();
      float ms; hipEventElapsedTime(&ms, e0, e1);
      ms /= reps;
      // flops per block-iteration: 16x16x32: 16 MFMA x 16384 x 8 waves ; 32x32x16: 8 MFMA x 32768 x 8 waves -- equal; e4m3: 16 x 65536 x 8
      const double fl = 20.0 * nblk * (double)iters * 8 * 16 * (shape == 128 ? 65536.0 : 16384.0);
      const double rate = fl / (ms * 1e-3);
      const double pw = pw_n ? pw_sum / pw_n : 0, ck = pw_n ? ck_sum / pw_n : 0;
      printf("| %s | %s | %.1f | %.0f | %.0f | %.0f | %.3f |\n", mode == 0 ? "random" : "zero", shape == 16 ? "16x16x32 bf16 (16 acc)" : shape == 32 ? "32x32x16 bf16 (8 acc)" : "16x16x128 e4m3 scaled (16 acc)",
             ms, rate / 1e12, pw, ck, pw > 0 ? pw / rate * 1e12 : 0.0);
      fflush(stdout);
    }
  }
  return 0;
}
