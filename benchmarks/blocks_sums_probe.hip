// Which matrix instruction keeps 32 bits in a sum of e4m3 products: the two 8-bit ones against e4m3 values taken as bf16 (exact), one wave, 16 x 16 sums over
// k values, against the same sums in 64 bits.  Error relative to the results (root of summed squares).
//   hipcc --offload-arch=gfx950 -O3 -std=c++17 -Xclang -target-feature -Xclang -packed-fp32-ops blocks_sums_probe.hip -o /tmp/blocks_sums_probe && /tmp/blocks_sums_probe
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#define CHECK(e) do { const hipError_t r_ = (e); if (r_ != hipSuccess) { fprintf(stderr, "%s: %s\n", #e, hipGetErrorString(r_)); return 1; } } while (0)

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// a, b: [16][blocks * 128] e4m3; out [16][16].  One wave: lane (r, g) holds 32 values of a block, those from 32 g on, of row r of either operand.
__global__ __launch_bounds__(64) void sums(const unsigned char* a, const unsigned char* b, float* out, int blocks, int kind) {
  const int r = threadIdx.x & 15, g = threadIdx.x >> 4;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int kb = 0; kb < blocks; ++kb) {
    const int at = (r * blocks + kb) * 128 + g * 32;
    const i32x8 x = *reinterpret_cast<const i32x8*>(a + at), y = *reinterpret_cast<const i32x8*>(b + at);
    if (kind == 0) acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc, 0, 0, 0, 127, 0, 127);
    else if (kind == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long p = (long)(unsigned)x[2 * i + 1] << 32 | (unsigned)x[2 * i], q = (long)(unsigned)y[2 * i + 1] << 32 | (unsigned)y[2 * i];
        acc = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(p, q, acc, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        bf16x8 p, q;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x2 pl = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[2 * i + h], 1.0f, false), ph = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)x[2 * i + h], 1.0f, true);
          const bf16x2 ql = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)y[2 * i + h], 1.0f, false), qh = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)y[2 * i + h], 1.0f, true);
          p[4 * h] = pl[0]; p[4 * h + 1] = pl[1]; p[4 * h + 2] = ph[0]; p[4 * h + 3] = ph[1];
          q[4 * h] = ql[0]; q[4 * h + 1] = ql[1]; q[4 * h + 2] = qh[0]; q[4 * h + 3] = qh[1];
        }
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, acc, 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) out[(g * 4 + i) * 16 + r] = acc[i];
}

double value(int c) {
  const int e = c >> 3 & 15, m = c & 7;
  const double v = e == 0 ? std::ldexp(m, -9) : std::ldexp(8 + m, e - 10);
  return c & 128 ? -v : v;
}
int nearest(double v) {       // the code of the e4m3 nearest to |v| <= 448 (codes 0 .. 126 ascend)
  int lo = 0;
  while (lo < 126 && value(lo + 1) <= std::fabs(v)) ++lo;
  if (lo < 126 && value(lo + 1) - std::fabs(v) < std::fabs(v) - value(lo)) ++lo;
  return lo | (v < 0 ? 128 : 0);
}

int main() {
  const int blocks = 16, k = blocks * 128;
  const char* names[3] = {"v_mfma_scale_f32_16x16x128_f8f6f4", "v_mfma_f32_16x16x32_fp8_fp8", "v_mfma_f32_16x16x32_bf16"};
  const char* what[3] = {"all magnitudes", "one power of two", "clipped activations x normal weights"};
  unsigned char *da, *db;
  float* d;
  CHECK(hipMalloc(&da, 16 * k)); CHECK(hipMalloc(&db, 16 * k)); CHECK(hipMalloc(&d, 1024));
  for (int dist = 0; dist < 3; ++dist) {
    std::mt19937 rng(dist + 1);
    std::normal_distribution<double> normal;
    std::vector<unsigned char> a(16 * k), b(16 * k);
    for (int i = 0; i < 16 * k; ++i) {
      if (dist == 2) { a[i] = nearest(std::fmin(std::fmax(normal(rng), 0.0), 4.0) * 112.0); b[i] = nearest(std::fmax(-448.0, std::fmin(448.0, normal(rng) * 120.0))); }
      else for (auto* p : {&a, &b}) (*p)[i] = (rng() & 1) << 7 | (dist == 0 ? rng() % 15 : 7) << 3 | (rng() & 7);
    }
    CHECK(hipMemcpy(da, a.data(), 16 * k, hipMemcpyHostToDevice)); CHECK(hipMemcpy(db, b.data(), 16 * k, hipMemcpyHostToDevice));
    for (int kind = 0; kind < 3; ++kind) {
      sums<<<1, 64>>>(da, db, d, blocks, kind);
      float o[256];
      CHECK(hipGetLastError());
      CHECK(hipMemcpy(o, d, 1024, hipMemcpyDeviceToHost));
      double err = 0, all = 0;
      for (int i = 0; i < 16; ++i)
        for (int j = 0; j < 16; ++j) {
          double s = 0;
          for (int t = 0; t < k; ++t) s += value(a[i * k + t]) * value(b[j * k + t]);
          err += (o[i * 16 + j] - s) * (o[i * 16 + j] - s);
          all += s * s;
        }
      printf("%-36s %-36s %.2g\n", what[dist], names[kind], std::sqrt(err / all));
    }
  }
  return 0;
}
