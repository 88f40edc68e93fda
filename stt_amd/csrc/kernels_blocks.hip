// stt_amd/csrc/kernels_blocks.hip -- 8-bit floating point with one power of two per block of 128 values (gfx950).
//
// A matrix "in blocks" is e4m3 values q (4 exponent bits, 3 mantissa bits, largest 448, no infinity) in rows padded with zeros to a multiple of
// 128, and one byte s per block of 128 values along a row -- of one row (activations) or of 128 rows (weights): value = q * 2^(s - 127).
//   power of a block:  t = max |x| over its finite values; 2^e the smallest power with t <= 448 * 2^e, e >= -127; s = e + 127 (t = 0: s = 127)
//   value:             q = the e4m3 nearest to x * 2^-e, ties to even; NaN for what is not finite
// A power of two costs an e4m3 value nothing (its own exponent absorbs it, the block's largest value keeps between 224 and 448 of the range) and
// makes quantisation exact arithmetic but for the one rounding to 3 mantissa bits: the same bits on every path, fused or not.
//
//   product:           y[m][n] = epi(sum_k x[m][k] w[n][k] + bias[n]), epi: nothing or min(max(y, 0), clip); NaN stays NaN
//
// The product runs on v_mfma_f32_16x16x32_bf16: v_cvt_scalef32_pk_bf16_fp8 turns two e4m3 values times their block's power into two bf16 values
// without rounding (4 significand bits, an 8-bit exponent), so the scales cost no arithmetic of their own and the sums of all blocks stay in one f32
// accumulator.  The 8-bit matrix instructions (v_mfma_scale_f32_16x16x128_f8f6f4, v_mfma_f32_16x16x32_fp8_fp8) would be twice as fast, but do not
// keep 32 bits: products far below the largest ones they are added to lose bits.  Measured over 2048 products of values of all magnitudes, error
// relative to the result: 5e-5 on either of them, 3e-7 on the bf16 form; clipped activations by normal weights 1e-5 against 4e-8
// (benchmarks/blocks_sums_probe.hip, profiles/blocks_sums.txt), which four layers in blocks one behind the other turned into 1.5 % of the result.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <mutex>
#include <type_traits>

#include "kernels.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) unsigned char lds_u8;
typedef const __attribute__((address_space(1))) void gvoid_c;

constexpr int kUnit = 127;      // the byte of 2^0

template <int T> struct Elem;
template <> struct Elem<BLOCKS_F32> { typedef float type; };
template <> struct Elem<BLOCKS_F16> { typedef _Float16 type; };
template <> struct Elem<BLOCKS_BF16> { typedef unsigned short type; };

__device__ __forceinline__ float bf16_f32(unsigned short v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ unsigned short f32_bf16(float v) { return __builtin_bit_cast(unsigned short, (__bf16)v); }   // nearest, ties to even; NaN stays NaN
template <int T> __device__ __forceinline__ float load1(const typename Elem<T>::type* p) {
  if constexpr (T == BLOCKS_BF16) return bf16_f32(*p);
  else return (float)*p;
}
template <int T> __device__ __forceinline__ void store1(typename Elem<T>::type* p, float v) {
  if constexpr (T == BLOCKS_BF16) *p = f32_bf16(v);
  else *p = (typename Elem<T>::type)v;
}
// eight values from column `col` of a row of `cols`; zeros behind its end.  vec: 16-byte accesses are aligned (checked on the host)
template <int T> __device__ __forceinline__ void load8(float v[8], const typename Elem<T>::type* row, int col, int cols, bool vec) {
  if (vec && col + 8 <= cols) {
    if constexpr (T == BLOCKS_F32) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(row + col), b = *reinterpret_cast<const f32x4*>(row + col + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    } else if constexpr (T == BLOCKS_F16) {
      const f16x8 a = *reinterpret_cast<const f16x8*>(row + col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
    } else {
      const u16x8 a = *reinterpret_cast<const u16x8*>(row + col);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = bf16_f32(a[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < cols ? load1<T>(row + col + i) : 0.0f;
  }
}
template <int T> __device__ __forceinline__ void store8(const float v[8], typename Elem<T>::type* row, int col, int cols, bool vec) {
  if (vec && col + 8 <= cols) {
    if constexpr (T == BLOCKS_F32) {
      *reinterpret_cast<f32x4*>(row + col) = (f32x4){v[0], v[1], v[2], v[3]};
      *reinterpret_cast<f32x4*>(row + col + 4) = (f32x4){v[4], v[5], v[6], v[7]};
    } else {
      u16x8 a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = T == BLOCKS_BF16 ? f32_bf16(v[i]) : __builtin_bit_cast(unsigned short, (_Float16)v[i]);
      *reinterpret_cast<u16x8*>(row + col) = a;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) if (col + i < cols) store1<T>(row + col + i, v[i]);
  }
}

// Largest magnitude as bits: the order of the bits is the order of the magnitudes, infinities and NaN above all finite values.  `top` over a block is
// first taken over everything; only where that turns out not to be finite (kInf and up) is the block looked through again for its finite values.
constexpr unsigned kInf = 0x7f800000u;
__device__ __forceinline__ unsigned mag_(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ unsigned finite_mag_(float v) {
  asm volatile("" : "+v"(v));          // (the rare second look: without this the compiler keeps the magnitudes of the first one in as many registers)
  const unsigned u = mag_(v);
  return u < kInf ? u : 0u;
}
template <int N> __device__ __forceinline__ unsigned top_of_(const float (&v)[N], bool all) {
  unsigned t = 0;
  if (all) {
#pragma unroll
    for (int i = 0; i < N; ++i) t = max(t, mag_(v[i]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) t = max(t, finite_mag_(v[i]));
  }
  return t;
}
// The byte of a block whose largest finite magnitude is `top`: 448 = 1.75 * 2^8, so its exponent field goes up by one where its mantissa is
// above 1.75 (the carry out of adding 0x1fffff), and down by 8.
__device__ __forceinline__ int scale_byte_(unsigned top) { return top == 0 ? kUnit : max((int)((top + 0x1fffffu) >> 23) - 8, 0); }
// The power of a scale byte as the conversions take it: the exponent field of an f32 (255 makes NaN).
__device__ __forceinline__ float power_(int byte) { return __uint_as_float((unsigned)byte << 23); }
// four values to four e4m3 bytes, v / power: ties to even, NaN for what is not finite (v_cvt_scalef32_pk_fp8_f32; |v| <= 448 * power otherwise)
__device__ __forceinline__ unsigned pack4_(float a, float b, float c, float d, float power) {
  s16x2 r = (s16x2){0, 0};
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, a, b, power, false);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, c, d, power, true);
  return __builtin_bit_cast(unsigned, r);
}

// ------------------------------------------------------------------------------------------- rows of 1 x 128
// A wave per four blocks of a row (one word of scale bytes), sixteen lanes a block, eight values a lane: one pass, 16 bytes a lane and load for 16-bit rows.
// HBM bounds it: 32000 x 2048 f16 in 37.7 us, 5.2 TB/s of what it reads and writes (a copy of 1 GiB: 5.1); f32, the same matrix each time, 55.3 us, 5.9.
template <int T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(BlocksQuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int quads = (a.cols + 511) >> 9;
  if (item >= a.rows * quads) return;
  const int64_t row = item / quads;
  const int kb = (int)(item - row * quads) * 4 + (lane >> 4), col = kb * 128 + (lane & 15) * 8;
  const int nb = (a.cols + 127) >> 7;
  float v[8];
  load8<T>(v, reinterpret_cast<const typename Elem<T>::type*>(a.x) + row * a.ldx, col, a.cols, a.vec != 0);
  unsigned top = top_of_(v, true);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
  if (__any(top >= kInf)) {
    top = top_of_(v, false);
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
  }
  const int byte = scale_byte_(top);
  const float power = power_(byte);
  if (kb < nb) {
    uint2 o;
    o.x = pack4_(v[0], v[1], v[2], v[3], power);
    o.y = pack4_(v[4], v[5], v[6], v[7], power);
    *reinterpret_cast<uint2*>(a.q + row * a.ldq + col) = o;
  }
  if ((lane & 15) == 0) a.scale[row * a.lds + kb] = (unsigned char)byte;
}

// ------------------------------------------------------------------------------------------- tiles of 128 x 128
// A workgroup per tile, the tile in registers between the search for its largest value and the conversion.  HBM: 8192 x 2048 f32 in 15.2 us, 5.5 TB/s; f16 9.9 us, 5.1.
template <int T>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(BlocksQuantArgs a) {
  __shared__ unsigned s_top[2][4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int kb = blockIdx.x, nb = (a.cols + 127) >> 7;
  const int64_t r0 = (int64_t)blockIdx.y * 128;
  if (kb >= nb) {                                    // padding of the row of scale bytes
    if (tid == 0) a.scale[(int64_t)blockIdx.y * a.lds + kb] = kUnit;
    return;
  }
  const int col = kb * 128 + (tid & 15) * 8, rl = tid >> 4;
  const typename Elem<T>::type* x = reinterpret_cast<const typename Elem<T>::type*>(a.x);
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + rl + 16 * i;
    if (row < a.rows) load8<T>(v[i], x + row * a.ldx, col, a.cols, a.vec != 0);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
  }
  auto tile_top = [&](int pass) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, top_of_(v[i], pass == 0));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = max(top, (unsigned)__shfl_xor((int)top, d));
    if (lane == 0) s_top[pass][tid >> 6] = top;
    __syncthreads();
    return max(max(s_top[pass][0], s_top[pass][1]), max(s_top[pass][2], s_top[pass][3]));
  };
  unsigned top = tile_top(0);
  if (top >= kInf) top = tile_top(1);                // (the same for every wave)
  const int byte = scale_byte_(top);
  const float power = power_(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + rl + 16 * i;
    if (row >= a.rows) break;
    uint2 o;
    o.x = pack4_(v[i][0], v[i][1], v[i][2], v[i][3], power);
    o.y = pack4_(v[i][4], v[i][5], v[i][6], v[i][7], power);
    *reinterpret_cast<uint2*>(a.q + row * a.ldq + col) = o;
  }
  if (tid == 0) a.scale[(int64_t)blockIdx.y * a.lds + kb] = (unsigned char)byte;
}

// ------------------------------------------------------------------------------------------- the way back
// As the rows kernel, the other way.  HBM: 32000 x 2048 to bf16 in 37.5 us, 5.3 TB/s, to f32 60, 5.4; 8192 x 2048 in tiles to f16 9.8, 5.1.
template <int T>
__global__ __launch_bounds__(256) void dequantize_kernel(BlocksDequantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int quads = (a.cols + 511) >> 9;
  if (item >= a.rows * quads) return;
  const int64_t row = item / quads;
  const int kb = (int)(item - row * quads) * 4 + (lane >> 4), col = kb * 128 + (lane & 15) * 8;
  if (col >= a.cols) return;
  const uint2 q = *reinterpret_cast<const uint2*>(a.q + row * a.ldq + col);
  const int byte = a.scale[(a.block_rows == 1 ? row : row >> 7) * a.lds + kb];
  float v[8];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int w = (int)(h ? q.y : q.x);
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[h * 4 + 0] = lo[0]; v[h * 4 + 1] = lo[1]; v[h * 4 + 2] = hi[0]; v[h * 4 + 3] = hi[1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = byte == 255 ? __uint_as_float(0x7fc00000u) : ldexpf(v[i], byte - 127);
  store8<T>(v, reinterpret_cast<typename Elem<T>::type*>(a.y) + row * a.ldy, col, a.cols, a.vec != 0);
}

// ------------------------------------------------------------------------------------------- the product
// sixteen e4m3 values times their power, as two operands of eight bf16
__device__ __forceinline__ void expand_(const i32x4& q, float power, bf16x8 f[2]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * h + i], power, false);
      const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)q[2 * h + i], power, true);
      f[h][4 * i] = lo[0]; f[h][4 * i + 1] = lo[1]; f[h][4 * i + 2] = hi[0]; f[h][4 * i + 3] = hi[1];
    }
}
// min(max(v, 0), clip) that keeps NaN
__device__ __forceinline__ float epi_(float v, bool relu, float clip) { return relu ? __builtin_elementwise_minimum(__builtin_elementwise_maximum(v, 0.0f), clip) : v; }
// four values of row m, columns n .. n + 3
__device__ __forceinline__ void store4_(const BlocksDenseArgs& a, int64_t m, int n, const float v[4]) {
  const bool whole = a.vec != 0 && n + 4 <= a.N;
  if (a.y_type == BLOCKS_F32) {
    float* y = reinterpret_cast<float*>(a.y) + m * a.ldy + n;
    if (whole) *reinterpret_cast<f32x4*>(y) = (f32x4){v[0], v[1], v[2], v[3]};
    else
      for (int r = 0; r < 4; ++r) if (n + r < a.N) y[r] = v[r];
  } else {
    unsigned short* y = reinterpret_cast<unsigned short*>(a.y) + m * a.ldy + n;
    u16x4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = a.y_type == BLOCKS_BF16 ? f32_bf16(v[r]) : __builtin_bit_cast(unsigned short, (_Float16)v[r]);
    if (whole) *reinterpret_cast<u16x4*>(y) = o;
    else
      for (int r = 0; r < 4; ++r) if (n + r < a.N) y[r] = o[r];
  }
}

// One lane's part of x for a block along k: 32 values of a row, those of the lane's quarter of the block.  load() asks for them, values() hands them on
// as e4m3 with their scale byte -- rows that are not in blocks yet are quantised here, four lanes to a row.
template <int T> struct XQuarter {
  float v[32];
  __device__ __forceinline__ void load(const BlocksDenseArgs& a, int64_t m, int kb, int g) {
    const typename Elem<T>::type* row = reinterpret_cast<const typename Elem<T>::type*>(a.x) + m * a.ldx;
#pragma unroll
    for (int c = 0; c < 4; ++c) load8<T>(v + 8 * c, row, kb * 128 + g * 32 + 8 * c, a.K, a.xvec != 0);
  }
  __device__ __forceinline__ void values(i32x4 q[2], int& byte) {
    auto row_top = [&](bool all) {
      unsigned t = top_of_(v, all);
      t = max(t, (unsigned)__shfl_xor((int)t, 16));
      return max(t, (unsigned)__shfl_xor((int)t, 32));
    };
    unsigned top = row_top(true);
    if (__any(top >= kInf)) top = row_top(false);
    byte = scale_byte_(top);
    const float power = power_(byte);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i >> 2][i & 3] = (int)pack4_(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], power);
  }
};
template <> struct XQuarter<BLOCKS_E4M3> {
  i32x4 lo, hi;
  int s;
  __device__ __forceinline__ void load(const BlocksDenseArgs& a, int64_t m, int kb, int g) {
    const i32x4* p = reinterpret_cast<const i32x4*>(reinterpret_cast<const unsigned char*>(a.x) + m * a.ldx + kb * 128 + g * 32);
    lo = p[0]; hi = p[1];
    s = a.x_scale[m * a.ldxs + kb];
  }
  __device__ __forceinline__ void values(i32x4 q[2], int& byte) { q[0] = lo; q[1] = hi; byte = s; }
};

// Few rows: 16 output features by 16 MT rows per workgroup, the blocks along k dealt to its eight waves; operands straight from L2 / HBM into
// registers, the waves' sums meet in LDS (in the order of the waves: the same bits every time).  What bounds it is how much a compute unit takes in,
// some 30 GB/s of its part of w and of all of x: sixteen features a workgroup put 2048 of them on 128 of the 256 units (16 rows, k = 2048: 4.4 us, of which
// a launch is 2 and 64 KB a workgroup the rest; asking for two or four blocks ahead changed nothing).  A block of 128 features a workgroup, which could
// write y in blocks itself, is on 16 units and took 18.7 us; other numbers of features have not been tried.
template <int T, int MT>
__global__ __launch_bounds__(512) void dense_few_kernel(BlocksDenseArgs a) {
  constexpr int KW = 8;
  __shared__ f32x4 part[KW][MT][64];
  __shared__ __attribute__((aligned(16))) float s_bias[16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int li = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const int nb = (a.K + 127) >> 7;
  const int n = min(n0 + li, a.N - 1);
  const unsigned char* wp = a.w + (int64_t)n * a.ldw + g * 32;
  const unsigned char* ws = a.w_scale + (int64_t)(n >> 7) * a.ldws;
  if (tid < 16) s_bias[tid] = a.bias && n0 + tid < a.N ? a.bias[n0 + tid] : 0.0f;
  int64_t m[MT];
  f32x4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int64_t row = m0 + j * 16 + li;
    m[j] = row < a.M ? row : a.M - 1;
    acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  }
  for (int kb = wave; kb < nb; kb += KW) {
    const i32x4* p = reinterpret_cast<const i32x4*>(wp + (int64_t)kb * 128);
    const i32x4 lo = p[0], hi = p[1];
    const int wb = ws[kb];
    XQuarter<T> x[MT];
#pragma unroll
    for (int j = 0; j < MT; ++j) x[j].load(a, m[j], kb, g);
    const float sw = power_(wb);
    bf16x8 fw[4];
    expand_(lo, sw, fw);
    expand_(hi, sw, fw + 2);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      i32x4 q[2];
      int byte;
      x[j].values(q, byte);
      const float sx = power_(byte);
      bf16x8 fx[4];
      expand_(q[0], sx, fx);
      expand_(q[1], sx, fx + 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[k], fx[k], acc[j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) part[wave][j][lane] = acc[j];
  __syncthreads();
  // four features n0 + 4 j .. + 3 of row ml; consecutive lanes, consecutive features
  if (tid < MT * 64) {
    const int ml = tid >> 2, j = tid & 3, nq = n0 + j * 4;
    const int64_t row = m0 + ml;
    f32x4 s = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KW; ++k) s += part[k][ml >> 4][j * 16 + (ml & 15)];
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = epi_(s[r] + s_bias[j * 4 + r], a.relu != 0, a.clip);
    if (row < a.M) store4_(a, row, nq, v);
  }
}

// Sixteen rows of a wave's results in 8 or 16 bits through LDS (its own part of it), so that they leave 16 bytes a lane along a row: straight from the
// accumulators a store writes an eighth to a quarter of a line in each of sixteen rows.  Measured when it came, us straight | through LDS: 6144 x 2048 features in
// blocks 55.4 | 52.6, 6144 x 8192 f16 189 | 173; f32, half a line a row and store, is better off straight (2048 x 8192 61.2 | 65.8).
// Lane (li, g) holds 4 values = `Q` bytes at feature 16 i + 4 g of row li.
template <int NI, int Q> struct RowsOut {
  static constexpr int BYTES = NI * 4 * Q, PITCH = BYTES + 16, CHUNKS = BYTES / 16;      // of a row; the pitch keeps a column's rows on different banks
  lds_u8* buf;
  int li, g, lane;
  template <class V> __device__ __forceinline__ void put(int i, V v) {
    static_assert(sizeof(V) == Q, "four values");
    *reinterpret_cast<__attribute__((address_space(3))) V*>(buf + li * PITCH + (i * 4 + g) * Q) = v;
  }
  // row r of the sixteen goes to y + r * ld, rows < `rows`
  __device__ __forceinline__ void leave(unsigned char* y, int64_t ld, int64_t rows) {
#pragma unroll
    for (int t = 0; t < (16 * CHUNKS + 63) / 64; ++t) {
      const int idx = t * 64 + lane, r = idx / CHUNKS, c = idx % CHUNKS;
      if (CHUNKS < 4 && r >= 16) break;
      const i32x4 v = *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(buf + r * PITCH + c * 16);
      if (r < rows) *reinterpret_cast<i32x4*>(y + r * ld + c * 16) = v;
    }
  }
};

// The results of a wave that holds the features n0 + no .. of a block of 128, 16 NI of them, in the rows m0 + 16 j + li: acc[i][j][r] is feature
// n0 + no + 16 i + 4 g + r of row m0 + 16 j + li.  bias: the block's 128 biases in LDS.  A row's largest value in blocks is the largest of WN waves'
// (tops, in LDS: [WN][rows of the workgroup], row `ml` the lane's first).  buf: this wave's 16 * 272 bytes of LDS.
template <int NI, int MJ, int WN, int BM, int Y>
__device__ __forceinline__ void tile_results_as_(const BlocksDenseArgs& a, f32x4 (&acc)[NI][MJ], int64_t m0, int ml, int n0, int no, int lane, const float* bias, unsigned* tops, lds_u8* buf) {
  const int li = lane & 15, g = lane >> 4;
  const int64_t m = m0 + li;
  const bool whole = n0 + 128 <= a.N && (Y == BLOCKS_E4M3 || a.wide != 0);
  auto result = [&](int i, int j) {
    f32x4 v = acc[i][j] + *reinterpret_cast<const f32x4*>(bias + no + i * 16 + g * 4);
    if (a.relu) {
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = epi_(v[r], true, a.clip);
    }
    return v;
  };
  if constexpr (Y != BLOCKS_E4M3) {
    typedef typename Elem<Y>::type elem;
    if (Y != BLOCKS_F32 && whole) {
      RowsOut<NI, 8> out{buf, li, g, lane};
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const f32x4 v = result(i, j);
          u16x4 o;
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = Y == BLOCKS_BF16 ? f32_bf16(v[r]) : __builtin_bit_cast(unsigned short, (_Float16)v[r]);
          out.put(i, o);
        }
        out.leave(reinterpret_cast<unsigned char*>(a.y) + ((m0 + j * 16) * a.ldy + n0 + no) * 2, a.ldy * 2, a.M - (m0 + j * 16));
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < MJ; ++j) {
          const f32x4 v = result(i, j);
          const int n = n0 + no + i * 16 + g * 4;
          elem* const y = reinterpret_cast<elem*>(a.y) + (m + j * 16) * a.ldy + n;
          if (m + j * 16 < a.M) {
            if (Y == BLOCKS_F32 && whole) *reinterpret_cast<f32x4*>(y) = v;
            else {
#pragma unroll
              for (int r = 0; r < 4; ++r) if (n + r < a.N) store1<Y>(y + r, v[r]);
            }
          }
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
        acc[i][j] = result(i, j);
        if (!whole) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][r] = n0 + no + i * 16 + g * 4 + r < a.N ? acc[i][j][r] : 0.0f;
        }
      }
    unsigned top[MJ];
    auto row_tops = [&](bool all) {
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
        top[j] = 0;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) top[j] = max(top[j], all ? mag_(acc[i][j][r]) : finite_mag_(acc[i][j][r]));
        top[j] = max(top[j], (unsigned)__shfl_xor((int)top[j], 16));
        top[j] = max(top[j], (unsigned)__shfl_xor((int)top[j], 32));
      }
    };
    row_tops(true);
    bool odd = false;
#pragma unroll
    for (int j = 0; j < MJ; ++j) odd |= top[j] >= kInf;
    if (__any(odd)) row_tops(false);
    if constexpr (WN > 1) {
      if (g == 0) {
#pragma unroll
        for (int j = 0; j < MJ; ++j) tops[(no / (NI * 16)) * BM + ml + j * 16] = top[j];
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < MJ; ++j)
#pragma unroll
        for (int w = 0; w < WN; ++w) top[j] = max(top[j], tops[w * BM + ml + j * 16]);
    }
    RowsOut<NI, 4> out{buf, li, g, lane};
#pragma unroll
    for (int j = 0; j < MJ; ++j) {
      const int byte = scale_byte_(top[j]);
      const float power = power_(byte);
#pragma unroll
      for (int i = 0; i < NI; ++i) out.put(i, pack4_(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], power));
      out.leave(reinterpret_cast<unsigned char*>(a.y) + (m0 + j * 16) * a.ldy + n0 + no, a.ldy, a.M - (m0 + j * 16));
      if (no == 0 && m + j * 16 < a.M) {
        const int blk = n0 >> 7, last = ((a.N + 127) >> 7) - 1, pad = ((last + 4) & ~3) - 1;
        unsigned char* ys = a.y_scale + (m + j * 16) * a.ldys + blk;
        if (g == 0) ys[0] = (unsigned char)byte;
        if (blk == last && g > 0 && blk + g <= pad) ys[g] = kUnit;
      }
    }
  }
}

// Many rows: 128 features by BM rows per workgroup of four waves, WN of them along the features.  Both operands are staged as e4m3 through LDS by
// global_load_lds, KS = 64 or 128 values along k a step and STAGES = 3 stages: two steps in flight behind a counted wait, half the LDS traffic of staged
// bf16; the scale words of four blocks along k go the same way.  The 16-byte chunks of a staged row are permuted so that the sixteen lanes a ds_read_b128 is
// serviced in are on different banks: chunk c of a 64-byte row r at slot c ^ (row bit 3) * 2, of a 128-byte row at c ^ (r / 2 mod 8).
// Large tiles: a wave of the 256-row tile turns 12 fragments into bf16 for 64 products a step of 64 (96 conversions, which the other workgroup's
// products hide); two such workgroups fit a compute unit, three of the 128-row tile.  32000 x 8192 x 2048 to f32: 870 - 890 us by the card, 1234 - 1206 TFLOP/s, the matrix
// cores busy 58 % of the time; a library's bf16 product of that shape takes 919 us and writes half as much.  The clock falls with the data (the same
// call on operands of all ones: 13 % less): power, not one unit, is what is left.
// Small tiles: one wave a SIMD unit, so a step's latencies -- barrier, LDS, conversion, product -- add up, and more stages in flight change nothing (64
// rows, 64 values a step, 3 / 5 / 7 stages: 15.6 / 15.1 / 15.0 us at k = 2048): 128 values a step halve the barriers (14.5) and 32 rows the work (10.6).
template <int BM, int WN, int STAGES, int KS>
__global__ __launch_bounds__(256, 2) void dense_tile_kernel(BlocksDenseArgs a) {
  constexpr int BN = 128, WM = 4 / WN, NI = 8 / WN, MJ = BM / 16 / WM;
  constexpr int STAGE = (BN + BM) * KS, XROWS = BM < 64 ? 64 : BM, SCALES = (XROWS + 64) * 4, SUB = 128 / KS, AHEAD = (STAGES - 1) / SUB;
  constexpr int RPI = 1024 / KS, ITS = (BN + BM) / RPI / 4;      // a staging instruction of a wave covers sixteen rows
  __shared__ __attribute__((aligned(16))) float s_bias[BN];
  __shared__ unsigned s_tops[WN == 1 ? 1 : WN * BM];
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds_blocks[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), li = lane & 15, g = lane >> 4;
  const int wn = wave % WN, wm = wave / WN;
  lds_u8* const lds = (lds_u8*)lds_blocks;
  const int tiles_n = (a.N + BN - 1) / BN;
  int tile_n;
  int64_t tile_m;
  {  // workgroup i runs on XCD i % 8: every XCD takes a run of tiles, 1024 rows at a time over all features, so that what it works on at once shares rows and
     // features (32000 x 8192 x 2048: 868 us with 1024 rows, 867 and 902 with 512 and 2048)
    constexpr unsigned GM = 1024 / BM;      // (less than 2^24 tiles: checked on the host)
    const unsigned tn = (unsigned)tiles_n, tiles_m = (unsigned)((a.M + BM - 1) / BM), total = tn * tiles_m, per = (total + 7) / 8;
    const unsigned idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || idx >= total) return;
    const unsigned first = idx / (GM * tn) * GM, high = min(tiles_m - first, GM), rem = idx - first * tn;
    tile_n = (int)(rem / high);
    tile_m = first + rem % high;
  }
  const int n0 = tile_n * BN;
  const int64_t m0 = tile_m * BM;
  if (tid < BN) s_bias[tid] = a.bias && n0 + tid < a.N ? a.bias[n0 + tid] : 0.0f;      // (visible behind the first barrier below, which the wait for this write stands in front of)
  const int nb = (a.K + 127) >> 7;
  auto swizzle = [](int r) { return KS == 64 ? ((r >> 3) & 1) << 1 : (r >> 1) & 7; };
  const unsigned char* src[ITS];
#pragma unroll
  for (int i = 0; i < ITS; ++i) {
    const int r = (wave + 4 * i) * RPI + lane / (KS / 16), c = (lane & (KS / 16 - 1)) ^ swizzle(r);      // rows 0 .. 127: w, then x
    if (4 * i < BN / RPI) src[i] = a.w + (int64_t)min(n0 + r, a.N - 1) * a.ldw + c * 16;
    else {
      int64_t m = m0 + (r - BN);
      m = m < a.M ? m : a.M - 1;
      src[i] = reinterpret_cast<const unsigned char*>(a.x) + m * a.ldx + c * 16;
    }
  }
  auto stage = [&](int buf) {
#pragma unroll
    for (int i = 0; i < ITS; ++i) {
      __builtin_amdgcn_global_load_lds((gvoid_c*)src[i], (__attribute__((address_space(3))) void*)(lds + buf * STAGE + (wave + 4 * i) * 1024), 16, 0, 0);
      src[i] += KS;
    }
  };
  // the scale bytes of four blocks along k at a time: a word per row of x and, from the last wave, the word of w
  lds_u8* const lds_s = lds + STAGES * STAGE;
  const unsigned char* xs;
  {
    const int64_t m = m0 + wave * 64 + lane;
    xs = a.x_scale + (m < a.M ? m : a.M - 1) * a.ldxs;
  }
  const unsigned char* ws = a.w_scale + (int64_t)tile_n * a.ldws;
  auto stage_scales = [&](int kb) {
    lds_u8* const to = lds_s + (kb >> 2 & 1) * SCALES;
    if (wave < XROWS / 64) __builtin_amdgcn_global_load_lds((gvoid_c*)(xs + kb), (__attribute__((address_space(3))) void*)(to + wave * 256), 4, 0, 0);
    if (wave == 3) __builtin_amdgcn_global_load_lds((gvoid_c*)(ws + kb), (__attribute__((address_space(3))) void*)(to + XROWS * 4), 4, 0, 0);
  };
  const int off = li * KS + ((g ^ swizzle(li)) << 4);
  f32x4 acc[NI][MJ];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  float sw, sx[MJ];
  auto step = [&](int buf) {
#pragma unroll
    for (int h = 0; h < KS / 64; ++h) {
      const lds_u8* const bw = lds + buf * STAGE + wn * NI * 16 * KS + (off ^ (h << 6));
      const lds_u8* const bx = lds + buf * STAGE + (BN + wm * MJ * 16) * KS + (off ^ (h << 6));
      bf16x8 fx[MJ][2];
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
        const i32x4 q = *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(bx + j * 16 * KS);
        expand_(q, sx[j], fx[j]);
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const i32x4 q = *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(bw + i * 16 * KS);
        bf16x8 fw[2];
        expand_(q, sw, fw);
#pragma unroll
        for (int j = 0; j < MJ; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[k], fx[j][k], acc[i][j], 0, 0, 0);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");      // this wave has read the stage before it reaches the next barrier
  };
  auto scales = [&](int kb) {
    const lds_u8* const from = lds_s + (kb >> 2 & 1) * SCALES + (kb & 3);
    sw = power_(from[XROWS * 4]);
#pragma unroll
    for (int j = 0; j < MJ; ++j) sx[j] = power_(from[((wm * MJ + j) * 16 + li) * 4]);
  };
  // Behind wait and barrier the oldest step in flight has landed for every wave, and every wave is done reading the step before it, whose stage takes
  // the next step to be asked for.  (Scale words are not counted: with them in flight a wait waits for more than it has to.)
#define BLOCKS_ARRIVE(n)                                                                             \
  do {                                                                                               \
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");                                         \
    __builtin_amdgcn_s_barrier();                                                                    \
    __builtin_amdgcn_sched_barrier(0);                                                               \
  } while (0)
#pragma unroll
  for (int p = 0; p < AHEAD; ++p) {
    if (p < nb) {
      if ((p & 3) == 0) stage_scales(p);
#pragma unroll
      for (int u = 0; u < SUB; ++u) stage(SUB * p + u);
    }
  }
  // The barriers below wait for no LDS write by themselves, and one block along k in a step of 128 passes a single one before f32 results read the biases.
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  int cur = 0;
  for (int kb = 0; kb + AHEAD < nb; ++kb) {
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      BLOCKS_ARRIVE(ITS * (STAGES - 2));
      if (u == 0) {
        if ((kb + AHEAD & 3) == 0) stage_scales(kb + AHEAD);
        scales(kb);
      }
      stage(cur >= 1 ? cur - 1 : STAGES - 1);
      step(cur);
      cur = cur == STAGES - 1 ? 0 : cur + 1;
    }
  }
  auto last = [&](auto left) {                          // `left` blocks are left, all of them in flight
    constexpr int L = decltype(left)::value;
    if (L <= nb) {
      BLOCKS_ARRIVE(ITS * (SUB * L - 1));
      scales(nb - L);
      step(cur);
      cur = cur == STAGES - 1 ? 0 : cur + 1;
      if constexpr (SUB == 2) {
        BLOCKS_ARRIVE(ITS * (2 * L - 2));
        step(cur);
        cur = cur == STAGES - 1 ? 0 : cur + 1;
      }
    }
  };
  if constexpr (AHEAD > 1) last(std::integral_constant<int, 2>());
  last(std::integral_constant<int, 1>());
  static_assert((STAGES - 1) % SUB == 0 && AHEAD <= 2, "whole blocks in flight, and scale words of two groups of four");
#undef BLOCKS_ARRIVE
  if (a.y_type != BLOCKS_F32) __syncthreads();      // every wave is done reading the stages: LDS is the results' now
  const int64_t mw = m0 + wm * MJ * 16;
  const int ml = wm * MJ * 16 + li, no = wn * NI * 16;
  lds_u8* const buf = lds + wave * (16 * 272);
  switch (a.y_type) {
    case BLOCKS_F32: tile_results_as_<NI, MJ, WN, BM, BLOCKS_F32>(a, acc, mw, ml, n0, no, lane, s_bias, s_tops, buf); break;
    case BLOCKS_F16: tile_results_as_<NI, MJ, WN, BM, BLOCKS_F16>(a, acc, mw, ml, n0, no, lane, s_bias, s_tops, buf); break;
    case BLOCKS_BF16: tile_results_as_<NI, MJ, WN, BM, BLOCKS_BF16>(a, acc, mw, ml, n0, no, lane, s_bias, s_tops, buf); break;
    default: tile_results_as_<NI, MJ, WN, BM, BLOCKS_E4M3>(a, acc, mw, ml, n0, no, lane, s_bias, s_tops, buf); break;
  }
}

// Workgroups of four waves, one item (four blocks of a row) each; over two dimensions, because a dimension holds less than 2^32 threads.
constexpr int64_t kGridX = 1 << 20, kGridY = 65535;
int64_t row_groups_(int64_t rows, int cols) { return (rows * (((int64_t)cols + 511) / 512) + 3) / 4; }
dim3 rows_grid_(int64_t rows, int cols) {
  const int64_t blocks = row_groups_(rows, cols), x = blocks < kGridX ? blocks : kGridX;
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

template <int T, int MT>
void few_(const BlocksDenseArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((dense_few_kernel<T, MT>), dim3((a.N + 15) / 16, (unsigned)((a.M + 16 * MT - 1) / (16 * MT))), dim3(512), 0, st, a);
}
// Tiles of 16 rows per workgroup of the few-rows form, 0 where the tiled form is taken.  The former costs what its workgroups cost -- some 4.4 us up to 256 of
// them, then in proportion -- and more rows a workgroup read the weights fewer times; the latter takes 10.5 us at k = 2048 for the latency of its steps,
// but does more work in a given time.  So: the fewest rows that need at most 256 workgroups, or up to 32 rows where those need at most 512.
// Measured at k = 2048, us for 1, 2, 4 tiles a workgroup | tiled: 64 x 2048 features 6.6, 5.7, 7.8 | 10.6; 16 x 8192 6.5, 7.3, 8.6 | 10.5;
// 32 x 8192 10.6, 8.9, 10.3 | 10.6; 64 x 8192 18.9, 15.2, 13.5 | 10.9; 128 x 2048 10.8, 9.0, 8.2 | 10.6; 256 x 2048 19.2, 15.5, 13.6 | 10.8.
// Both parts of the work grow with k, so k is not asked for: at 128, 494 and 4096 the choice is within a tenth of the best (profiles/blocks_forms.txt) but for
// 128 x 2048 at k = 128 (3.8 | 3.2 with one tile) and the border of 29 features, 6144 rows: 9.7 | 8.8 with one tile, 24 | 17 at k = 4096.
int few_tiles_(int64_t M, int N) {
  const int64_t n = (N + 15) / 16;
  for (int mt = 1; mt <= 4; mt *= 2) {
    const int64_t groups = (M + 16 * mt - 1) / (16 * mt) * n;
    if (groups <= 256 || (M <= 16 * mt && mt <= 2 && groups <= 512)) return mt;
  }
  return 0;
}

// Rows of a tile: larger tiles do more work for what they stage, smaller ones fill the chip sooner.  Measured at k = 2048, f32 results, us for 32 / 64 / 128 / 256 rows:
// 512 x 2048 features 11.3 / 14.9 / 23.4 / 33.4 and 1024 x 2048 16.3 / 16.3 / 23.9 / 33.9 (256 and 512 tiles of 32 rows); 512 x 8192 28.9 / 22.7 / 25.9 /
// 35.4 and 2048 x 2048 30.0 / 23.5 / 27.0 / 35.6 (256 tiles of 128 rows); 1024 x 8192 53.8 / 40.1 / 36.2 / 36.6 and 6144 x 2048 74.2 / 55.9 / 50.4 /
// 54.1 (256 and 384 tiles of 256 rows: less than two workgroups for every compute unit); 2048 x 8192 97 / 75 / 65 / 59; 6144 x 8192 285 / 223 / 188 / 171.
// At k = 128, 494 and 4096 the choice is within a tenth of the best too (profiles/blocks_forms.txt).
int tile_rows_(int64_t M, int N) {
  const int64_t tiles_n = ((int64_t)N + 127) / 128;
  if (tiles_n * ((M + 31) / 32) <= 256) return 32;
  if (tiles_n * ((M + 127) / 128) <= 256) return 64;
  return tiles_n * ((M + 255) / 256) < 512 ? 128 : 256;
}
// Workgroups of the tiled form: a multiple of eight, one run of tiles for every XCD.
int64_t tile_groups_(int64_t M, int N, int rows) { return (((int64_t)N + 127) / 128 * ((M + rows - 1) / rows) + 7) / 8 * 8; }

template <int BM, int WN, int STAGES, int KS>
void tile_(const BlocksDenseArgs& a, hipStream_t st) {
  const int lds = max(STAGES * (128 + BM) * KS + 2 * (max(BM, 64) + 64) * 4, min(a.lds_floor, 128 * 1024));
  const int64_t grid = tile_groups_(a.M, a.N, BM);
  static std::once_flag once[16];
  int dev = 0;
  (void)hipGetDevice(&dev);
  std::call_once(once[dev & 15], []() { (void)hipFuncSetAttribute(reinterpret_cast<const void*>(dense_tile_kernel<BM, WN, STAGES, KS>), hipFuncAttributeMaxDynamicSharedMemorySize, 128 * 1024); });
  hipLaunchKernelGGL((dense_tile_kernel<BM, WN, STAGES, KS>), dim3((unsigned)grid), dim3(256), lds, st, a);
}

}  // namespace

bool blocks_rows_fit(int64_t rows, int cols) { return row_groups_(rows, cols) <= kGridX * kGridY; }
bool blocks_tiles_fit(int64_t rows) { return (rows + 127) / 128 <= kGridY; }

void launch_blocks_quantize(const BlocksQuantArgs& a, hipStream_t st) {
  if (a.rows < 1) return;
  if (a.block_rows == 1) {
    const dim3 grid = rows_grid_(a.rows, a.cols), block(256);
    switch (a.type) {
      case BLOCKS_F32: hipLaunchKernelGGL(quantize_rows_kernel<BLOCKS_F32>, grid, block, 0, st, a); break;
      case BLOCKS_F16: hipLaunchKernelGGL(quantize_rows_kernel<BLOCKS_F16>, grid, block, 0, st, a); break;
      default: hipLaunchKernelGGL(quantize_rows_kernel<BLOCKS_BF16>, grid, block, 0, st, a); break;
    }
  } else {
    const dim3 grid((unsigned)(a.cols + 511) / 512 * 4, (unsigned)((a.rows + 127) / 128)), block(256);
    switch (a.type) {
      case BLOCKS_F32: hipLaunchKernelGGL(quantize_tiles_kernel<BLOCKS_F32>, grid, block, 0, st, a); break;
      case BLOCKS_F16: hipLaunchKernelGGL(quantize_tiles_kernel<BLOCKS_F16>, grid, block, 0, st, a); break;
      default: hipLaunchKernelGGL(quantize_tiles_kernel<BLOCKS_BF16>, grid, block, 0, st, a); break;
    }
  }
}

void launch_blocks_dequantize(const BlocksDequantArgs& a, hipStream_t st) {
  if (a.rows < 1) return;
  const dim3 grid = rows_grid_(a.rows, a.cols), block(256);
  switch (a.type) {
    case BLOCKS_F32: hipLaunchKernelGGL(dequantize_kernel<BLOCKS_F32>, grid, block, 0, st, a); break;
    case BLOCKS_F16: hipLaunchKernelGGL(dequantize_kernel<BLOCKS_F16>, grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL(dequantize_kernel<BLOCKS_BF16>, grid, block, 0, st, a); break;
  }
}

namespace {

// How a call runs and what it keeps in the workspace: x in blocks where the product does not quantise it on the way, and y as f32 rows where it is wanted in
// blocks from the few-rows form, whose workgroups hold 16 of a block's 128 features.
struct Plan {
  int mt = 0;                          // few_tiles_()
  bool fused = false;                  // x is quantised by the few-rows form on the way: once for every 16 features
  int64_t ldq = 0, lds = 0, ldy = 0;   // of x in blocks, of y in f32
  size_t x_bytes = 0, y_bytes = 0;
  // Quantising on the way saves a launch (some 2 us) and costs in proportion to rows x features / 16: up to 256 workgroups of 16 rows.  Measured, us on the
  // way | first, f16, k = 2048: 16 x 2048 5.8 | 6.7; 32 x 2048 6.1 | 6.8; 64 x 2048 10.5 | 8.0; 1009 x 29 5.7 | 8.1; 2048 x 29 6.0 | 10.3; 4000 x 29 9.3 |
  // 14.8; f32, twice the bytes: 16 x 2048 7.2 | 6.7; 64 x 2048 12.1 | 8.1; 1009 x 29 7.7 | 8.3; 2048 x 29 11.9 | 10.3; 4000 x 29 19.8 | 14.5.  The border moves
  // with k: at 128 it would lie higher (64 x 2048 3.5 | 5.1), for f32 rows at 4096 lower (16 x 2048 11.7 | 9.1) -- profiles/blocks_forms.txt.
  Plan(int x_type, int y_type, int64_t M, int N, int K, int ordered) {
    mt = ordered ? 0 : few_tiles_(M, N);
    fused = x_type != BLOCKS_E4M3 && mt == 1 && (M + 15) / 16 * ((N + 15) / 16) <= 256;
    if (x_type != BLOCKS_E4M3 && !fused) {
      ldq = ((int64_t)K + 127) / 128 * 128; lds = ((int64_t)K + 511) / 512 * 4;
      x_bytes = ((size_t)M * (ldq + lds) + 15) / 16 * 16;
    }
    if (mt && y_type == BLOCKS_E4M3) {
      ldy = ((int64_t)N + 3) / 4 * 4;
      y_bytes = (size_t)M * ldy * 4;
    }
  }
};

}  // namespace

size_t blocks_dense_workspace(int x_type, int y_type, int64_t M, int N, int K, int ordered) {
  if (M < 1) return 0;
  const Plan p(x_type, y_type, M, N, K, ordered);
  return p.x_bytes + p.y_bytes;
}

bool blocks_dense_fits(int x_type, int y_type, int64_t M, int N, int K, int ordered) {
  if (M < 1) return true;
  const Plan p(x_type, y_type, M, N, K, ordered);
  if (p.x_bytes && !blocks_rows_fit(M, K)) return false;
  if (p.mt) return !p.y_bytes || blocks_rows_fit(M, N);
  return tile_groups_(M, N, tile_rows_(M, N)) * 256 <= 0xffffffffLL;
}

void launch_blocks_dense(const BlocksDenseArgs& args, void* workspace, hipStream_t st) {
  BlocksDenseArgs a = args;
  if (a.M < 1) return;
  const Plan p(a.x_type, a.y_type, a.M, a.N, a.K, a.ordered);
  if (p.x_bytes) {
    BlocksQuantArgs q{};
    q.x = a.x; q.ldx = a.ldx; q.rows = a.M; q.cols = a.K; q.type = a.x_type; q.block_rows = 1; q.vec = a.xvec;
    q.ldq = p.ldq; q.lds = p.lds; q.q = static_cast<unsigned char*>(workspace); q.scale = q.q + a.M * q.ldq;
    launch_blocks_quantize(q, st);
    a.x = q.q; a.x_scale = q.scale; a.ldx = q.ldq; a.ldxs = q.lds; a.x_type = BLOCKS_E4M3;
  }
  if (p.mt) {
    if (p.y_bytes) { a.y = static_cast<unsigned char*>(workspace) + p.x_bytes; a.y_type = BLOCKS_F32; a.ldy = p.ldy; a.vec = 1; }
    if (a.x_type == BLOCKS_F32) few_<BLOCKS_F32, 1>(a, st);
    else if (a.x_type == BLOCKS_F16) few_<BLOCKS_F16, 1>(a, st);
    else if (a.x_type == BLOCKS_BF16) few_<BLOCKS_BF16, 1>(a, st);
    else if (p.mt == 1) few_<BLOCKS_E4M3, 1>(a, st);
    else if (p.mt == 2) few_<BLOCKS_E4M3, 2>(a, st);
    else few_<BLOCKS_E4M3, 4>(a, st);
    if (p.y_bytes) {
      BlocksQuantArgs q{};
      q.x = a.y; q.ldx = a.ldy; q.rows = a.M; q.cols = a.N; q.type = BLOCKS_F32; q.block_rows = 1; q.vec = 1;
      q.q = static_cast<unsigned char*>(args.y); q.scale = args.y_scale; q.ldq = args.ldy; q.lds = args.ldys;
      launch_blocks_quantize(q, st);
    }
    return;
  }
  switch (tile_rows_(a.M, a.N)) {
    case 32: tile_<32, 4, 3, 128>(a, st); break;
    case 64: tile_<64, 2, 3, 128>(a, st); break;
    case 128: tile_<128, 1, 3, 64>(a, st); break;
    default: tile_<256, 1, 3, 64>(a, st); break;
  }
}
