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
// relative to the result: 5e-5 on either of them, 3e-7 on the bf16 form; on layer outputs 1e-5 against 4e-8, which four layers in blocks
// one behind the other turn into 1.5 % of the result.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <mutex>
#include <stdexcept>

#include "kernels.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
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
__device__ __forceinline__ unsigned short f32_bf16(float v) {      // nearest, ties to even; NaN stays NaN
  const unsigned u = __float_as_uint(v);
  return (u & 0x7fffffffu) > 0x7f800000u ? (unsigned short)((u >> 16) | 0x40u) : (unsigned short)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
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

__device__ __forceinline__ bool finite_(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ float top_(float top, float v) { return finite_(v) ? fmaxf(top, fabsf(v)) : top; }
// The byte of a block whose largest finite magnitude is `top`: 448 = 1.75 * 2^8, so the exponent field of `top` goes up by one where its
// mantissa is above 1.75 (the carry out of adding 0x1fffff), and down by 8.
__device__ __forceinline__ int scale_byte_(float top) {
  const unsigned u = __float_as_uint(top);
  const int e = (int)((u + 0x1fffffu) >> 23) - 8;
  return u == 0 ? kUnit : max(e, 0);
}
__device__ __forceinline__ float unscale_(int byte) { return __uint_as_float((unsigned)(254 - byte) << 23); }   // 2^(127 - byte): byte is at most 247
// four values to four e4m3 bytes (v_cvt_pk_fp8_f32: ties to even; |v * inv| <= 448)
__device__ __forceinline__ unsigned pack4_(float a, float b, float c, float d, float inv) {
  const float nan = __uint_as_float(0x7fc00000u);
  a = finite_(a) ? a * inv : nan; b = finite_(b) ? b * inv : nan; c = finite_(c) ? c * inv : nan; d = finite_(d) ? d * inv : nan;
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// ------------------------------------------------------------------------------------------- rows of 1 x 128
// A wave per four blocks of a row (one word of scale bytes), sixteen lanes a block, eight values a lane.
template <int T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(BlocksQuantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int quads = (a.cols + 511) >> 9;
  if (item >= a.rows * quads) return;
  const int64_t row = item / quads;
  const int kb = (int)(item - row * quads) * 4 + (lane >> 4), col = kb * 128 + (lane & 15) * 8;
  const int nb = (a.cols + 127) >> 7;
  float v[8];
  load8<T>(v, reinterpret_cast<const typename Elem<T>::type*>(a.x) + row * a.ldx, col, a.cols, a.vec != 0);
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = top_(top, v[i]);
#pragma unroll
  for (int d = 1; d < 16; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  const int byte = scale_byte_(top);
  const float inv = unscale_(byte);
  if (kb < nb) {
    uint2 o;
    o.x = pack4_(v[0], v[1], v[2], v[3], inv);
    o.y = pack4_(v[4], v[5], v[6], v[7], inv);
    *reinterpret_cast<uint2*>(a.q + row * a.ldq + col) = o;
  }
  if ((lane & 15) == 0) a.scale[row * a.lds + kb] = (unsigned char)byte;
}

// ------------------------------------------------------------------------------------------- tiles of 128 x 128
template <int T>
__global__ __launch_bounds__(256) void quantize_tiles_kernel(BlocksQuantArgs a) {
  __shared__ float s_top[4];
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
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + rl + 16 * i;
    if (row < a.rows) load8<T>(v[i], x + row * a.ldx, col, a.cols, a.vec != 0);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) top = top_(top, v[i][j]);
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
  if (lane == 0) s_top[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  const int byte = scale_byte_(top);
  const float inv = unscale_(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t row = r0 + rl + 16 * i;
    if (row >= a.rows) break;
    uint2 o;
    o.x = pack4_(v[i][0], v[i][1], v[i][2], v[i][3], inv);
    o.y = pack4_(v[i][4], v[i][5], v[i][6], v[i][7], inv);
    *reinterpret_cast<uint2*>(a.q + row * a.ldq + col) = o;
  }
  if (tid == 0) a.scale[(int64_t)blockIdx.y * a.lds + kb] = (unsigned char)byte;
}

// ------------------------------------------------------------------------------------------- the way back
template <int T>
__global__ __launch_bounds__(256) void dequantize_kernel(BlocksDequantArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
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
// The power of a scale byte as the conversion takes it: the exponent field of an f32 (255 makes NaN).
__device__ __forceinline__ float power_(int byte) { return __uint_as_float((unsigned)byte << 23); }
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
__device__ __forceinline__ float epi_(float v, bool relu, float clip) {
  if (!relu) return v;
  v = v < 0.0f ? 0.0f : v;
  return v > clip ? clip : v;
}
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

// One lane's part of x for the block kb: 32 values of row m, those of the lane's quarter of the block; sx their scale byte.
template <int T>
__device__ __forceinline__ void x_quarter_(const BlocksDenseArgs& a, int64_t m, int kb, int g, i32x4 q[2], int& sx) {
  const int col = kb * 128 + g * 32;
  if constexpr (T == BLOCKS_E4M3) {
    const i32x4* p = reinterpret_cast<const i32x4*>(reinterpret_cast<const unsigned char*>(a.x) + m * a.ldx + col);
    q[0] = p[0]; q[1] = p[1];
    sx = a.x_scale[m * a.ldxs + kb];
  } else {
    const typename Elem<T>::type* row = reinterpret_cast<const typename Elem<T>::type*>(a.x) + m * a.ldx;
    float v[32];
    float top = 0.0f;
#pragma unroll
    for (int c = 0; c < 4; ++c) load8<T>(v + 8 * c, row, col + 8 * c, a.K, a.xvec != 0);
#pragma unroll
    for (int i = 0; i < 32; ++i) top = top_(top, v[i]);
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    sx = scale_byte_(top);
    const float inv = unscale_(sx);
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i >> 2][i & 3] = (int)pack4_(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv);
  }
}

// Few rows: NTW tiles of 16 output features by 16 MT rows per workgroup, the blocks along k dealt to KW waves per tile; operands straight
// from L2 / HBM into registers, the waves' sums meet in LDS (in the order of the waves: the same bits every time).  Rows that are not in
// blocks yet are quantised in registers on the way.  NTW = 8 (a block of 128 features) where y is written in blocks.
template <int T, int MT, int NTW, int KW>
__global__ __launch_bounds__(64 * NTW * KW) void dense_few_kernel(BlocksDenseArgs a) {
  __shared__ f32x4 part[KW][NTW][MT][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nt = wave % NTW, kw = wave / NTW, li = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * (16 * NTW);
  const int64_t m0 = (int64_t)blockIdx.y * (16 * MT);
  const int nb = (a.K + 127) >> 7;
  const int n = min(n0 + nt * 16 + li, a.N - 1);
  const unsigned char* wp = a.w + (int64_t)n * a.ldw + g * 32;
  const unsigned char* ws = a.w_scale + (int64_t)(n >> 7) * a.ldws;
  f32x4 acc[MT];
#pragma unroll
  for (int j = 0; j < MT; ++j) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  for (int kb = kw; kb < nb; kb += KW) {
    const i32x4* p = reinterpret_cast<const i32x4*>(wp + (int64_t)kb * 128);
    const i32x4 lo = p[0], hi = p[1];
    const float sw = power_(ws[kb]);
    bf16x8 fw[4];
    expand_(lo, sw, fw);
    expand_(hi, sw, fw + 2);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      int64_t m = m0 + j * 16 + li;
      m = m < a.M ? m : a.M - 1;
      i32x4 q[2];
      int sx;
      x_quarter_<T>(a, m, kb, g, q, sx);
      bf16x8 fx[4];
      expand_(q[0], power_(sx), fx);
      expand_(q[1], power_(sx), fx + 2);
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[k], fx[k], acc[j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) part[kw][nt][j][lane] = acc[j];
  __syncthreads();
  // quad (m, j): four features n0 + 4 j .. + 3 of row m; consecutive lanes, consecutive features
  constexpr int Q = NTW * 4;
  for (int i = tid; i < MT * 16 * Q; i += 64 * NTW * KW) {
    const int ml = i / Q, j = i % Q;
    const int64_t m = m0 + ml;
    const int nq = n0 + j * 4;
    f32x4 s = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KW; ++k) s += part[k][j >> 2][ml >> 4][(j & 3) * 16 + (ml & 15)];
    float v[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = nq + r < a.N ? epi_(s[r] + (a.bias ? a.bias[nq + r] : 0.0f), a.relu != 0, a.clip) : 0.0f;
    if constexpr (NTW < 8) {
      if (m < a.M) store4_(a, m, nq, v);
    } else {
      float top = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) top = top_(top, v[r]);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
      const int byte = scale_byte_(top);
      if (m < a.M) {
        reinterpret_cast<unsigned*>(reinterpret_cast<unsigned char*>(a.y) + m * a.ldy + n0)[j] = pack4_(v[0], v[1], v[2], v[3], unscale_(byte));
        const int b = n0 >> 7, last = ((a.N + 127) >> 7) - 1, pad = ((last + 4) & ~3) - 1;
        if (j == 0) a.y_scale[m * a.ldys + b] = (unsigned char)byte;
        if (b == last && j > 0 && b + j <= pad) a.y_scale[m * a.ldys + b + j] = kUnit;
      }
    }
  }
}

// Many rows: BN features by BM rows per workgroup, a wave 128 features (a block of y) by 16 MJ rows; both operands' blocks of 128 along k staged
// through LDS by global_load_lds, two stages, one barrier a block.  Row r of a staged tile is 128 bytes, its 16-byte chunk c at slot
// c ^ (r & 7): a lane reads chunks g and g + 4 of its row (the same ones for both operands, so that the order along k inside a block
// does not matter), which keeps the sixteen lanes a ds_read_b128 is serviced in on different banks.
template <int BN, int BM, int WM>
__global__ __launch_bounds__(64 * (BN / 128) * WM) void dense_tile_kernel(BlocksDenseArgs a) {
  constexpr int WAVES = (BN / 128) * WM, MJ = BM / WM / 16;
  constexpr int STAGE = (BN + BM) * 128, ITS = (BN + BM) / 8 / WAVES;      // a staging instruction of a wave covers eight rows
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds_blocks[];
  lds_u8* const lds = (lds_u8*)lds_blocks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wn = wave / WM, wm = wave % WM, li = lane & 15, g = lane >> 4;
  const int tiles_n = (a.N + BN - 1) / BN;
  const int tile_n = (int)(blockIdx.x % tiles_n);
  const int64_t tile_m = blockIdx.x / tiles_n;
  const int n0 = tile_n * BN;
  const int64_t m0 = tile_m * BM;
  const int nb = (a.K + 127) >> 7;
  const unsigned char* src[ITS];
#pragma unroll
  for (int i = 0; i < ITS; ++i) {
    const int r = (wave * ITS + i) * 8 + (lane >> 3), c = (lane & 7) ^ (r & 7);      // rows 0 .. BN - 1: w, then x (BN is a multiple of 8)
    if (r < BN) src[i] = a.w + (int64_t)min(n0 + r, a.N - 1) * a.ldw + c * 16;
    else {
      int64_t m = m0 + (r - BN);
      m = m < a.M ? m : a.M - 1;
      src[i] = reinterpret_cast<const unsigned char*>(a.x) + m * a.ldx + c * 16;
    }
  }
  auto stage = [&](int buf, int kb) {
#pragma unroll
    for (int i = 0; i < ITS; ++i)
      __builtin_amdgcn_global_load_lds((gvoid_c*)(src[i] + (int64_t)kb * 128), (__attribute__((address_space(3))) void*)(lds + buf * STAGE + (wave * ITS + i) * 1024), 16, 0, 0);
  };
  const unsigned char* xs[MJ];
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    int64_t m = m0 + (wm * MJ + j) * 16 + li;
    m = m < a.M ? m : a.M - 1;
    xs[j] = a.x_scale + m * a.ldxs;
  }
  const unsigned char* ws = a.w_scale + (int64_t)min((n0 >> 7) + wn, (a.N - 1) >> 7) * a.ldws;
  const int c0 = (g ^ (li & 7)) * 16;
  f32x4 acc[8][MJ];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < MJ; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
  stage(0, 0);
  for (int kb = 0; kb < nb; ++kb) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();             // block kb has landed; every wave is done reading block kb - 1, whose stage takes kb + 1
    if (kb + 1 < nb) stage((kb + 1) & 1, kb + 1);
    const lds_u8* const bw = lds + (kb & 1) * STAGE + (wn * 128 + li) * 128;
    const lds_u8* const bx = lds + (kb & 1) * STAGE + (BN + wm * MJ * 16 + li) * 128;
    const float sw = power_(ws[kb]);
    float sx[MJ];
#pragma unroll
    for (int j = 0; j < MJ; ++j) sx[j] = power_(xs[j][kb]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {      // chunks g, then g + 4: 64 values along k each
      bf16x8 fx[MJ][2];
#pragma unroll
      for (int j = 0; j < MJ; ++j) {
        const i32x4 q = *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(bx + j * 2048 + (c0 ^ (h * 64)));
        expand_(q, sx[j], fx[j]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bf16x8 fw[2];
        const i32x4 q = *reinterpret_cast<const __attribute__((address_space(3))) i32x4*>(bw + i * 2048 + (c0 ^ (h * 64)));
        expand_(q, sw, fw);
#pragma unroll
        for (int j = 0; j < MJ; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[k], fx[j][k], acc[i][j], 0, 0, 0);
      }
    }
  }
  const int nw = n0 + wn * 128;                  // this wave's block of features
  if (nw >= a.N) return;
#pragma unroll
  for (int j = 0; j < MJ; ++j) {
    const int64_t m = m0 + (wm * MJ + j) * 16 + li;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int n = nw + i * 16 + g * 4;
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        v[r] = n + r < a.N ? epi_(acc[i][j][r] + (a.bias ? a.bias[n + r] : 0.0f), a.relu != 0, a.clip) : 0.0f;
        acc[i][j][r] = v[r];
        top = top_(top, v[r]);
      }
      if (a.y_type != BLOCKS_E4M3 && m < a.M) store4_(a, m, n, v);
    }
    if (a.y_type == BLOCKS_E4M3) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const int byte = scale_byte_(top);
      const float inv = unscale_(byte);
      if (m < a.M) {
        unsigned char* y = reinterpret_cast<unsigned char*>(a.y) + m * a.ldy + nw + g * 4;
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<unsigned*>(y + i * 16) = pack4_(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3], inv);
        const int b = nw >> 7, last = ((a.N + 127) >> 7) - 1, pad = ((last + 4) & ~3) - 1;
        if (g == 0) a.y_scale[m * a.ldys + b] = (unsigned char)byte;
        if (b == last && g > 0 && b + g <= pad) a.y_scale[m * a.ldys + b + g] = kUnit;
      }
    }
  }
}

template <int T, int MT>
void few_(const BlocksDenseArgs& a, hipStream_t st) {
  const unsigned gy = (unsigned)((a.M + 16 * MT - 1) / (16 * MT));
  if (a.y_type == BLOCKS_E4M3) hipLaunchKernelGGL((dense_few_kernel<T, MT, 8, 2>), dim3((a.N + 127) / 128, gy), dim3(1024), 0, st, a);
  else hipLaunchKernelGGL((dense_few_kernel<T, MT, 1, 8>), dim3((a.N + 15) / 16, gy), dim3(512), 0, st, a);
}
template <int T>
void few_rows_(const BlocksDenseArgs& a, hipStream_t st) {
  if (a.M <= 16) few_<T, 1>(a, st);
  else if (a.M <= 32) few_<T, 2>(a, st);
  else few_<T, 4>(a, st);
}

template <int BN, int BM, int WM>
void tile_(const BlocksDenseArgs& a, hipStream_t st) {
  constexpr int lds = 2 * (BN + BM) * 128;
  const int64_t tiles = (int64_t)((a.N + BN - 1) / BN) * ((a.M + BM - 1) / BM);
  if (tiles > 0x7fffffff) throw std::runtime_error("launch_blocks_dense: too many rows for one launch");
  static std::once_flag once[16];
  int dev = 0;
  (void)hipGetDevice(&dev);
  std::call_once(once[dev & 15], []() { (void)hipFuncSetAttribute(reinterpret_cast<const void*>(dense_tile_kernel<BN, BM, WM>), hipFuncAttributeMaxDynamicSharedMemorySize, lds); });
  hipLaunchKernelGGL((dense_tile_kernel<BN, BM, WM>), dim3((unsigned)tiles), dim3(64 * (BN / 128) * WM), lds, st, a);
}

}  // namespace

bool blocks_dense_fused(int64_t M) { return M <= 64; }

void launch_blocks_quantize(const BlocksQuantArgs& a, hipStream_t st) {
  if (a.rows < 1) return;
  const int64_t quads = (a.cols + 511) / 512;
  if (a.block_rows == 1) {
    const int64_t blocks = (a.rows * quads + 3) / 4;
    if (blocks > 0x7fffffff) throw std::runtime_error("launch_blocks_quantize: too many rows for one launch");
    const dim3 grid((unsigned)blocks), block(256);
    switch (a.type) {
      case BLOCKS_F32: hipLaunchKernelGGL(quantize_rows_kernel<BLOCKS_F32>, grid, block, 0, st, a); break;
      case BLOCKS_F16: hipLaunchKernelGGL(quantize_rows_kernel<BLOCKS_F16>, grid, block, 0, st, a); break;
      default: hipLaunchKernelGGL(quantize_rows_kernel<BLOCKS_BF16>, grid, block, 0, st, a); break;
    }
  } else {
    const int64_t tiles = (a.rows + 127) / 128;
    if (tiles > 65535) throw std::runtime_error("launch_blocks_quantize: too many rows for one launch");
    const dim3 grid((unsigned)quads * 4, (unsigned)tiles), block(256);
    switch (a.type) {
      case BLOCKS_F32: hipLaunchKernelGGL(quantize_tiles_kernel<BLOCKS_F32>, grid, block, 0, st, a); break;
      case BLOCKS_F16: hipLaunchKernelGGL(quantize_tiles_kernel<BLOCKS_F16>, grid, block, 0, st, a); break;
      default: hipLaunchKernelGGL(quantize_tiles_kernel<BLOCKS_BF16>, grid, block, 0, st, a); break;
    }
  }
}

void launch_blocks_dequantize(const BlocksDequantArgs& a, hipStream_t st) {
  if (a.rows < 1) return;
  const int64_t blocks = (a.rows * ((a.cols + 511) / 512) + 3) / 4;
  if (blocks > 0x7fffffff) throw std::runtime_error("launch_blocks_dequantize: too many rows for one launch");
  const dim3 grid((unsigned)blocks), block(256);
  switch (a.type) {
    case BLOCKS_F32: hipLaunchKernelGGL(dequantize_kernel<BLOCKS_F32>, grid, block, 0, st, a); break;
    case BLOCKS_F16: hipLaunchKernelGGL(dequantize_kernel<BLOCKS_F16>, grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL(dequantize_kernel<BLOCKS_BF16>, grid, block, 0, st, a); break;
  }
}

void launch_blocks_dense(const BlocksDenseArgs& a, hipStream_t st) {
  if (a.M < 1) return;
  if (blocks_dense_fused(a.M)) {
    switch (a.x_type) {
      case BLOCKS_F32: few_rows_<BLOCKS_F32>(a, st); break;
      case BLOCKS_F16: few_rows_<BLOCKS_F16>(a, st); break;
      case BLOCKS_BF16: few_rows_<BLOCKS_BF16>(a, st); break;
      default: few_rows_<BLOCKS_E4M3>(a, st); break;
    }
    return;
  }
  if (a.x_type != BLOCKS_E4M3) throw std::runtime_error("launch_blocks_dense: rows of this many have to be in blocks");
  // The 256-square tile does twice the work per byte it stages and wins from about one workgroup per compute unit on (2048 x 8192 x 2048:
  // 82 us against 88; 32000 x 8192 x 2048: 1336 against 1544); below that the 128-square one fills more of the chip (6144 x 2048 x 2048 is
  // 192 of the large tiles: three such layers and one of 8192 features 469 us against 484).
  if ((int64_t)((a.N + 255) / 256) * ((a.M + 255) / 256) >= 240) tile_<256, 256, 4>(a, st);
  else tile_<128, 128, 4>(a, st);
}
