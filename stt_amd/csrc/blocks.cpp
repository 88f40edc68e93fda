// stt_amd/csrc/blocks.cpp -- C entries of the block-scaled 8-bit operators (include/stt_amd.h: STTX_QuantizeBlocks & co.; kernels_blocks.hip).
//
// Device pointers in and out, on the caller's stream: a call checks its arguments, enqueues one or two kernels and returns.  It allocates
// nothing, waits for nothing and keeps nothing, so it may be recorded into a HIP graph and called from several threads at once.
#include <hip/hip_runtime.h>

#include <iostream>
#include <stdexcept>
#include <string>

#include "../../include/coqui-stt.h"
#include "../../include/stt_amd.h"
#include "engine.h"
#include "kernels.h"

namespace {

// What is wrong with a call, before anything was enqueued: STT_ERR_INVALID_SHAPE.
struct BadCall : std::runtime_error { using std::runtime_error::runtime_error; };
void want(bool ok, const char* what) { if (!ok) throw BadCall(what); }

template <class F> int entry(const char* name, F&& f) {
  try { f(); return STT_ERR_OK; }
  catch (const BadCall& e) { std::cerr << "stt_amd: " << name << ": " << e.what() << std::endl; return STT_ERR_INVALID_SHAPE; }
  catch (const std::exception& e) { std::cerr << "stt_amd: " << name << ": " << e.what() << std::endl; return STT_ERR_FAIL_RUN_SESS; }
}

// The stream's device for the time of a launch (a null stream is the current device's own).
struct OnDeviceOf {
  int before = -1;
  explicit OnDeviceOf(hipStream_t st) {
    if (!st) return;
    int cur = 0;
    hipDevice_t dev = 0;
    HIP_CHECK(hipGetDevice(&cur));
    HIP_CHECK(hipStreamGetDevice(st, &dev));
    if ((int)dev != cur) { HIP_CHECK(hipSetDevice((int)dev)); before = cur; }
  }
  ~OnDeviceOf() { if (before >= 0) (void)hipSetDevice(before); }
};

constexpr long long kMaxRows = 0x7fffffffLL, kMaxCols = 0x7fffffffLL - 511;
long long up(long long n, long long to) { return (n + to - 1) / to * to; }
bool aligned(const void* p, size_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
size_t elem(int type) { return type == STTX_F32 ? 4 : 2; }
bool plain(int type) { return type == STTX_F32 || type == STTX_F16 || type == STTX_BF16; }

void want_sizes(long long rows, long long cols) {
  want(rows >= 0 && rows <= kMaxRows, "rows out of range");
  want(cols >= 1 && cols <= kMaxCols, "columns out of range");
}
void want_plain(const void* p, int type, long long rows, long long cols, long long ld, bool written) {
  want(plain(type), "unknown element type");
  want(rows == 0 || p != nullptr, "null pointer");
  want(aligned(p, elem(type)), "pointer not aligned to its element type");
  want(ld >= (written ? cols : 0) || rows <= 1, "row stride out of range");
  want(ld >= 0 && ld <= (1LL << 40), "row stride out of range");
}
void want_blocks(const void* q, long long ldq, const void* scale, long long lds, long long rows, long long cols) {
  want(rows == 0 || (q != nullptr && scale != nullptr), "null pointer");
  want(aligned(q, 16) && ldq % 16 == 0, "e4m3 rows have to start at multiples of 16 bytes");
  want(ldq >= up(cols, 128) && ldq <= (1LL << 40), "e4m3 rows hold their columns rounded up to 128");
  want(aligned(scale, 4) && lds % 4 == 0, "rows of scale bytes have to start at multiples of 4 bytes");
  want(lds >= up(up(cols, 128) / 128, 4) && lds <= (1LL << 40), "rows of scale bytes hold their blocks rounded up to 4");
}
int vec16(const void* p, int type, long long ld) { return aligned(p, 16) && ld * (long long)elem(type) % 16 == 0; }

static_assert((int)STTX_F32 == BLOCKS_F32 && (int)STTX_F16 == BLOCKS_F16 && (int)STTX_BF16 == BLOCKS_BF16 && (int)STTX_E4M3 == BLOCKS_E4M3, "element types");

}  // namespace

extern "C" {

int STTX_QuantizeBlocks(const void* aX, int aType, long long aRows, long long aCols, long long aLdX, int aBlockRows, unsigned char* aQ, long long aLdQ,
                        unsigned char* aScale, long long aLdScale, void* aStream) {
  return entry("STTX_QuantizeBlocks", [&]() {
    want_sizes(aRows, aCols);
    want(aBlockRows == 1 || aBlockRows == 128, "blocks have 1 or 128 rows");
    want(aBlockRows == 1 ? blocks_rows_fit(aRows, (int)aCols) : blocks_tiles_fit(aRows), "too many rows for one launch");
    want_plain(aX, aType, aRows, aCols, aLdX, false);
    want_blocks(aQ, aLdQ, aScale, aLdScale, aRows, aCols);
    if (aRows == 0) return;
    const hipStream_t st = static_cast<hipStream_t>(aStream);
    OnDeviceOf on(st);
    BlocksQuantArgs a{};
    a.x = aX; a.q = aQ; a.scale = aScale; a.rows = aRows; a.ldx = aLdX; a.ldq = aLdQ; a.lds = aLdScale;
    a.cols = (int)aCols; a.type = aType; a.block_rows = aBlockRows; a.vec = vec16(aX, aType, aLdX);
    launch_blocks_quantize(a, st);
    HIP_CHECK(hipGetLastError());
  });
}

int STTX_DequantizeBlocks(const unsigned char* aQ, long long aLdQ, const unsigned char* aScale, long long aLdScale, long long aRows, long long aCols, int aBlockRows,
                          void* aY, int aType, long long aLdY, void* aStream) {
  return entry("STTX_DequantizeBlocks", [&]() {
    want_sizes(aRows, aCols);
    want(aBlockRows == 1 || aBlockRows == 128, "blocks have 1 or 128 rows");
    want(blocks_rows_fit(aRows, (int)aCols), "too many rows for one launch");
    want_blocks(aQ, aLdQ, aScale, aLdScale, aRows, aCols);
    want_plain(aY, aType, aRows, aCols, aLdY, true);
    if (aRows == 0) return;
    const hipStream_t st = static_cast<hipStream_t>(aStream);
    OnDeviceOf on(st);
    BlocksDequantArgs a{};
    a.q = aQ; a.scale = aScale; a.y = aY; a.rows = aRows; a.ldq = aLdQ; a.lds = aLdScale; a.ldy = aLdY;
    a.cols = (int)aCols; a.type = aType; a.block_rows = aBlockRows; a.vec = vec16(aY, aType, aLdY);
    launch_blocks_dequantize(a, st);
    HIP_CHECK(hipGetLastError());
  });
}

unsigned long long STTX_DenseBlocksWorkspace(int aXType, int aYType, long long aRows, long long aIn, long long aOut) {
  const auto type = [](int t) { return plain(t) || t == STTX_E4M3; };
  if (!type(aXType) || !type(aYType) || aRows < 1 || aRows > kMaxRows || aIn < 1 || aIn > kMaxCols || aOut < 1 || aOut > kMaxCols) return 0;
  return blocks_dense_workspace(aXType, aYType, aRows, (int)aOut, (int)aIn);
}

int STTX_DenseBlocks(const STTX_DenseBlocksArgs* aArgs) {
  return entry("STTX_DenseBlocks", [&]() {
    want(aArgs != nullptr, "null pointer");
    const STTX_DenseBlocksArgs& c = *aArgs;
    want_sizes(c.rows, c.in);
    want(c.out >= 1 && c.out <= kMaxCols, "columns out of range");
    if (c.x_type == STTX_E4M3) want_blocks(c.x, c.x_ld, c.x_scale, c.x_scale_ld, c.rows, c.in);
    else want_plain(c.x, c.x_type, c.rows, c.in, c.x_ld, false);
    want_blocks(c.w, c.w_ld, c.w_scale, c.w_scale_ld, c.out, c.in);
    want(aligned(c.bias, 4), "pointer not aligned to its element type");
    if (c.y_type == STTX_E4M3) want_blocks(c.y, c.y_ld, c.y_scale, c.y_scale_ld, c.rows, c.out);
    else want_plain(c.y, c.y_type, c.rows, c.out, c.y_ld, true);
    want(blocks_dense_fits(c.x_type, c.y_type, c.rows, (int)c.out, (int)c.in), "too many rows for one launch");
    want(c.relu_clip > 0.0f || c.relu_clip == 0.0f, "the clip of the ReLU is positive, or 0 for no ReLU");
    if (c.rows == 0) return;
    const unsigned long long need = STTX_DenseBlocksWorkspace(c.x_type, c.y_type, c.rows, c.in, c.out);
    want(need == 0 || (c.workspace != nullptr && aligned(c.workspace, 16) && c.workspace_bytes >= need), "workspace too small (STTX_DenseBlocksWorkspace) or not aligned to 16 bytes");
    const hipStream_t st = static_cast<hipStream_t>(c.stream);
    OnDeviceOf on(st);
    BlocksDenseArgs a{};
    a.x = c.x; a.x_scale = c.x_scale; a.w = c.w; a.w_scale = c.w_scale; a.bias = c.bias; a.y = c.y; a.y_scale = c.y_scale;
    a.M = c.rows; a.ldx = c.x_ld; a.ldxs = c.x_scale_ld; a.ldw = c.w_ld; a.ldws = c.w_scale_ld; a.ldy = c.y_ld; a.ldys = c.y_scale_ld;
    a.N = (int)c.out; a.K = (int)c.in; a.x_type = c.x_type; a.y_type = c.y_type; a.relu = c.relu_clip > 0.0f; a.clip = c.relu_clip;
    if (c.x_type != STTX_E4M3) a.xvec = vec16(c.x, c.x_type, c.x_ld);
    if (c.y_type != STTX_E4M3) { a.vec = aligned(c.y, 4 * elem(c.y_type)) && c.y_ld % 4 == 0; a.wide = vec16(c.y, c.y_type, c.y_ld); }
    launch_blocks_dense(a, c.workspace, st);
    HIP_CHECK(hipGetLastError());
  });
}

}  // extern "C"
