// What the operators over the caller's device buffers share: the pool's addressing, the
// status bits, conversions between the 16-bit types and f32, and the host checks.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "../../include/yue2_cuda.h"
#include "common.cuh"
#include "engine.h"
#include "kernels.h"

namespace y2 {

// Yue2KvPool as kernels take it: 64-bit strides, so pools of any size are addressed.
struct PoolView {
  uint16_t* base;
  long long pages;
  long long page_stride;  // elements of one page (all layers)
  int blocks;             // layers * 2 * kv blocks of [64][dim] in a page
  int kv, dim;
};

Y2_DEV void status_or(int32_t* status, int bit) { atomicOr(status, bit); }

// 16-bit values of either type to and from f32 (round to nearest even)
template <bool F16>
Y2_DEV float lo16(uint32_t w) {
  if constexpr (F16) return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu)));
  return bf_lo(w);
}
template <bool F16>
Y2_DEV float hi16(uint32_t w) {
  if constexpr (F16) return __half2float(__ushort_as_half((unsigned short)(w >> 16)));
  return bf_hi(w);
}
template <bool F16>
Y2_DEV uint32_t pack16(float lo, float hi) {
  if constexpr (F16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_bf16x2(lo, hi);
}
template <bool F16>
Y2_DEV void unpack8(const uint4& w, float (&v)[8]) {
  v[0] = lo16<F16>(w.x), v[1] = hi16<F16>(w.x), v[2] = lo16<F16>(w.y), v[3] = hi16<F16>(w.y);
  v[4] = lo16<F16>(w.z), v[5] = hi16<F16>(w.z), v[6] = lo16<F16>(w.w), v[7] = hi16<F16>(w.w);
}

// ---- host checks; each returns 0 or the error of fail()
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int check_status(const int32_t* status) {
  if (!status || ((uintptr_t)status & 3)) return fail(YUE2_ERR_INVALID, "status must be a device int32");
  return 0;
}

// The pool's shape; `attention` restricts dim to the attention kernels' 64 and 128.
inline int check_pool(const Yue2KvPool* p, bool attention, PoolView& v) {
  if (!p || !p->base) return fail(YUE2_ERR_INVALID, "null KV pool");
  if (!aligned16(p->base)) return fail(YUE2_ERR_INVALID, "the KV pool must be 16-byte aligned");
  if (p->dtype != YUE2_DTYPE_BF16 && p->dtype != YUE2_DTYPE_F16)
    return fail(YUE2_ERR_INVALID, "KV pool values must be bf16 or f16");
  if (p->dim != 64 && p->dim != 128 && (attention || p->dim != 256))
    return fail(YUE2_ERR_INVALID, attention ? "attention takes a head dim of 64 or 128"
                                            : "the KV pool's head dim must be 64, 128 or 256");
  if (p->pages == 0 || p->pages > (1ull << 30) || p->layers == 0 || p->layers > 4096 || p->kv == 0 || p->kv > 1024)
    return fail(YUE2_ERR_INVALID, "KV pool shape out of range (pages <= 2^30, layers <= 4096, kv heads <= 1024)");
  v.base = static_cast<uint16_t*>(p->base);
  v.pages = (long long)p->pages;
  v.blocks = (int)(p->layers * 2 * p->kv);
  v.page_stride = (long long)v.blocks * kPageTokens * (long long)p->dim;
  v.kv = (int)p->kv;
  v.dim = (int)p->dim;
  return 0;
}

// A [rows, heads, dim] buffer: base, adjacent heads, row stride in elements. NULL is
// allowed only when it has no rows.
inline int check_rows(const void* p, uint64_t rows, uint64_t heads, uint64_t dim, uint64_t stride, const char* what) {
  if (rows == 0) return 0;
  if (!p || !aligned16(p))
    return fail(YUE2_ERR_INVALID, std::string(what) + " must be a 16-byte aligned device pointer");
  if (stride % 8 || stride < heads * dim || stride > (1ull << 32))
    return fail(YUE2_ERR_INVALID, std::string(what) + ": the row stride must be a multiple of 8 that holds every head");
  return 0;
}

// A list of `size`-byte entries (NULL passes: who needs one looks for it first).
inline int check_list(const void* p, size_t size, const char* what) {
  if ((uintptr_t)p & (size - 1))
    return fail(YUE2_ERR_INVALID, std::string(what) + " must be aligned to its " + std::to_string(size) + "-byte entries");
  return 0;
}

inline int check_heads(uint64_t heads, uint64_t kv) {
  if (heads == 0 || kv == 0 || heads > 1024 || kv > 1024 || heads % kv)
    return fail(YUE2_ERR_INVALID, "heads must be a multiple of kv, both in [1, 1024]");
  return 0;
}

// SMs of the current device.
inline int sm_count(int& sms) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return e == cudaSuccess ? 0 : cuda_fail(e, "device attributes");
}

inline int check_scale(float scale) {
  if (!std::isfinite(scale)) return fail(YUE2_ERR_INVALID, "scale must be finite");
  return 0;
}

}  // namespace y2
