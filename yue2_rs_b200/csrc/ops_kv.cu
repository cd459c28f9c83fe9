// Operators that write the pages of a caller-owned K/V pool: QK norm + rotation + append,
// page copies and position moves. All three are bound by HBM (every value read once and
// written once); a page is [layers][K|V][kv] blocks of [64 positions][dim], so a position is
// layers * 2 * kv separate runs of dim * 2 bytes.
// Measured on one B200, captured, against the 6,544 GB/s of a plain copy: append of 8,192 rows of
// 40 heads of 128 with packed K out 32 us (5.8 TB/s), two rows of 12 heads 2.2 us; the tails of 8
// pages in 28 layers (58 MB) 11.6 us; accepting 8 of 64 nodes of 16 trees (29 MB in runs of 256
// bytes) 9.8 us: the chain of list, table and row, then three blocks of a warp one after the
// other with half of its row places empty; evicting 4,001 of 8,192 positions (918 MB) 147 us
// (6.2 TB/s).
#include <algorithm>
#include <string>

#include "ops.cuh"

namespace y2 {
namespace {

// ------------------------------------------------------------------ QK norm + rotation + append
// y = x * rsqrt(mean(x^2) + eps) * gain, then (a, b) = (y_i, y_{i + D/2}) becomes
// (a cos - b sin, b cos + a sin). One head is D/8 lanes, each with 4 elements of the first
// half and their 4 partners of the second (two 8-byte loads and stores), so that the
// rotation needs no exchange between lanes: the arithmetic, not only the bytes, bounds this
// pass. One CTA per row: its groups of D/8 lanes take the row's heads in turn and keep the
// row's cos and sin and the gains in registers.
struct AppendParams {
  const uint16_t* qkv;
  uint16_t *q_out, *k_out;
  const float *q_norm, *k_norm, *cos, *sin;
  const int32_t* positions;
  const int64_t* slots;
  int32_t* status;
  PoolView pool;
  long long qkv_stride, q_stride, k_stride, table_rows;
  int heads, layer;
  float eps;
};

// 8,192 rows of 40 heads of 128, captured: 31.4 us with 64 threads, 33.9 with 128, 41.5 with 256 (two rows
// alone: 3.4, 2.3 and 2.0).
constexpr int kAppendThreads = 64;

Y2_DEV void load4(const float* p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}

// UNROLL heads of a group are loaded before the row's position, which the loads of cos and sin
// wait for, is known. The gains stay in registers: read again for every head they kept L1
// 80% busy and took a third of the pass.
template <int D, bool F16, int UNROLL>
__global__ void __launch_bounds__(kAppendThreads) qk_rope_append_kernel(const AppendParams p) {
  constexpr int L = D / 8;                     // lanes per head
  constexpr int GROUPS = kAppendThreads / L;   // heads in flight
  const long long row = blockIdx.x;
  const int group = threadIdx.x / L, l = threadIdx.x % L;
  const int kv = p.pool.kv, total = p.heads + 2 * kv;
  const int pos = p.positions[row];
  const long long slot = p.slots[row];
  const uint16_t* src = p.qkv + row * p.qkv_stride + l * 4;
  float c[4], s[4], gq[8], gk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) gq[e] = gk[e] = 1.f;
  if (p.q_norm) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float a[4], b[4];
      load4(p.q_norm + half * (D / 2) + l * 4, a);
      load4(p.k_norm + half * (D / 2) + l * 4, b);
#pragma unroll
      for (int e = 0; e < 4; ++e) gq[4 * half + e] = a[e], gk[4 * half + e] = b[e];
    }
  }
  const bool inside = pos >= 0 && pos < p.table_rows;
  const bool store = slot >= 0 && (slot >> kPageLog2) < p.pool.pages;
  uint16_t* page = p.pool.base + (store ? (slot >> kPageLog2) * p.pool.page_stride : 0) +
                   (long long)p.layer * 2 * kv * (kPageTokens * D) + (slot & (kPageTokens - 1)) * D + l * 4;
  for (int h0 = group; h0 - group < total; h0 += GROUPS * UNROLL) {
    uint2 lo[UNROLL], hi[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * GROUPS;
      lo[u] = hi[u] = make_uint2(0, 0);
      if (h < total) {
        lo[u] = *reinterpret_cast<const uint2*>(src + (long long)h * D);
        hi[u] = *reinterpret_cast<const uint2*>(src + (long long)h * D + D / 2);
      }
    }
    if (h0 == group) {
      if (!inside || (slot >= 0 && !store)) {
        if (threadIdx.x == 0) status_or(p.status, inside ? YUE2_STATUS_PAGE : YUE2_STATUS_RANGE);
        if (!inside) return;
      }
      load4(p.cos + (long long)pos * (D / 2) + l * 4, c);
      load4(p.sin + (long long)pos * (D / 2) + l * 4, s);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * GROUPS;
      const bool is_q = h < p.heads, is_v = h >= p.heads + kv;
      const bool copies = __all_sync(0xffffffffu, is_v);  // a warp of value heads only copies
      if (!copies) {
        float a[4] = {lo16<F16>(lo[u].x), hi16<F16>(lo[u].x), lo16<F16>(lo[u].y), hi16<F16>(lo[u].y)};
        float b[4] = {lo16<F16>(hi[u].x), hi16<F16>(hi[u].x), lo16<F16>(hi[u].y), hi16<F16>(hi[u].y)};
        if (p.q_norm) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) ss = fmaf(b[e], b[e], fmaf(a[e], a[e], ss));
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float scale = rsqrtf(ss * (1.0f / D) + p.eps);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] *= scale * (is_q ? gq[e] : gk[e]);
            b[e] *= scale * (is_q ? gq[4 + e] : gk[4 + e]);
          }
        }
        float y[4], z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[e] = a[e] * c[e] - b[e] * s[e];
          z[e] = b[e] * c[e] + a[e] * s[e];
        }
        if (!is_v) {
          lo[u] = make_uint2(pack16<F16>(y[0], y[1]), pack16<F16>(y[2], y[3]));
          hi[u] = make_uint2(pack16<F16>(z[0], z[1]), pack16<F16>(z[2], z[3]));
        }
      }
      if (h >= total) continue;
      auto put = [&](uint16_t* to) {
        *reinterpret_cast<uint2*>(to) = lo[u];
        *reinterpret_cast<uint2*>(to + D / 2) = hi[u];
      };
      if (is_q) {
        put(p.q_out + row * p.q_stride + (long long)h * D + l * 4);
      } else {
        const int j = h - p.heads;  // K heads then V heads, as the pool's blocks of a layer
        if (!is_v && p.k_out) put(p.k_out + row * p.k_stride + (long long)j * D + l * 4);
        if (store) put(page + (long long)j * (kPageTokens * D));
      }
    }
  }
}

// The heads of a group are loaded together where they are up to three, otherwise five at a time. 8,192
// rows, captured, with 1 / 2 / 3 / 5 loaded together (8 for the last): one head a group (4 + 4 of 64)
// 6.3 / 6.5 / 6.9 / 7.7 us, two (4 + 4 of 128) 11.9 / 10.7 / 10.9 / -, three (8 + 4 of 128)
// 16.0 / 15.2 / 13.4 / 14.4, eight (16 + 16) 35.4 / 30.1 / 28.7 / 27.6 (29.3), ten (24 + 16) 42.4 / 35.5
// / 34.2 / 31.4 (38.4).
template <int D, bool F16>
void launch_append(const AppendParams& p, unsigned rows, cudaStream_t st) {
  constexpr int GROUPS = kAppendThreads / (D / 8);
  const int rounds = (p.heads + 2 * p.pool.kv + GROUPS - 1) / GROUPS;
  if (rounds <= 1) qk_rope_append_kernel<D, F16, 1><<<rows, kAppendThreads, 0, st>>>(p);
  else if (rounds == 2) qk_rope_append_kernel<D, F16, 2><<<rows, kAppendThreads, 0, st>>>(p);
  else if (rounds == 3) qk_rope_append_kernel<D, F16, 3><<<rows, kAppendThreads, 0, st>>>(p);
  else qk_rope_append_kernel<D, F16, 5><<<rows, kAppendThreads, 0, st>>>(p);
}

// ------------------------------------------------------------------ page copy
// CTA (block b, pair i): the first count[i] positions of one [64][dim] block, 32 KB at most,
// four 16-byte words of a thread in flight.
constexpr int kMoveThreads = 256;

__global__ void __launch_bounds__(kMoveThreads) kv_copy_kernel(PoolView pool, const int32_t* src, const int32_t* dst,
                                                               const int32_t* count, int32_t* status) {
  const long long i = blockIdx.y;
  const long long a = src[i], b = dst[i];
  const int n = count ? count[i] : kPageTokens;
  if (a < 0 || a >= pool.pages || b < 0 || b >= pool.pages || n < 0 || n > kPageTokens) {
    if (threadIdx.x == 0 && blockIdx.x == 0)
      status_or(status, n < 0 || n > kPageTokens ? YUE2_STATUS_RANGE : YUE2_STATUS_PAGE);
    return;
  }
  const long long block = (long long)blockIdx.x * kPageTokens * pool.dim;
  const uint4* from = reinterpret_cast<const uint4*>(pool.base + a * pool.page_stride + block);
  uint4* to = reinterpret_cast<uint4*>(pool.base + b * pool.page_stride + block);
  const int words = n * pool.dim / 8;
  for (int w0 = threadIdx.x; w0 < words; w0 += 4 * kMoveThreads) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (w0 + u * kMoveThreads < words) v[u] = from[w0 + u * kMoveThreads];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (w0 + u * kMoveThreads < words) to[w0 + u * kMoveThreads] = v[u];
  }
}

// ------------------------------------------------------------------ position moves
// A warp moves rows of dim * 2 bytes, kMoveRows of them at a time in list order, in a few of the
// page's blocks: the list and the page tables are looked up once for all of those. In place,
// keep is strictly increasing and keep[i] >= begin + i, so a write lands on no position that a
// later entry reads; an earlier entry's read is of the same or an earlier group, which the
// warp has finished (or orders with __syncwarp) before it writes. Out of place nothing read is
// written and the groups of a list go to several CTAs.
struct GatherParams {
  PoolView pool;
  const int32_t *src_table, *dst_table, *begin, *cu, *keep;
  int32_t* status;
  long long src_pages, dst_pages, total;
  int per_warp;  // blocks of a page that a warp takes
};
constexpr int kMoveUnroll = 8;  // rows in flight per lane

template <int D>
__global__ void __launch_bounds__(kMoveThreads) kv_gather_kernel(const GatherParams p) {
  constexpr int L = D / 8;                         // lanes per row
  constexpr int ROWS = 32 / L * kMoveUnroll;       // rows of a group
  const int s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int block0 = (blockIdx.x * (kMoveThreads / 32) + warp) * p.per_warp, block1 = min(block0 + p.per_warp, p.pool.blocks);
  const bool in_place = p.dst_table == nullptr;
  const int first = p.cu[s], last = p.cu[s + 1], begin = p.begin[s];
  const bool reports = block0 == 0;  // one warp tells what is wrong with an entry
  if (first < 0 || last < first || last > p.total || begin < 0) {
    if (reports && lane == 0 && blockIdx.z == 0) status_or(p.status, YUE2_STATUS_RANGE);
    return;
  }
  const int32_t* src_row = p.src_table + (long long)s * p.src_pages;
  const int32_t* dst_row = in_place ? src_row : p.dst_table + (long long)s * p.dst_pages;
  const long long dst_pages = in_place ? p.src_pages : p.dst_pages;
  const int sub = lane / L, l = lane % L, n = last - first;
  for (int c0 = ROWS * blockIdx.z; c0 < n; c0 += ROWS * gridDim.z) {
    const uint16_t* from[kMoveUnroll];
    uint16_t* to[kMoveUnroll];
#pragma unroll
    for (int u = 0; u < kMoveUnroll; ++u) {
      const int i = c0 + u * (32 / L) + sub;
      to[u] = nullptr;
      from[u] = nullptr;
      if (i >= n) continue;
      const long long x = p.keep[first + i], y = (long long)begin + i;
      // the order that in-place moves rely on, for this entry and the one before it
      const bool order = !in_place || (x >= y && (i == 0 || p.keep[first + i - 1] < x));
      if (x < 0 || (x >> kPageLog2) >= p.src_pages || (y >> kPageLog2) >= dst_pages || !order) {
        if (reports && l == 0) status_or(p.status, YUE2_STATUS_RANGE);
        continue;
      }
      const long long a = src_row[x >> kPageLog2], b = dst_row[y >> kPageLog2];
      if (a < 0 || a >= p.pool.pages || b < 0 || b >= p.pool.pages) {
        if (reports && l == 0) status_or(p.status, YUE2_STATUS_PAGE);
        continue;
      }
      from[u] = p.pool.base + a * p.pool.page_stride + (x & (kPageTokens - 1)) * D + l * 8;
      to[u] = p.pool.base + b * p.pool.page_stride + (y & (kPageTokens - 1)) * D + l * 8;
    }
    for (int block = block0; block < block1; ++block) {
      const long long off = (long long)block * (kPageTokens * D);
      uint4 v[kMoveUnroll];
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u)
        if (to[u]) v[u] = *reinterpret_cast<const uint4*>(from[u] + off);
      __syncwarp();
#pragma unroll
      for (int u = 0; u < kMoveUnroll; ++u)
        if (to[u]) *reinterpret_cast<uint4*>(to[u] + off) = v[u];
      __syncwarp();
    }
  }
}

}  // namespace
}  // namespace y2

using namespace y2;

extern "C" {

int yue2_qk_rope_append(const void* qkv, uint64_t rows, uint64_t heads, uint64_t qkv_stride, const float* q_norm,
                        const float* k_norm, float eps, const float* cos, const float* sin, uint64_t table_rows,
                        const int32_t* positions, const Yue2KvPool* pool, uint64_t layer, const int64_t* slots,
                        void* q_out, uint64_t q_stride, void* k_out, uint64_t k_stride, int32_t* status,
                        void* stream) {
  AppendParams p = {};
  int rc = check_pool(pool, false, p.pool);
  if (rc || (rc = check_status(status))) return rc;
  if (heads == 0 || heads > 1024 || rows > (uint64_t)INT32_MAX)
    return fail(YUE2_ERR_INVALID, "heads must be in [1, 1024] and rows below 2^31");
  if (layer >= pool->layers) return fail(YUE2_ERR_INVALID, "layer outside the KV pool");
  if ((rc = check_rows(qkv, rows, heads + 2 * pool->kv, pool->dim, qkv_stride, "qkv"))) return rc;
  if ((rc = check_rows(q_out, rows, heads, pool->dim, q_stride, "q_out"))) return rc;
  if (k_out && (rc = check_rows(k_out, rows, pool->kv, pool->dim, k_stride, "k_out"))) return rc;
  if (!q_norm != !k_norm || !aligned16(q_norm) || !aligned16(k_norm))
    return fail(YUE2_ERR_INVALID, "q_norm and k_norm go together and are 16-byte aligned");
  if (rows && (!positions || !slots || !cos || !sin || !aligned16(cos) || !aligned16(sin)))
    return fail(YUE2_ERR_INVALID, "positions, slots and 16-byte aligned cos and sin tables are needed");
  if (!(eps >= 0.f)) return fail(YUE2_ERR_INVALID, "eps must not be negative");
  if (rows == 0) return 0;
  if ((rc = check_list(positions, 4, "positions")) || (rc = check_list(slots, 8, "slots"))) return rc;
  p.qkv = (const uint16_t*)qkv;
  p.q_out = (uint16_t*)q_out;
  p.k_out = (uint16_t*)k_out;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.cos = cos;
  p.sin = sin;
  p.positions = positions;
  p.slots = slots;
  p.status = status;
  p.qkv_stride = (long long)qkv_stride;
  p.q_stride = (long long)q_stride;
  p.k_stride = (long long)k_stride;
  p.table_rows = (long long)(table_rows < (uint64_t)INT64_MAX ? table_rows : INT64_MAX);
  p.heads = (int)heads;
  p.layer = (int)layer;
  p.eps = eps;
  const bool f16 = pool->dtype == YUE2_DTYPE_F16;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
#define Y2_APPEND(DD)                                               \
  case DD:                                                          \
    if (f16) launch_append<DD, true>(p, (unsigned)rows, st);        \
    else launch_append<DD, false>(p, (unsigned)rows, st);           \
    break;
  switch (p.pool.dim) {
    Y2_APPEND(64)
    Y2_APPEND(128)
    Y2_APPEND(256)
  }
#undef Y2_APPEND
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail(e, "qk_rope_append launch");
}

int yue2_kv_copy(const Yue2KvPool* pool, const int32_t* src, const int32_t* dst, const int32_t* count, uint64_t n,
                 int32_t* status, void* stream) {
  PoolView v;
  int rc = check_pool(pool, false, v);
  if (rc || (rc = check_status(status))) return rc;
  if (n > 65535) return fail(YUE2_ERR_INVALID, "at most 65,535 page pairs per call");
  if (n && (!src || !dst)) return fail(YUE2_ERR_INVALID, "null page list");
  if (n == 0) return 0;
  if ((rc = check_list(src, 4, "src")) || (rc = check_list(dst, 4, "dst")) || (rc = check_list(count, 4, "count"))) return rc;
  kv_copy_kernel<<<dim3((unsigned)v.blocks, (unsigned)n), kMoveThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      v, src, dst, count, status);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail(e, "kv_copy launch");
}

int yue2_kv_gather(const Yue2KvPool* pool, const int32_t* src_table, uint64_t src_pages, const int32_t* dst_table,
                   uint64_t dst_pages, const int32_t* begin, const int32_t* cu, const int32_t* keep, uint64_t seqs,
                   uint64_t total, int32_t* status, void* stream) {
  GatherParams p = {};
  int rc = check_pool(pool, false, p.pool);
  if (rc || (rc = check_status(status))) return rc;
  if (seqs > 65535 || total > (uint64_t)INT32_MAX || src_pages > (1u << 26) || dst_pages > (1u << 26))
    return fail(YUE2_ERR_INVALID, "at most 65,535 sequences, 2^31 - 1 list entries and 2^26 pages per table row");
  if (seqs == 0 || total == 0) return 0;
  if (!src_table || !begin || !cu || !keep) return fail(YUE2_ERR_INVALID, "null table or list");
  if ((rc = check_list(src_table, 4, "src_table")) || (rc = check_list(dst_table, 4, "dst_table")) ||
      (rc = check_list(begin, 4, "begin")) || (rc = check_list(cu, 4, "cu")) || (rc = check_list(keep, 4, "keep")))
    return rc;
  p.src_table = src_table;
  p.dst_table = dst_table;
  p.begin = begin;
  p.cu = cu;
  p.keep = keep;
  p.status = status;
  p.src_pages = (long long)src_pages;
  p.dst_pages = (long long)dst_pages;
  p.total = (long long)total;
  // Out of place: a warp group per group of rows of the average list, at most 256 shares. A warp
  // takes several blocks, four at most, as long as that leaves about 16 warps for each SM.
  int sms = 0;
  if ((rc = sm_count(sms))) return rc;
  const uint64_t rows = 256 / pool->dim * kMoveUnroll;
  const uint64_t shares = dst_table ? std::min<uint64_t>(256, (total / seqs + rows - 1) / rows) : 1;
  const unsigned z = (unsigned)std::max<uint64_t>(1, shares);
  p.per_warp = (int)std::max<uint64_t>(1, std::min<uint64_t>(4, (uint64_t)p.pool.blocks * seqs * z / (16 * (uint64_t)sms)));
  const int per_cta = kMoveThreads / 32 * p.per_warp;
  const dim3 grid((unsigned)((p.pool.blocks + per_cta - 1) / per_cta), (unsigned)seqs, z);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (p.pool.dim) {
    case 64: kv_gather_kernel<64><<<grid, kMoveThreads, 0, st>>>(p); break;
    case 128: kv_gather_kernel<128><<<grid, kMoveThreads, 0, st>>>(p); break;
    case 256: kv_gather_kernel<256><<<grid, kMoveThreads, 0, st>>>(p); break;
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail(e, "kv_gather launch");
}

}  // extern "C"
