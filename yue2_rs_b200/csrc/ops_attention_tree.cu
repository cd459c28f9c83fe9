// yue2_attention_tree: attention of drafted tokens over paged K/V. First form: one warp per
// (row, head) walks the visible keys with an online softmax in f32; lanes hold D/32 elements
// of q and of the output.
#include <cmath>
#include <string>

#include "ops.cuh"

namespace y2 {
namespace {

constexpr int kMaxSeqs = 1024;
constexpr int kMaxNodes = 64;

template <int D, bool F16>
struct RowState {
  static constexpr int DL = D / 32;
  float q[DL], o[DL], m = -INFINITY, l = 0.f;
  Y2_DEV static void load(const uint16_t* p, float (&v)[DL]) {
#pragma unroll
    for (int e = 0; e < DL; e += 2) {
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p + e);
      v[e] = lo16<F16>(w), v[e + 1] = hi16<F16>(w);
    }
  }
  Y2_DEV void begin(const uint16_t* p) {
    load(p, q);
#pragma unroll
    for (int e = 0; e < DL; ++e) o[e] = 0.f;
  }
  Y2_DEV void key(const uint16_t* kp, const uint16_t* vp, float scale) {
    float k[DL], v[DL], s = 0.f;
    load(kp, k);
    load(vp, v);
#pragma unroll
    for (int e = 0; e < DL; ++e) s = fmaf(q[e], k[e], s);
    s = warp_sum(s) * scale;
    const float mn = fmaxf(m, s);
    const float a = m == -INFINITY ? 0.f : expf(m - mn), w = expf(s - mn);
    m = mn;
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < DL; ++e) o[e] = fmaf(w, v[e], o[e] * a);
  }
  Y2_DEV void end(uint16_t* p) {
    const float inv = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
#pragma unroll
    for (int e = 0; e < DL; e += 2) *reinterpret_cast<uint32_t*>(p + e) = pack16<F16>(o[e] * inv, o[e + 1] * inv);
  }
};

// The sequence that holds `row`, or -1. Offsets outside [0, rows] or decreasing are reported.
Y2_DEV int find_seq(const int32_t* cu, int seqs, int rows, int row, int32_t* status) {
  int found = -1;
  for (int s = 0; s < seqs; ++s) {
    const int a = cu[s], b = cu[s + 1];
    if (a < 0 || b < a || b > rows) {
      status_or(status, YUE2_STATUS_RANGE);
      continue;
    }
    if (row >= a && row < b && found < 0) found = s;
  }
  return found;
}

struct TreeParams {
  const uint16_t* q;
  uint16_t* out;
  PoolView pool;
  const int32_t *table, *context, *cu;
  const uint64_t* mask;
  int32_t* status;
  long long q_stride, out_stride, table_pages;
  int seqs, rows, heads, layer;
  float scale;
};

template <int D, bool F16>
__global__ void __launch_bounds__(128) tree_kernel(const TreeParams p) {
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const int s = find_seq(p.cu, p.seqs, p.rows, row, p.status);
  if (s < 0) return;
  const int i = row - p.cu[s], nodes = p.cu[s + 1] - p.cu[s];
  const long long ctx = p.context[s];
  if (nodes > kMaxNodes || ctx < 0 || ctx + nodes > p.table_pages * kPageTokens) {
    status_or(p.status, YUE2_STATUS_RANGE);
    return;
  }
  const int32_t* table = p.table + s * p.table_pages;
  const uint64_t mask = p.mask ? p.mask[row] : ~0ull >> (63 - i);
  for (int h = threadIdx.x >> 5; h < p.heads; h += 4) {
    const int g = h / (p.heads / p.pool.kv);
    RowState<D, F16> r;
    r.begin(p.q + row * p.q_stride + h * D + lane * (D / 32));
    for (long long j = 0; j < ctx + nodes; ++j) {
      if (j >= ctx && !(mask >> (j - ctx) & 1)) continue;
      const long long page = table[j >> kPageLog2];
      if (page < 0 || page >= p.pool.pages) {
        status_or(p.status, YUE2_STATUS_PAGE);
        continue;
      }
      const uint16_t* kp = p.pool.base + page * p.pool.page_stride +
                           ((long long)(p.layer * 2) * p.pool.kv + g) * (kPageTokens * D) +
                           (j & (kPageTokens - 1)) * D + lane * (D / 32);
      r.key(kp, kp + (long long)p.pool.kv * (kPageTokens * D), p.scale);
    }
    r.end(p.out + row * p.out_stride + h * D + lane * (D / 32));
  }
}

}  // namespace
}  // namespace y2

using namespace y2;

extern "C" {

uint64_t yue2_attention_tree_workspace(uint64_t, uint64_t, uint64_t, uint64_t, const Yue2KvPool*) { return 0; }

int yue2_attention_tree(const void* q, uint64_t rows, uint64_t heads, uint64_t q_stride, const Yue2KvPool* pool,
                        uint64_t layer, const int32_t* table, uint64_t seqs, uint64_t table_pages,
                        const int32_t* context, const int32_t* cu, const uint64_t* mask, float scale, void* out,
                        uint64_t out_stride, void* workspace, uint64_t workspace_bytes, int32_t* status,
                        void* stream) {
  TreeParams p = {};
  int rc = check_pool(pool, true, p.pool);
  if (rc || (rc = check_heads(heads, pool->kv)) || (rc = check_status(status)) || (rc = check_scale(scale))) return rc;
  if (layer >= pool->layers) return fail(YUE2_ERR_INVALID, "layer outside the KV pool");
  if (seqs > (uint64_t)kMaxSeqs || table_pages > (1u << 24))
    return fail(YUE2_ERR_INVALID, "at most 1,024 sequences and 2^24 pages per table row");
  if (rows > (uint64_t)kMaxNodes * kMaxSeqs) return fail(YUE2_ERR_INVALID, "at most 64 drafted rows per sequence");
  if ((rc = check_rows(q, rows, heads, pool->dim, q_stride, "q")) ||
      (rc = check_rows(out, rows, heads, pool->dim, out_stride, "out")))
    return rc;
  if (seqs == 0 || rows == 0) return 0;
  if (!table || !context || !cu) return fail(YUE2_ERR_INVALID, "null page table, context or row offsets");
  (void)workspace;
  (void)workspace_bytes;
  p.q = (const uint16_t*)q;
  p.out = (uint16_t*)out;
  p.table = table;
  p.context = context;
  p.cu = cu;
  p.mask = mask;
  p.status = status;
  p.q_stride = (long long)q_stride;
  p.out_stride = (long long)out_stride;
  p.table_pages = (long long)table_pages;
  p.seqs = (int)seqs;
  p.rows = (int)rows;
  p.heads = (int)heads;
  p.layer = (int)layer;
  p.scale = scale;
  const dim3 grid((unsigned)rows);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f16 = pool->dtype == YUE2_DTYPE_F16;
  if (p.pool.dim == 64) {
    if (f16) tree_kernel<64, true><<<grid, 128, 0, st>>>(p);
    else tree_kernel<64, false><<<grid, 128, 0, st>>>(p);
  } else {
    if (f16) tree_kernel<128, true><<<grid, 128, 0, st>>>(p);
    else tree_kernel<128, false><<<grid, 128, 0, st>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail(e, "attention_tree launch");
}

}  // extern "C"
