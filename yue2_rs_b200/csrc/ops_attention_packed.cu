// yue2_attention_packed: attention over whole packed sequences on the 5th-generation tensor
// cores.
//
// A unit of work is 256 query rows of one head of one sequence: two sides of 128 rows that
// share the stream of 128-key K and V tiles. Persistent CTAs (one per SM, 10 warps):
//   warps 0-3, 4-7  softmax of side 0 and 1, thread = row = TMEM lane: scores from TMEM, weights
//                   back to TMEM, the output at the end (softmax_settled and softmax_masked in ops_tc.cuh);
//   warp 8          issues the products: while side 0's softmax runs, the tensor cores do side 1's
//                   P.V and next scores, and the other way round (one warp for both keeps the
//                   sides in turn: with a warp each they fell into step, both in softmax and
//                   then both in products, a third slower). P.V starts when three quarters
//                   of the weights are there, so that the last quarter's exponentials run
//                   under it;
//   warp 9          picks the units, publishes them to the others and loads Q and the K, V ring by
//                   TMA.
// Units go out by block index from the highest down, dealt to the CTAs there and back (0..G-1,
// G-1..0, ..), found from the offsets on the device, so the host needs no lengths. With the causal
// mask that is longest first. Without it a unit's cost is its sequence's, so sequences of different
// lengths are dealt unevenly: 4,098 + 1,501 rows of 24 heads put 132 pairs of tiles on the busiest
// of 148 CTAs, with a mean of 100. Heads of one block are neighbours, so that a group's K and V
// come from L2.
//
// What bounds it: a pair of 128 x 128 tiles is 2,048 cycles of products and takes about 3,200; the
// rest is the product warp's own time between them (a wait that finds its barrier done still
// costs about 110 cycles) and the softmax, whose two sides share the special-function units.
// Measured on one B200, captured, call after call (1.6 to 1.8 GHz under this load): 8,192 rows of 24
// heads, all seen, 755 us (1,090 TFLOP/s, 0.65 of the measured bf16 GEMM peak, 0.75 in the CTAs that
// are busy to the end); 777..16,384 tokens causal 1,640 us (1,090 TFLOP/s, 0.65); 4,098 + 1,501 rows,
// all seen, 253 us. Two prompts of 1,024 tokens 30 us: the first weights are there after 6.6, a pair
// of tiles of a first unit takes 2.4 (the first and the last of a side are masked, the last one's
// values are cleaned before its softmax), an output 1.4, a quarter of the CTAs have a second unit
// and the last of them ends at 25, 7.5 pairs in all; the rest passes between the calls.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "ops_tc.cuh"

namespace y2 {
namespace {

using namespace opt;

constexpr int kMaxSeqs = 1024;
constexpr uint64_t kMaxTokens = 1u << 18;
constexpr int kThreads = 320;
constexpr int kBlock = 2 * kRows;  // query rows of a unit
constexpr int kUnits = 4;          // published units in flight

struct PackedArgs {
  const uint16_t* v;
  uint16_t* out;
  const int32_t* cu;
  int32_t* status;
  long long v_stride, out_stride;
  int seqs, tokens, heads, group, causal, negate;
  float c;  // |scale| log2(e)
};

struct Unit {
  int first, n;     // the sequence's rows
  int block, head;  // rows 256 * block .. of it; head < 0: no more units
  int found;        // a value that is not finite was taken out of a masked tile
};

template <int D>
struct Layout {
  static constexpr int TILE = kRows * D * 2;  // bytes of a Q, K or V tile
  static constexpr int SLOTS = D == 128 ? 5 : 8;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_BAR = OFF_KV + SLOTS * TILE;
  static constexpr int BARS = 2 * SLOTS + 2 * kUnits + 2 + 8 + 1;
  static constexpr int OFF_UNIT = OFF_BAR + BARS * 8;
  static constexpr int OFF_MISC = OFF_UNIT + kUnits * (int)sizeof(Unit);
  static constexpr int BYTES = OFF_MISC + 16;
};

struct Seq {
  int first, n;
};
Y2_DEV Seq seq_of(const PackedArgs& a, int s) {
  const int lo = a.cu[s], hi = a.cu[s + 1];
  if (lo < 0 || hi < lo || hi > a.tokens) return {0, -1};
  return {lo, hi - lo};
}

// The order of units (one warp): by block index from the highest down, within it by sequence
// then head.
struct Walk {
  int level, base, count;
};
Y2_DEV int blocks_of(const PackedArgs& a, int s) {
  return s < a.seqs ? (seq_of(a, s).n + kBlock - 1) / kBlock : 0;  // -1 rows: 0
}
Y2_DEV int count_above(const PackedArgs& a, int level) {
  const int lane = threadIdx.x & 31;
  int n = 0;
  for (int s = 0; s < a.seqs; s += 32) n += __popc(__ballot_sync(0xffffffffu, blocks_of(a, s + lane) > level));
  return n;
}
Y2_DEV void walk_begin(const PackedArgs& a, Walk& w) {
  const int lane = threadIdx.x & 31;
  int most = 0, sum = 0;  // at most 2^10 sequences of 2^18 rows
  bool bad = false;
  for (int s = lane; s < a.seqs; s += 32) {
    bad |= seq_of(a, s).n < 0;
    sum += max(0, seq_of(a, s).n);
    most = max(most, blocks_of(a, s));
  }
  most = __reduce_max_sync(0xffffffffu, most);
  // offsets that go back and forth would give more rows than there are, up to hundreds of times
  // the work of any valid call: none is done
  if (__reduce_add_sync(0xffffffffu, sum) > a.tokens) bad = true, most = 0;
  if (bad && blockIdx.x == 0) status_or(a.status, YUE2_STATUS_RANGE);
  w.level = most - 1;
  w.base = 0;
  w.count = most > 0 ? count_above(a, w.level) : 0;
}
Y2_DEV Unit walk_to(const PackedArgs& a, Walk& w, int u) {
  const int lane = threadIdx.x & 31;
  while (w.level >= 0 && u >= w.base + w.count * a.heads) {
    w.base += w.count * a.heads;
    --w.level;
    w.count = w.level >= 0 ? count_above(a, w.level) : 0;
  }
  Unit r = {0, 0, 0, -1, 0};
  if (w.level < 0) return r;
  int nth = (u - w.base) / a.heads;
  const int head = (u - w.base) % a.heads;
  for (int s = 0; s < a.seqs; s += 32) {
    const uint32_t has = __ballot_sync(0xffffffffu, blocks_of(a, s + lane) > w.level);
    if (nth < __popc(has)) {
      const int at = s + __fns(has, 0, nth + 1);
      const Seq q = seq_of(a, at);
      r = {q.first, q.n, w.level, head, 0};
      break;
    }
    nth -= __popc(has);
  }
  return r;
}

// Rows of a side (0: it has nothing to do), and its tiles of 128 keys.
Y2_DEV int side_rows(const Unit& u, int side) { return max(0, min(kRows, u.n - u.block * kBlock - side * kRows)); }
Y2_DEV int side_tiles(const PackedArgs& a, const Unit& u, int side) {
  if (side_rows(u, side) == 0) return 0;
  return a.causal ? 2 * u.block + side + 1 : (u.n + kKeys - 1) / kKeys;
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    attention_packed_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mk,
                            const __grid_constant__ CUtensorMap mv, const PackedArgs a) {
  using L = Layout<D>;
  constexpr int SLOTS = L::SLOTS, TILE = L::TILE;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bar = (uint64_t*)(smem + L::OFF_BAR);
  uint64_t *kv_full = bar, *kv_empty = bar + SLOTS, *unit_full = kv_empty + SLOTS, *unit_empty = unit_full + kUnits;
  uint64_t *q_full = unit_empty + kUnits, *q_empty = q_full + 1, *drain = q_empty + 1;
  // per side: scores written, three quarters of the weights, all of them, the last P.V done
  uint64_t *s_full = drain + 1, *p_part = s_full + 2, *p_full = p_part + 2, *o_full = p_full + 2;
  Unit* units = (Unit*)(smem + L::OFF_UNIT);
  uint32_t* tmem_slot = (uint32_t*)(smem + L::OFF_MISC);
  volatile int* ending = (volatile int*)(smem + L::OFF_MISC + 4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < SLOTS; ++i) {
      tc::mbar_init(kv_full + i, 1);
      tc::mbar_init(kv_empty + i, 1);
    }
    for (int i = 0; i < kUnits; ++i) {
      tc::mbar_init(unit_full + i, 1);
      tc::mbar_init(unit_empty + i, 9);
    }
    tc::mbar_init(q_full, 1);
    tc::mbar_init(q_empty, 1);
    tc::mbar_init(drain, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(s_full + i, 1);
      tc::mbar_init(p_part + i, 4);
      tc::mbar_init(p_full + i, 4);
      tc::mbar_init(o_full + i, 1);
    }
    *ending = 0;
    tc::mbar_init_fence();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax and output
    const int side = warp >> 2, t = threadIdx.x & (kRows - 1);
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t s_addr = lanes + s_col(side), o_addr = lanes + o_col(side);
    uint32_t s_phase = 0, o_phase = 0, kv_count = 0;
    for (int k = 0;; ++k) {
      const int us = k % kUnits;
      if (!__all_sync(0xffffffffu, wait(unit_full + us, (k / kUnits) & 1, ending, a.status))) break;
      const Unit u = units[us];
      if (u.head < 0) break;
      const int tiles = side_tiles(a, u, side), rows = side_rows(u, side);
      const int row = u.block * kBlock + side * kRows + t;  // within the sequence
      const int last = a.causal ? min(row, u.n - 1) : u.n - 1;
      RowStats st;
      st.begin(t < rows);
      bool ok = true;
      for (int j = 0; j < tiles; ++j) {
        ok = __all_sync(0xffffffffu, wait(s_full + side, s_phase, ending, a.status));
        if (!ok) break;
        s_phase ^= 1;
        tc::fence_after();
        // the weights in TMEM so far, to the warp that issues the products: one arrival a warp
        auto announce = [&](uint64_t* b) {
          wait_stores();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(b + side);
        };
        // only the last tile of a side has keys that some row does not see; the values of the
        // last tile of either side are cleaned by both, whichever comes first. Without the causal
        // mask those are the keys past the end alone, and no row has a value to add later.
        const bool masked = j == tiles - 1 && (a.causal || u.n % kKeys);
        const bool clean = masked || (a.causal && j == tiles - 1 - side);
        const int seen = masked ? last - j * kKeys + 1 : kKeys;  // keys [0, seen) of the tile
        uint32_t vis[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = seen - 32 * q;
          vis[q] = r >= 32 ? 0xffffffffu : r <= 0 ? 0u : (1u << r) - 1;
        }
        if (clean) {
          const uint32_t at = kv_count + 2 * j + 1;
          ok = __all_sync(0xffffffffu, wait(kv_full + at % SLOTS, (at / SLOTS) & 1, ending, a.status));
          if (!ok) break;
          const bool dead = j * kKeys + t >= u.n;
          for (int slab = 0; (a.causal || dead) && slab < D / 64; ++slab)
            clean_values<F16>(smem + L::OFF_KV + (at % SLOTS) * TILE + slab * (kKeys * 128), t, dead, &units[us].found);
          tc::fence_proxy_async();
        }
        auto part = [&] { announce(p_part); };
        if (masked || a.negate || j == 0 || !softmax_settled<D, F16>(s_addr, a.c, st, part))
          softmax_masked<D, F16, 4>(s_addr, o_addr, a.c, a.negate, j == 0, vis, st, part);
        announce(p_full);
      }
      if (!ok) break;
      kv_count += 2 * max(side_tiles(a, u, 0), side_tiles(a, u, 1));
      if (tiles) {
        if (!__all_sync(0xffffffffu, wait(o_full + side, o_phase, ending, a.status))) break;
        o_phase ^= 1;
        tc::fence_after();
        const float l = st.total(), inv = 1.0f / l;
        const bool some = l != 0.f;  // else every score is -inf: zeros
        const bool found = some && *(volatile int*)&units[us].found;
        char* to[4];
        quad_rows(t < rows ? a.out + (long long)(u.first + row) * a.out_stride + u.head * D : nullptr, to);
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          load32(o_addr + 32 * q, o);
          wait_loads();
          arrived(o);
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = some ? __uint_as_float(o[i]) * inv : 0.f;
          if (found && t < rows)  // keys of the unit's masked tiles that this row sees
            for (int key = u.block * kBlock; key <= last; ++key)
              add_nonfinite<F16>(a.v + (long long)(u.first + key) * a.v_stride + (u.head / a.group) * D + 32 * q, f);
          uint4 w[4];
          pack32<F16>(f, w);
          quad_store(to, 64 * q, w);
        }
        tc::fence_before();
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(unit_empty + us);
    }
  } else if (warp == 8) {
    // ---------------------------------------------------------------- products
    const uint32_t base = uniform(tmem), qs = tc::smem_u32(smem), kvs = tc::smem_u32(smem + L::OFF_KV);
    uint32_t p_phase[2] = {0, 0}, q_phase = 0, kv_count = 0;
    auto ready = [&](uint64_t* b, uint32_t parity) {
      const bool r = __all_sync(0xffffffffu, wait(b, parity, ending, a.status)) != 0;
      tc::fence_after();
      return r;
    };
    auto kv_wait = [&](uint32_t at) { return ready(kv_full + at % SLOTS, (at / SLOTS) & 1); };
    auto kv_addr = [&](uint32_t at) { return kvs + (at % SLOTS) * TILE; };
    for (int k = 0;; ++k) {
      const int us = k % kUnits;
      if (!ready(unit_full + us, (k / kUnits) & 1)) break;
      const Unit u = units[us];
      if ((int)uniform(u.head) < 0) break;
      const int tiles[2] = {(int)uniform(side_tiles(a, u, 0)), (int)uniform(side_tiles(a, u, 1))}, all = max(tiles[0], tiles[1]);
      if (!ready(q_full, q_phase)) break;
      q_phase ^= 1;
      bool ok = kv_wait(kv_count);
      if (!ok) break;
      if (elect_one()) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
          if (tiles[s]) {
            issue_scores<D, F16>(base + s_col(s), qs + s * TILE, kv_addr(kv_count));
            tc::commit(s_full + s);
          }
        tc::commit(kv_empty + kv_count % SLOTS);
        if (all == 1) tc::commit(q_empty);
      }
      __syncwarp();
      for (int j = 0; j < all; ++j) {
        const uint32_t vt = kv_count + 2 * j + 1, kt = vt + 1;
        ok = kv_wait(vt) && (j + 1 >= all || kv_wait(kt));
        if (!ok) break;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (j >= tiles[s]) continue;
          ok = ready(p_part + s, p_phase[s]);
          if (!ok) break;
          if (elect_one()) issue_values<D, F16>(base + o_col(s), base + s_col(s), kv_addr(vt), 0, 6, j > 0);
          __syncwarp();
          ok = ready(p_full + s, p_phase[s]);
          if (!ok) break;
          p_phase[s] ^= 1;
          if (elect_one()) {
            issue_values<D, F16>(base + o_col(s), base + s_col(s), kv_addr(vt), 6, 8, true);
            if (j == tiles[s] - 1) {
              tc::commit(o_full + s);
            } else {
              issue_scores<D, F16>(base + s_col(s), qs + s * TILE, kv_addr(kt));
              tc::commit(s_full + s);
            }
            if (s == 1 || j >= tiles[1]) {  // the last side to use these tiles
              tc::commit(kv_empty + vt % SLOTS);
              if (j + 1 < all) tc::commit(kv_empty + kt % SLOTS);
              if (j + 2 == all) tc::commit(q_empty);
            }
          }
          __syncwarp();
        }
        if (!ok) break;
      }
      if (!ok) break;
      kv_count += 2 * all;
      if (lane == 0) tc::mbar_arrive(unit_empty + us);
    }
    // every product is done before the TMEM goes (at once, unless a wait gave up)
    if (elect_one()) tc::commit(drain);
    __syncwarp();
    settle(drain, 0, a.status);
  } else {
    // ---------------------------------------------------------------- units and loads
    Walk w;
    walk_begin(a, w);
    uint32_t kv_count = 0, q_count = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      const int g = (int)gridDim.x;
      const Unit u = walk_to(a, w, k * g + (k & 1 ? g - 1 - (int)blockIdx.x : (int)blockIdx.x));
      const int us = k % kUnits;
      ok = __all_sync(0xffffffffu, wait(unit_empty + us, ((k / kUnits) & 1) ^ 1, ending, a.status));
      if (!ok) break;
      if (lane == 0) {
        units[us] = u;
        tc::mbar_arrive(unit_full + us);
      }
      __syncwarp();
      if (u.head < 0) break;
      const int both = side_rows(u, 1) > 0, tiles = max(side_tiles(a, u, 0), side_tiles(a, u, 1));
      ok = __all_sync(0xffffffffu, wait(q_empty, (q_count & 1) ^ 1, ending, a.status));
      if (!ok) break;
      ++q_count;
      const int row = u.first + u.block * kBlock, kvh = u.head / a.group;
      if (lane == 0) {
        tc::mbar_arrive_expect_tx(q_full, (both ? 2 : 1) * TILE);
        for (int s = 0; s <= both; ++s)
          for (int x = 0; x < D; x += 64)
            tma_load_3d(smem + s * TILE + x / 64 * (kRows * 128), &mq, q_full, x, u.head, row + s * kRows);
      }
      for (int j = 0; j < 2 * tiles; ++j, ++kv_count) {
        const int slot = kv_count % SLOTS;
        ok = __all_sync(0xffffffffu, wait(kv_empty + slot, ((kv_count / SLOTS) & 1) ^ 1, ending, a.status));
        if (!ok) break;
        if (lane == 0) {
          tc::mbar_arrive_expect_tx(kv_full + slot, TILE);
          unsigned char* dst = smem + L::OFF_KV + slot * TILE;
          for (int x = 0; x < D; x += 64)
            tma_load_3d(dst + x / 64 * (kRows * 128), j & 1 ? &mv : &mk, kv_full + slot, x, kvh, u.first + (j >> 1) * kKeys);
        }
        __syncwarp();
      }
    }
    // no copy in flight outlives the CTA (when a wait gave up, some may not have been used)
    if (!ok) {
      for (uint32_t i = kv_count > SLOTS ? kv_count - SLOTS : 0; i < kv_count; ++i)
        settle(kv_full + i % SLOTS, (i / SLOTS) & 1, a.status);
      if (q_count) settle(q_full, (q_count - 1) & 1, a.status);
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 8) {
    tc::fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

template <int D, bool F16>
int launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const PackedArgs& a, cudaStream_t st) {
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaDeviceGetAttribute");
  static std::atomic<uint64_t> ready{0};  // devices on which the shared-memory limit is set
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(attention_packed_kernel<D, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::BYTES);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const long long most = ((long long)a.tokens / kBlock + std::min(a.seqs, a.tokens)) * a.heads;
  attention_packed_kernel<D, F16><<<(unsigned)std::min<long long>(sms, most), kThreads, Layout<D>::BYTES, st>>>(mq, mk, mv, a);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : cuda_fail(e, "attention_packed launch");
}

}  // namespace
}  // namespace y2

using namespace y2;

extern "C" int yue2_attention_packed(const void* q, const void* k, const void* v, void* out, const int32_t* cu,
                                     uint64_t seqs, uint64_t tokens, uint64_t heads, uint64_t kv, uint64_t dim,
                                     uint64_t q_stride, uint64_t k_stride, uint64_t v_stride, uint64_t out_stride,
                                     int32_t dtype, int32_t causal, float scale, int32_t* status, void* stream) {
  int rc = check_heads(heads, kv);
  if (rc || (rc = check_status(status)) || (rc = check_scale(scale))) return rc;
  if (dim != 64 && dim != 128) return fail(YUE2_ERR_INVALID, "attention takes a head dim of 64 or 128");
  if (dtype != YUE2_DTYPE_BF16 && dtype != YUE2_DTYPE_F16) return fail(YUE2_ERR_INVALID, "values must be bf16 or f16");
  if (seqs > (uint64_t)kMaxSeqs || tokens > kMaxTokens)
    return fail(YUE2_ERR_INVALID, "at most 1,024 sequences and 262,144 tokens per call");
  if ((rc = check_rows(q, tokens, heads, dim, q_stride, "q")) || (rc = check_rows(k, tokens, kv, dim, k_stride, "k")) ||
      (rc = check_rows(v, tokens, kv, dim, v_stride, "v")) || (rc = check_rows(out, tokens, heads, dim, out_stride, "out")))
    return rc;
  if (seqs == 0 || tokens == 0) return 0;
  if (!cu) return fail(YUE2_ERR_INVALID, "null sequence offsets");
  if ((rc = check_list(cu, 4, "cu"))) return rc;
  const bool f16 = dtype == YUE2_DTYPE_F16;
  CUtensorMap mq, mk, mv;
  if (!opt::make_rows_map(&mq, f16, q, tokens, heads, dim, q_stride, 1, opt::kRows) ||
      !opt::make_rows_map(&mk, f16, k, tokens, kv, dim, k_stride, 1, opt::kRows) ||
      !opt::make_rows_map(&mv, f16, v, tokens, kv, dim, v_stride, 1, opt::kRows))
    return fail(YUE2_ERR_INVALID, "q, k or v cannot be described to the copy engine (base, strides)");
  PackedArgs a = {};
  a.v = (const uint16_t*)v;
  a.out = (uint16_t*)out;
  a.cu = cu;
  a.status = status;
  a.v_stride = (long long)v_stride;
  a.out_stride = (long long)out_stride;
  a.seqs = (int)seqs;
  a.tokens = (int)tokens;
  a.heads = (int)heads;
  a.group = (int)(heads / kv);
  a.causal = causal != 0;
  a.negate = scale < 0.f;
  a.c = opt::weight_scale(scale);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dim == 64) return f16 ? launch<64, true>(mq, mk, mv, a, st) : launch<64, false>(mq, mk, mv, a, st);
  return f16 ? launch<128, true>(mq, mk, mv, a, st) : launch<128, false>(mq, mk, mv, a, st);
}
