// yue2_attention_tree: attention of drafted tokens over paged K/V on the 5th-generation tensor
// cores, bound by reading the pages.
//
// The G = heads / kv query heads of a group share K and V, so a tile has rows (node, head): 128
// of them are a side (floor(128 / G) nodes). An item of work is one kv head of one
// sequence with up to two sides of rows; its keys come in tiles of 128 (two pages). When the
// rows fill one side, both sides hold them and take the tiles in turn, and their results are
// merged in TMEM: two softmax warps then keep up with HBM even when a single warp has rows.
//
// The items form one line (a fixed cost, then their tiles), cut into equal shares for the CTAs
// (one per SM), so that one long context among short ones loads every SM alike. An item cut between CTAs
// leaves partial results (output, maximum and sum, f32) that a second kernel merges in tile
// order; items that lie in one share are finished at once. The shares follow from the
// lengths on the device, so the host needs none of them.
//
// A CTA is ten warps as in attention_packed: softmax of the sides, products, page loads (TMA).
//
// Measured on one B200, captured; the parts with timers in a copy. Trees of 64 and 48 nodes over
// 24,512 and 20,001 positions (24 / 8 heads of 128) 60 us against 28 us for the bytes alone: the first
// weights are there after 6.6 (shares 2.4, page table and first tiles 2.6, softmax 1.6), each of 17
// more tiles takes 2.0 (two sides of products and softmax; the bytes alone 1.5), the output or
// partial results 3.1, and the last CTA ends at 50; the other 10 are the launches and the merge. A
// batch of eight trees at 63..8,191 positions 42 us against 18: 6.3, nine tiles of 1.9, 3, the last CTA
// at 35, then 7. One token of two sequences at 1,030 positions 14.6 us, all of it latency: 6.3 to
// the first weights, 9.7 for the last CTA, then 5.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "ops_tc.cuh"

namespace y2 {
namespace {

using namespace opt;

constexpr int kMaxSeqs = 1024;
constexpr int kMaxNodes = 64;
constexpr int kMaxGroup = 128;  // query heads per kv head: one node's rows fit a side
constexpr int kThreads = 320;
constexpr int kUnits = 4;
constexpr int kMergeThreads = 256;

struct TreeArgs {
  uint16_t* out;
  const uint16_t* pool;
  const int32_t *table, *context, *cu;
  const uint64_t* mask;
  int32_t* status;
  float* part;  // [2 * CTAs][slot_rows][D] outputs, then [2 * CTAs][slot_rows][2] maximum and sum
  long long out_stride, pages, page_stride, table_pages;
  int seqs, rows, heads, kv, group, nodes, layer, blocks, negate, ctas, slot_rows;
  float c;  // |scale| log2(e)
};

// One sequence: rows first .. first + n - 1, its context, tiles of 128 keys and row blocks of
// up to 2 * a.nodes nodes. n = 0: nothing to do. A bad entry is reported once.
struct SeqWork {
  int first, n, tiles, parts;
  long long ctx;
};
Y2_DEV SeqWork seq_work(const TreeArgs& a, int s, bool report) {
  SeqWork w = {0, 0, 0, 0, 0};
  const int lo = a.cu[s], hi = a.cu[s + 1], ctx = a.context[s];
  if (lo < 0 || hi < lo || hi > a.rows || hi - lo > kMaxNodes || ctx < 0 ||
      (hi > lo && (long long)ctx + hi - lo > a.table_pages * kPageTokens)) {
    if (report) status_or(a.status, YUE2_STATUS_RANGE);
    return w;
  }
  if (hi == lo) return w;
  w.first = lo;
  w.n = hi - lo;
  w.ctx = ctx;
  w.tiles = (int)((w.ctx + w.n + kKeys - 1) / kKeys);
  w.parts = (w.n + 2 * a.nodes - 1) / (2 * a.nodes);
  return w;
}

// The line of work: an item is kItemCost units (its loads of q, masked tiles and output
// take about as long as that many tiles) and then one unit a tile. CTA c of `used` takes the
// units [share(c), share(c + 1)). Lines of 2^31 units and more are refused.
constexpr int kItemCost = 2;
Y2_DEV int item_length(const SeqWork& w) { return w.n ? w.tiles + kItemCost : 0; }
Y2_DEV int seq_length(const TreeArgs& a, const SeqWork& w) {
  return (int)min((long long)INT32_MAX, (long long)item_length(w) * w.parts * a.kv);
}
struct Shares {
  int used, each, more;  // the first `more` CTAs take one unit more than `each`
  Y2_DEV Shares(const TreeArgs& a, int all) {
    used = min(a.ctas, max(all, 1));
    each = all / used;
    more = all % used;
  }
  Y2_DEV int begin(int c) const { return c * each + min(c, more); }
  Y2_DEV int owner(int x) const {
    const int wide = more * (each + 1);
    return x < wide ? x / (each + 1) : more + (x - wide) / each;
  }
};

struct Unit {
  int first, n, node, head;  // the sequence's rows, the block's first node, the kv head (< 0: end)
  int seq, t0, t1;           // tiles [t0, t1)
  int slot;                  // partial results to this slot; < 0: the item is complete
  long long ctx;
  int found;
};

template <int D>
struct Layout {
  static constexpr int TILE = kRows * D * 2;
  static constexpr int SLOTS = D == 128 ? 5 : 8;
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_BAR = OFF_KV + SLOTS * TILE;
  static constexpr int BARS = 2 * SLOTS + 2 * kUnits + 2 + 1 + 8 + 2;
  static constexpr int OFF_UNIT = OFF_BAR + BARS * 8;
  static constexpr int OFF_ML = OFF_UNIT + kUnits * (int)sizeof(Unit);
  static constexpr int OFF_MISC = OFF_ML + kRows * 8;
  static constexpr int BYTES = OFF_MISC + 16;
};

// A unit's sides. One side of nodes: both hold it and side s takes tiles t0 + s, t0 + s + 2, ..
Y2_DEV bool in_turn(const TreeArgs& a, const Unit& u) { return u.n - u.node <= a.nodes; }
Y2_DEV int side_tiles(const TreeArgs& a, const Unit& u, int side) {
  const int t = u.t1 - u.t0;
  return in_turn(a, u) ? (t + 1 - side) / 2 : t;
}

// Bits [p, p + 32) of what a node sees: the context, then its mask over the n drafted positions.
Y2_DEV uint32_t seen_bits(long long p, long long ctx, uint64_t mask) {
  const long long sh = p - ctx;
  if (sh >= 64) return 0;
  if (sh >= 0) return (uint32_t)(mask >> sh);
  if (sh <= -32) return 0xffffffffu;
  return (uint32_t)(mask << -sh) | ((1u << -sh) - 1);
}

template <int D, bool F16>
__global__ void __launch_bounds__(kThreads, 1)
    attention_tree_kernel(const __grid_constant__ CUtensorMap mq, const __grid_constant__ CUtensorMap mkv, const TreeArgs a) {
  using L = Layout<D>;
  constexpr int SLOTS = L::SLOTS, TILE = L::TILE;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bar = (uint64_t*)(smem + L::OFF_BAR);
  uint64_t *kv_full = bar, *kv_empty = bar + SLOTS, *unit_full = kv_empty + SLOTS, *unit_empty = unit_full + kUnits;
  uint64_t *q_full = unit_empty + kUnits, *q_empty = q_full + 1, *drain = q_empty + 1;
  // per side: scores written, three quarters of the weights, all of them, the last P.V done
  uint64_t *s_full = drain + 1, *p_part = s_full + 2, *p_full = p_part + 2, *o_full = p_full + 2;
  uint64_t *ml_full = o_full + 2, *ml_empty = ml_full + 1;  // side 1's statistics, for the merge
  Unit* units = (Unit*)(smem + L::OFF_UNIT);
  float2* ml = (float2*)(smem + L::OFF_ML);
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
    tc::mbar_init(ml_full, 4);
    tc::mbar_init(ml_empty, 4);
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
  pdl_trigger();  // the merge may be set up meanwhile; it waits for this grid's results

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax and output
    const int side = warp >> 2, t = threadIdx.x & (kRows - 1);
    const uint32_t lanes = tmem + ((uint32_t)(warp & 3) << 21);
    const uint32_t s_addr = lanes + s_col(side), o_addr = lanes + o_col(side);
    uint32_t s_phase = 0, o_phase = 0, ml_phase = 0, kv_count = 0;
    for (int k = 0;; ++k) {
      const int us = k % kUnits;
      if (!__all_sync(0xffffffffu, wait(unit_full + us, (k / kUnits) & 1, ending, a.status))) break;
      const Unit u = units[us];
      if (u.head < 0) break;
      const bool turns = in_turn(a, u);
      const int tiles = side_tiles(a, u, side), stride = turns ? 2 : 1;
      const int node0 = u.node + (turns ? 0 : side * a.nodes);
      const int rows = min(a.nodes, u.n - node0) * a.group;
      const int node = node0 + t / a.group;  // of the sequence
      const bool live = t < rows, warp_live = (warp & 3) * 32 < rows;
      const uint64_t drafted = u.n < 64 ? (1ull << u.n) - 1 : ~0ull;
      uint64_t mask = 0;
      if (live) mask = a.mask ? a.mask[u.first + node] & drafted : (node < 63 ? (2ull << node) - 1 : ~0ull);
      RowStats st;
      st.begin(live);
      bool ok = true;
      for (int i = 0; i < tiles; ++i) {
        const int j = u.t0 + (turns ? side : 0) + i * stride;  // tile of the sequence
        ok = __all_sync(0xffffffffu, wait(s_full + side, s_phase, ending, a.status));
        if (!ok) break;
        s_phase ^= 1;
        tc::fence_after();
        auto announce = [&](uint64_t* b) {
          wait_stores();
          tc::fence_before();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(b + side);
        };
        auto part = [&] { announce(p_part); };
        const long long key0 = (long long)j * kKeys;
        const bool masked = key0 + kKeys > u.ctx;  // the tile reaches into the drafted positions
        if (masked) {
          const uint32_t at = kv_count + 2 * (j - u.t0) + 1;
          ok = __all_sync(0xffffffffu, wait(kv_full + at % SLOTS, (at / SLOTS) & 1, ending, a.status));
          if (!ok) break;
          if (key0 + t >= u.ctx)
            for (int slab = 0; slab < D / 64; ++slab)
              clean_values<F16>(smem + L::OFF_KV + (at % SLOTS) * TILE + slab * (kKeys * 128), t, key0 + t >= u.ctx + u.n,
                                &units[us].found);
          tc::fence_proxy_async();
        }
        if (!warp_live) {
          part();
        } else if (masked || a.negate || !softmax_tile<D, F16>(s_addr, o_addr, a.c, i == 0, st, part)) {
          uint32_t vis[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) vis[q] = seen_bits(key0 + 32 * q, u.ctx, mask);
          softmax_masked<D, F16, 1>(s_addr, o_addr, a.c, a.negate, i == 0, vis, st, part);
        }
        announce(p_full);
      }
      if (!ok) break;
      kv_count += 2 * (u.t1 - u.t0);
      if (tiles) {
        ok = __all_sync(0xffffffffu, wait(o_full + side, o_phase, ending, a.status));
        if (!ok) break;
        o_phase ^= 1;
        tc::fence_after();
      }
      // the two sides of one set of rows: side 1 hands over its statistics, side 0 reads both outputs
      const bool merge = turns && u.t1 - u.t0 > 1;
      float l = st.total(), w0 = 1.f, w1 = 0.f, m = st.m;
      if (merge && side == 1) {
        ml[t] = make_float2(st.m, l);
        tc::fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(ml_full);
        ok = __all_sync(0xffffffffu, wait(ml_empty, ml_phase, ending, a.status));
        if (!ok) break;
        ml_phase ^= 1;
        tc::fence_after();
      } else if (merge) {
        ok = __all_sync(0xffffffffu, wait(ml_full, ml_phase, ending, a.status));
        if (!ok) break;
        ml_phase ^= 1;
        tc::fence_after();
        const float2 o = ml[t];
        m = max3(m, o.x, o.x);
        if (m != -INFINITY) {
          w0 = st.m == -INFINITY ? 0.f : ex2(apart(a.c, st.m, m));
          w1 = o.x == -INFINITY ? 0.f : ex2(apart(a.c, o.x, m));
        }
        l = l * w0 + o.y * w1;
      }
      if (warp_live && (side == 0 || !turns)) {
        const bool found = *(volatile int*)&units[us].found;
        const float inv = 1.0f / l;
        const bool some = l != 0.f;  // else nothing seen, or scores of -inf alone: zeros
        const int row = u.first + node, head = u.head * a.group + t % a.group;
        const long long prow = (long long)u.slot * a.slot_rows + (node - u.node) * a.group + t % a.group;
        void* mine = u.slot >= 0 ? (void*)(a.part + prow * D) : (void*)(a.out + (long long)row * a.out_stride + (long long)head * D);
        char* to[4];
        quad_rows(live ? mine : nullptr, to);
#pragma unroll 1
        for (int q = 0; q < D / 32; ++q) {
          uint32_t o[32];
          load32(o_addr + 32 * q, o);
          wait_loads();
          arrived(o);
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = w0 == 0.f ? 0.f : __uint_as_float(o[i]) * w0;
          if (merge) {
            load32(lanes + o_col(1) + 32 * q, o);
            wait_loads();
            arrived(o);
            if (w1 != 0.f) {
#pragma unroll
              for (int i = 0; i < 32; ++i) f[i] = fmaf(__uint_as_float(o[i]), w1, f[i]);
            }
          }
          if (found && live) {  // drafted values that are not finite, of the keys of these tiles
            for (int d = 0; d < u.n; ++d) {
              const long long key = u.ctx + d;
              if (!(mask >> d & 1) || key < (long long)u.t0 * kKeys || key >= (long long)u.t1 * kKeys) continue;
              const long long page = a.table[(long long)u.seq * a.table_pages + (key >> kPageLog2)];
              if (page < 0 || page >= a.pages) continue;
              add_nonfinite<F16>(a.pool + page * a.page_stride +
                                     ((long long)(a.layer * 2 + 1) * a.kv + u.head) * (kPageTokens * D) +
                                     (key & (kPageTokens - 1)) * D + 32 * q,
                                 f);
            }
          }
          uint4 v[4];
          if (u.slot >= 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float* x = f + 16 * h + 4 * i;
                v[i] = make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
              }
              quad_store(to, 128 * q + 64 * h, v);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = some ? f[i] * inv : 0.f;
            pack32<F16>(f, v);
            quad_store(to, 64 * q, v);
          }
        }
        if (live && u.slot >= 0)
          reinterpret_cast<float2*>(a.part + 2ll * a.ctas * a.slot_rows * D)[prow] = make_float2(m, l);
      }
      tc::fence_before();
      __syncwarp();
      if (merge && side == 0 && lane == 0) tc::mbar_arrive(ml_empty);
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
      const bool turns = uniform(in_turn(a, u)) != 0;
      const int all = (int)uniform(u.t1 - u.t0);
      if (!ready(q_full, q_phase)) break;
      q_phase ^= 1;
      // the first scores of both sides: of tile 0, or of tiles 0 and 1 in turn
      const int firsts = turns ? min(all, 2) : 1;
      bool ok = true;
      for (int j = 0; j < firsts && ok; ++j) {
        ok = kv_wait(kv_count + 2 * j);
        if (!ok) break;
        if (elect_one()) {
#pragma unroll
          for (int s = 0; s < 2; ++s)
            if (!turns || s == j) {
              issue_scores<D, F16>(base + s_col(s), qs + (turns ? 0 : s * TILE), kv_addr(kv_count + 2 * j));
              tc::commit(s_full + s);
            }
          tc::commit(kv_empty + (kv_count + 2 * j) % SLOTS);
          if (j + 1 == all) tc::commit(q_empty);
        }
        __syncwarp();
      }
      if (!ok) break;
      const int ahead = turns ? 2 : 1;  // the side's next scores
      for (int j = 0; j < all; ++j) {
        const uint32_t vt = kv_count + 2 * j + 1, kt = kv_count + 2 * (j + ahead);
        ok = kv_wait(vt) && (j + ahead >= all || kv_wait(kt));
        if (!ok) break;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (turns && s != (j & 1)) continue;
          ok = ready(p_part + s, p_phase[s]);
          if (!ok) break;
          if (elect_one()) issue_values<D, F16>(base + o_col(s), base + s_col(s), kv_addr(vt), 0, 6, j >= ahead);
          __syncwarp();
          ok = ready(p_full + s, p_phase[s]);
          if (!ok) break;
          p_phase[s] ^= 1;
          if (elect_one()) {
            issue_values<D, F16>(base + o_col(s), base + s_col(s), kv_addr(vt), 6, 8, true);
            if (j + ahead >= all) {
              tc::commit(o_full + s);
            } else {
              issue_scores<D, F16>(base + s_col(s), qs + (turns ? 0 : s * TILE), kv_addr(kt));
              tc::commit(s_full + s);
            }
            if (turns || s == 1) {  // the last use of these tiles
              tc::commit(kv_empty + vt % SLOTS);
              if (j + ahead < all) tc::commit(kv_empty + kt % SLOTS);
              if (j + ahead + 1 == all) tc::commit(q_empty);
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
    // ---------------------------------------------------------------- shares and page loads
    const bool report = blockIdx.x == 0;
    // lane l keeps sequence l (most calls have no more), so that the walk needs no second look
    const SeqWork lane_work = lane < a.seqs ? seq_work(a, lane, report) : SeqWork{0, 0, 0, 0, 0};
    auto work_of = [&](int s) {
      if (s >= 32) return seq_work(a, s, false);
      SeqWork w;
      w.first = __shfl_sync(0xffffffffu, lane_work.first, s);
      w.n = __shfl_sync(0xffffffffu, lane_work.n, s);
      w.tiles = __shfl_sync(0xffffffffu, lane_work.tiles, s);
      w.parts = __shfl_sync(0xffffffffu, lane_work.parts, s);
      w.ctx = __shfl_sync(0xffffffffu, lane_work.ctx, s);
      return w;
    };
    long long sum = seq_length(a, lane_work);
    for (int s = lane + 32; s < a.seqs; s += 32) sum += seq_length(a, seq_work(a, s, report));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const bool fits = sum < INT32_MAX;
    if (!fits && report && lane == 0) status_or(a.status, YUE2_STATUS_RANGE);
    const int all = fits ? (int)sum : 0;
    const Shares shares(a, all);
    const bool mine = (int)blockIdx.x < shares.used;
    int at = mine ? shares.begin(blockIdx.x) : all;
    const int end = mine ? shares.begin(blockIdx.x + 1) : all;
    // the sequence that holds unit `at`, and the units before it
    int seq = 0, before = 0;
    if (at < end) {
      for (;; seq += 32) {
        const int own = seq == 0 ? seq_length(a, lane_work)
                        : seq + lane < a.seqs ? seq_length(a, seq_work(a, seq + lane, false)) : 0;
        int upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + upto > at);
        if (past) {
          const int l = __ffs(past) - 1;
          seq += l;
          before += __shfl_sync(0xffffffffu, upto - own, l);
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    SeqWork w = {0, 0, 0, 0, 0};
    if (at < end) w = work_of(seq);
    int length = item_length(w), total = seq_length(a, w);
    uint32_t kv_count = 0, q_count = 0;
    bool ok = true;
    for (int k = 0; ok; ++k) {
      Unit u = {0, 0, 0, -1, 0, 0, 0, -1, 0, 0};
      while (at < end) {
        while (at >= before + total) {
          before += total;
          w = work_of(++seq);
          length = item_length(w), total = seq_length(a, w);
        }
        const int item = (at - before) / length, item0 = before + item * length;
        u.t0 = max(0, at - item0 - kItemCost);
        u.t1 = min(w.tiles, end - item0 - kItemCost);
        at = min(end, item0 + length);
        if (u.t1 <= u.t0) continue;  // only of the fixed cost: the next CTA has the tiles
        u.first = w.first;
        u.n = w.n;
        u.node = (item % w.parts) * 2 * a.nodes;
        u.head = item / w.parts;
        u.seq = seq;
        u.ctx = w.ctx;
        if (u.t0 > 0) u.slot = 2 * blockIdx.x;
        else if (u.t1 < w.tiles) u.slot = 2 * blockIdx.x + 1;
        break;
      }
      const int us = k % kUnits;
      ok = __all_sync(0xffffffffu, wait(unit_empty + us, ((k / kUnits) & 1) ^ 1, ending, a.status));
      if (!ok) break;
      if (lane == 0) {
        units[us] = u;
        tc::mbar_arrive(unit_full + us);
      }
      __syncwarp();
      if (u.head < 0) break;
      ok = __all_sync(0xffffffffu, wait(q_empty, (q_count & 1) ^ 1, ending, a.status));
      if (!ok) break;
      ++q_count;
      const bool turns = in_turn(a, u);
      if (lane == 0) {
        const int sides = turns ? 1 : 2;
        tc::mbar_arrive_expect_tx(q_full, sides * a.nodes * a.group * D * 2);
        for (int s = 0; s < sides; ++s)
          for (int x = 0; x < D; x += 64)
            tma_load_3d(smem + s * TILE + x / 64 * (kRows * 128), &mq, q_full, x, u.head * a.group,
                        u.first + u.node + s * a.nodes);
      }
      const int32_t* table = a.table + (long long)u.seq * a.table_pages;
      const int held = (int)((u.ctx + u.n + kPageTokens - 1) >> kPageLog2);  // pages of the sequence
      int pages[2] = {0, 0};
      for (int j = 0; j < 2 * (u.t1 - u.t0); ++j, ++kv_count) {
        const int slot = kv_count % SLOTS, tile = u.t0 + (j >> 1);
        const int count = min(2, held - 2 * tile);
        if (!(j & 1)) {
          for (int h = 0; h < count; ++h) {
            pages[h] = table[2 * tile + h];
            if (pages[h] < 0 || pages[h] >= a.pages) {  // any page in its place: the rows are void
              if (lane == 0) status_or(a.status, YUE2_STATUS_PAGE);
              pages[h] = 0;
            }
          }
        }
        ok = __all_sync(0xffffffffu, wait(kv_empty + slot, ((kv_count / SLOTS) & 1) ^ 1, ending, a.status));
        if (!ok) break;
        if (lane == 0) {
          tc::mbar_arrive_expect_tx(kv_full + slot, count * kPageTokens * D * 2);
          unsigned char* dst = smem + L::OFF_KV + slot * TILE;
          for (int h = 0; h < count; ++h) {
            const int row = (int)(((long long)pages[h] * a.blocks + (a.layer * 2 + (j & 1)) * a.kv + u.head) * kPageTokens);
            for (int x = 0; x < D; x += 64)
              tc::tma_load_2d(dst + x / 64 * (kRows * 128) + h * (kPageTokens * 128), &mkv, kv_full + slot, x, row);
          }
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

// Rows of items that were cut: the partial results of their shares, in tile order. A CTA takes
// eight heads of a row, a warp each. Its 40 registers a thread and little shared memory fit beside an
// attention CTA, so that it is set up before that ends.
template <int D, bool F16>
__global__ void __launch_bounds__(kMergeThreads, 6) tree_merge_kernel(const TreeArgs a) {
  __shared__ int s_seq;
  __shared__ long long s_sum[2][kMergeThreads / 32];
  const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y * (kMergeThreads / 32) + warp;
  if (threadIdx.x == 0) s_seq = a.seqs;
  __syncthreads();
  long long sums[2] = {0, 0};  // units of all sequences, and of those before this one
  for (int s = threadIdx.x; s < a.seqs; s += kMergeThreads) {
    const SeqWork w = seq_work(a, s, false);
    if (row >= w.first && row < w.first + w.n) atomicMin(&s_seq, s);
    sums[0] += seq_length(a, w);
  }
  __syncthreads();
  const int seq = s_seq;
  for (int s = threadIdx.x; s < seq; s += kMergeThreads) sums[1] += seq_length(a, seq_work(a, s, false));
  for (int i = 0; i < 2; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sums[i] += __shfl_xor_sync(0xffffffffu, sums[i], o);
    if (lane == 0) s_sum[i][warp] = sums[i];
  }
  __syncthreads();
  long long all = 0, before = 0;
  for (int i = 0; i < kMergeThreads / 32; ++i) all += s_sum[0][i], before += s_sum[1][i];
  const bool some = seq < a.seqs && h < a.heads && all < INT32_MAX;
  const SeqWork w = some ? seq_work(a, seq, false) : SeqWork{0, 0, 0, 0, 0};
  const Shares shares(a, some ? (int)all : 0);
  const int node = row - w.first, block = node / (2 * a.nodes), length = item_length(w);
  const int x0 = some ? (int)before + ((h / a.group) * w.parts + block) * length : 0;
  const int c0 = some ? shares.owner(x0 + kItemCost) : 0, c1 = some ? shares.owner(x0 + length - 1) : 0;
  pdl_wait();             // by every thread, whatever its row
  if (c0 == c1) return;  // nothing to do, or finished by its CTA
  constexpr int E = D / 32;
  const float2* stats = reinterpret_cast<const float2*>(a.part + 2ll * a.ctas * a.slot_rows * D);
  const long long r = (node - block * 2 * a.nodes) * a.group + h % a.group;
  auto slot = [&](int c) { return (2ll * c + (c == c0)) * a.slot_rows + r; };
  float m = -INFINITY;
  for (int c = c0 + lane; c <= c1; c += 32) m = max3(m, stats[slot(c)].x, -INFINITY);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max3(m, __shfl_xor_sync(0xffffffffu, m, o), -INFINITY);
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int base = c0; base <= c1; base += 32) {
    float f = 0.f;
    if (base + lane <= c1) {
      const float2 s = stats[slot(base + lane)];
      // not below the smallest positive number, so that infinities stay what they are (and sums of
      // large values vanish: the smallest normal number left 2^-126 of them); a share in which the
      // row saw nothing has none
      f = s.x == -INFINITY ? 0.f : max3(ex2(apart(a.c, s.x, m)), 1.4e-45f, 0.f);
      l = fmaf(s.y, f, l);
    }
    const int n = min(32, c1 - base + 1);
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      const float* p = a.part + slot(base + i) * D + lane * E;
      if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        o[0] = fmaf(x.x, fi, o[0]), o[1] = fmaf(x.y, fi, o[1]), o[2] = fmaf(x.z, fi, o[2]), o[3] = fmaf(x.w, fi, o[3]);
      } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        o[0] = fmaf(x.x, fi, o[0]), o[1] = fmaf(x.y, fi, o[1]);
      }
    }
  }
  l = warp_sum(l);
  const float inv = 1.0f / l;
  uint16_t* dst = a.out + (long long)row * a.out_stride + (long long)h * D + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = l != 0.f ? o[e] * inv : 0.f;
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack16<F16>(o[e], o[e + 1]);
}

// Nodes of a side, CTAs and the rows of a partial result.
struct Plan {
  int nodes, ctas, slot_rows;
  uint64_t bytes;
};
Plan plan_for(uint64_t rows, uint64_t heads, uint64_t kv, uint64_t dim, uint64_t seqs, uint64_t table_pages, int sms) {
  Plan p;
  const uint64_t group = heads / kv;
  p.nodes = (int)(kRows / group);
  const uint64_t most = std::min<uint64_t>(rows, kMaxNodes);  // of one sequence
  const uint64_t parts = (most + 2 * p.nodes - 1) / (2 * p.nodes), tiles = (table_pages + 1) / 2;
  p.ctas = (int)std::max<uint64_t>(1, std::min<uint64_t>(sms, std::min<uint64_t>(seqs, rows) * kv * parts * tiles));
  p.slot_rows = (int)(std::min<uint64_t>(most, 2 * p.nodes) * group);
  p.bytes = tiles > 1 ? 2ull * p.ctas * p.slot_rows * (dim + 2) * 4 : 0;
  return p;
}

template <int D, bool F16>
int launch(const CUtensorMap& mq, const CUtensorMap& mkv, const TreeArgs& a, bool merge, cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_fail(e, "cudaGetDevice");
  static std::atomic<uint64_t> ready{0};  // devices on which the shared-memory limit is set
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    e = cudaFuncSetAttribute(attention_tree_kernel<D, F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::BYTES);
    if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  attention_tree_kernel<D, F16><<<(unsigned)a.ctas, kThreads, Layout<D>::BYTES, st>>>(mq, mkv, a);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "attention_tree launch");
  if (!merge) return 0;
  TreeArgs copy = a;
  void* args[] = {&copy};
  e = launch_with(st, true, dim3((unsigned)a.rows, (unsigned)((a.heads + 7) / 8)), dim3(kMergeThreads), 0, (const void*)tree_merge_kernel<D, F16>, args);
  return e == cudaSuccess ? 0 : cuda_fail(e, "attention_tree merge launch");
}

}  // namespace
}  // namespace y2

using namespace y2;

extern "C" {

uint64_t yue2_attention_tree_workspace(uint64_t rows, uint64_t heads, uint64_t seqs, uint64_t table_pages,
                                       const Yue2KvPool* pool) {
  int sms = 0;
  if (!pool || !rows || !seqs || !heads || !pool->kv || heads % pool->kv || heads / pool->kv > kMaxGroup || sm_count(sms))
    return 0;
  return plan_for(rows, heads, pool->kv, pool->dim, seqs, table_pages, sms).bytes;
}

int yue2_attention_tree(const void* q, uint64_t rows, uint64_t heads, uint64_t q_stride, const Yue2KvPool* pool,
                        uint64_t layer, const int32_t* table, uint64_t seqs, uint64_t table_pages,
                        const int32_t* context, const int32_t* cu, const uint64_t* mask, float scale, void* out,
                        uint64_t out_stride, void* workspace, uint64_t workspace_bytes, int32_t* status,
                        void* stream) {
  PoolView v = {};
  int rc = check_pool(pool, true, v);
  if (rc || (rc = check_heads(heads, pool->kv)) || (rc = check_status(status)) || (rc = check_scale(scale))) return rc;
  if (heads / pool->kv > kMaxGroup) return fail(YUE2_ERR_INVALID, "at most 128 query heads per kv head");
  if (layer >= pool->layers) return fail(YUE2_ERR_INVALID, "layer outside the KV pool");
  if (seqs > (uint64_t)kMaxSeqs || table_pages > (1u << 24))
    return fail(YUE2_ERR_INVALID, "at most 1,024 sequences and 2^24 pages per table row");
  if (rows > (uint64_t)kMaxNodes * kMaxSeqs) return fail(YUE2_ERR_INVALID, "at most 64 drafted rows per sequence");
  if ((rc = check_rows(q, rows, heads, pool->dim, q_stride, "q")) ||
      (rc = check_rows(out, rows, heads, pool->dim, out_stride, "out")))
    return rc;
  if (seqs == 0 || rows == 0) return 0;
  if (!table || !context || !cu) return fail(YUE2_ERR_INVALID, "null page table, context or row offsets");
  if ((rc = check_list(table, 4, "table")) || (rc = check_list(context, 4, "context")) || (rc = check_list(cu, 4, "cu")) ||
      (rc = check_list(mask, 8, "mask")))
    return rc;
  const uint64_t pool_rows = (uint64_t)v.pages * v.blocks * kPageTokens;
  if (pool_rows > (uint64_t)INT32_MAX) return fail(YUE2_ERR_INVALID, "the KV pool has more than 2^31 head rows");
  int sms = 0;
  if ((rc = sm_count(sms))) return rc;
  const Plan plan = plan_for(rows, heads, pool->kv, pool->dim, seqs, table_pages, sms);
  if (plan.bytes && (!workspace || !aligned16(workspace) || workspace_bytes < plan.bytes))
    return fail(YUE2_ERR_INVALID, "the workspace must be 16-byte aligned and hold yue2_attention_tree_workspace bytes");
  const bool f16 = pool->dtype == YUE2_DTYPE_F16;
  const uint64_t dim = pool->dim;
  CUtensorMap mq, mkv;
  const cuuint64_t dims[2] = {dim, pool_rows}, strides[1] = {dim * 2};
  if (!opt::make_rows_map(&mq, f16, q, rows, heads, dim, q_stride, (int)(heads / pool->kv), plan.nodes) ||
      !opt::make_map(&mkv, f16, pool->base, 2, dims, strides, kPageTokens, 1))
    return fail(YUE2_ERR_INVALID, "q or the KV pool cannot be described to the copy engine (base, strides)");
  TreeArgs a = {};
  a.out = (uint16_t*)out;
  a.pool = v.base;
  a.table = table;
  a.context = context;
  a.cu = cu;
  a.mask = mask;
  a.status = status;
  a.part = (float*)workspace;
  a.out_stride = (long long)out_stride;
  a.pages = v.pages;
  a.page_stride = v.page_stride;
  a.table_pages = (long long)table_pages;
  a.seqs = (int)seqs;
  a.rows = (int)rows;
  a.heads = (int)heads;
  a.kv = v.kv;
  a.group = (int)(heads / pool->kv);
  a.nodes = plan.nodes;
  a.layer = (int)layer;
  a.blocks = v.blocks;
  a.negate = scale < 0.f;
  a.ctas = plan.ctas;
  a.slot_rows = plan.slot_rows;
  a.c = opt::weight_scale(scale);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool merge = plan.bytes > 0;
  if (dim == 64) return f16 ? launch<64, true>(mq, mkv, a, merge, st) : launch<64, false>(mq, mkv, a, merge, st);
  return f16 ? launch<128, true>(mq, mkv, a, merge, st) : launch<128, false>(mq, mkv, a, merge, st);
}

}  // extern "C"
