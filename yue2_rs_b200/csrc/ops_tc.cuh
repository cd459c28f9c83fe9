// Tensor-core pieces of the attention operators: 128-row score tiles in TMEM, the softmax
// step over one of them, bounded waits that end the whole CTA, and the operand descriptors.
//
// A side (128 query rows, one per TMEM lane and thread) owns 128 columns of scores S and D
// columns of output O in TMEM. S = Q.K^T comes from shared memory (both K-major); the
// probabilities go back over S as packed 16-bit pairs and are the A operand of O += P.V from
// TMEM, V being the [keys][dim] tile as it lies in memory (the MN-major B operand).
#pragma once
#include <cuda.h>

#include "ops.cuh"
#include "tcgen05.cuh"

namespace y2 {
namespace opt {

constexpr int kRows = 128;   // query rows of a side
constexpr int kKeys = 128;   // keys of a tile
constexpr int kTmemCols = 512;
__host__ __device__ constexpr int s_col(int side) { return 128 * side; }        // scores and probabilities
__host__ __device__ constexpr int o_col(int side) { return 256 + 128 * side; }  // outputs
// The block is launched with 12 warps of 168 registers (504 = 3 * 168 per lane of the three
// warpgroups); the two softmax warpgroups hold a row of 128 scores and take more, the warps
// that issue products and copies give theirs: 216 + 216 + 72 = 504.
constexpr int kThreads = 384;
Y2_DEV void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 216;"); }
Y2_DEV void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 72;"); }
constexpr long long kWaitCycles = 4000000000ll;  // about two seconds: a wait this long has failed

// Waits for the phase of the given parity; false when the CTA is ending. A wait that lasts too
// long ends it and reports.
Y2_DEV bool wait(uint64_t* bar, uint32_t parity, volatile int* ending, int32_t* status) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (tc::mbar_try_wait(bar, parity)) return true;
    if (*ending) return false;
    if (clock64() - t0 > kWaitCycles) {
      status_or(status, YUE2_STATUS_STALL);
      *ending = 1;
      return false;
    }
  }
}

// The same for what is in flight when the CTA ends: it has to arrive whatever happened.
Y2_DEV void settle(uint64_t* bar, uint32_t parity, int32_t* status) {
  for (long i = 0; i < 1L << 22; ++i)
    if (tc::mbar_try_wait(bar, parity)) return;
  status_or(status, YUE2_STATUS_STALL);
}

Y2_DEV void tma_load_3d(void* dst, const void* map, uint64_t* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
          tc::smem_u32(dst)),
      "l"((uint64_t)map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Instruction descriptor of kind::f16 with f32 accumulation, M 128; b_mn: B is MN-major.
template <bool F16>
__host__ __device__ constexpr uint32_t idesc(int N, bool b_mn) {
  return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(kRows >> 4) << 24);
}
// B descriptor of a V tile in slabs of [128 keys][64 dims] (128-byte swizzle): 64-dim chunks
// one slab apart (leading offset), 8-key groups 1024 B apart (stride offset). A step of 16
// keys adds 2048 B to the start.
Y2_DEV uint64_t vdesc(uint32_t saddr) {
  uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
  d |= (uint64_t)((kKeys * 128) >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// D[tmem] (+)= A[tmem] . B[smem], issued by one thread.
Y2_DEV void mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t id, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(id), "r"(accumulate)
      : "memory");
}

// S = Q.K^T of one side: Q and K in slabs of [128 rows][64 dims].
template <int D, bool F16>
Y2_DEV void issue_scores(uint32_t tmem_s, uint32_t qs, uint32_t ks) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = (kk >> 2) * (kRows * 128) + (kk & 3) * 32;
    tc::mma_bf16(tmem_s, tc::sdesc_sw128(qs + off), tc::sdesc_sw128(ks + off), idesc<F16>(kKeys, false), kk > 0);
  }
}
// O (+)= P.V of one side.
template <int D, bool F16>
Y2_DEV void issue_values(uint32_t tmem_o, uint32_t tmem_p, uint32_t vs, bool accumulate) {
#pragma unroll
  for (int kk = 0; kk < kKeys / 16; ++kk)
    mma_ts(tmem_o, tmem_p + kk * 8, vdesc(vs + kk * 2048), idesc<F16>(D, true), accumulate || kk > 0);
}

// 32 columns of this thread's lane, in flight until wait_loads(); `arrived` orders the uses.
Y2_DEV void load32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),
        "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),
        "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
Y2_DEV void wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
Y2_DEV void arrived(uint32_t (&v)[32]) {
  asm volatile(""
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]),
                 "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]),
                 "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]),
                 "+r"(v[30]), "+r"(v[31])::"memory");
}
Y2_DEV void store32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
Y2_DEV void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

Y2_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The running statistics of a thread's row: m is the score that the exponent is taken
// relative to (not always the maximum so far, see below), l the sum of the weights.
struct RowStats {
  float m, l;
};

// One tile of a side's softmax: scores S in TMEM become weights p = 2^(c (s - m)), packed over
// S, and l += sum p. c = |scale| log2(e), `negate` for a negative scale. With `masked`, bit i of `vis`
// says whether the row sees key i of the tile. m moves, and O and l are scaled by 2^(c (m_old - m_new)),
// only when a score exceeds it by more than a factor 2^8 of weight: until then the
// weights are at most 2^8, exact in the f32 sums, and the final division by l removes the
// factor; so most tiles leave O alone. p is rounded to 16 bits (relative error of half a
// step, as the output's own rounding; l sums the unrounded weights). Every lane of the warp takes part.
template <int D, bool F16>
Y2_DEV void softmax_tile(uint32_t s_addr, uint32_t o_addr, float c, bool negate, bool first, bool masked,
                         const uint32_t (&vis)[4], RowStats& st) {
  uint32_t v[4][32];
#pragma unroll
  for (int q = 0; q < 4; ++q) load32(s_addr + 32 * q, v[q]);
  wait_loads();
#pragma unroll
  for (int q = 0; q < 4; ++q) arrived(v[q]);
  if (negate) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 32; ++i) v[q][i] ^= 0x80000000u;
  }
  if (masked) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!(vis[q] >> i & 1)) v[q][i] = 0xff800000u;
  }
  float mx[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    mx[q] = __uint_as_float(v[q][0]);
#pragma unroll
    for (int i = 1; i < 32; ++i) mx[q] = fmaxf(mx[q], __uint_as_float(v[q][i]));
  }
  const float mn = fmaxf(st.m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])));
  const bool move = first || (mn - st.m) * c > 8.0f;
  if (!first && __any_sync(0xffffffffu, move)) {
    const float alpha = move ? ex2((st.m - mn) * c) : 1.0f;
    st.l *= alpha;
#pragma unroll
    for (int q = 0; q < D / 32; ++q) {
      uint32_t o[32];
      load32(o_addr + 32 * q, o);
      wait_loads();
      arrived(o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
      store32(o_addr + 32 * q, o);
    }
  }
  if (move) st.m = mn;
  const float mc = st.m == -INFINITY ? 0.f : st.m * c;
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t p[2][32];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float a = ex2(fmaf(__uint_as_float(v[q][i]), c, -mc)), b = ex2(fmaf(__uint_as_float(v[q][i + 1]), c, -mc));
      sum[q] += a;
      sum[q] += b;
      p[q >> 1][(q & 1) * 16 + i / 2] = pack16<F16>(a, b);
    }
  st.l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  store32(s_addr, p[0]);
  store32(s_addr + 32, p[1]);
  wait_stores();
}

// Key `r` of a V tile in shared memory (slabs of [128][64 dims], 128-byte swizzle) where some
// row of the tile does not see it: a value that is not finite would reach those rows as
// 0 * inf, so it becomes zero here, and true is returned for the rows that do see it to add
// it at the end. dead: no row sees the key, all of it becomes zero.
template <int D, bool F16>
Y2_DEV bool clean_value_row(unsigned char* vs, int r, bool dead) {
  constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
  bool found = false;
#pragma unroll
  for (int s = 0; s < D / 64; ++s)
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) {
      uint4* at = reinterpret_cast<uint4*>(vs + s * (kKeys * 128) + tc::sw128(r, ch));
      if (dead) {
        *at = make_uint4(0, 0, 0, 0);
        continue;
      }
      uint4 w = *at;
      uint32_t* x = reinterpret_cast<uint32_t*>(&w);
      bool bad = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if ((x[i] & EXP) == EXP) x[i] &= 0xffff0000u, bad = true;
        if ((x[i] >> 16 & EXP) == EXP) x[i] &= 0x0000ffffu, bad = true;
      }
      if (bad) *at = w, found = true;
    }
  return found;
}

// Adds the values of a key that are not finite (32 of them at `v`) to a row's outputs.
template <bool F16>
Y2_DEV void add_nonfinite(const uint16_t* v, float (&o)[32]) {
  for (int i = 0; i < 32; i += 8) {
    float x[8];
    unpack8<F16>(*reinterpret_cast<const uint4*>(v + i), x);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!isfinite(x[e])) {
#pragma unroll
        for (int k = 0; k < 32; k += 8)
          if (k == i) o[k + e] += x[e];
      }
  }
}

}  // namespace opt
}  // namespace y2
