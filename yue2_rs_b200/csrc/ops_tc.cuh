// Tensor-core pieces of the attention operators: 128-row score tiles in TMEM, the softmax
// step over one of them, bounded waits that end the whole CTA, and the operand descriptors.
//
// A side (128 query rows, one per TMEM lane and thread) owns 128 columns of scores S and D
// columns of output O in TMEM. S = Q.K^T comes from shared memory (both K-major); the
// probabilities go back over S as packed 16-bit pairs and are the A operand of O += P.V from
// TMEM, V being the [keys][dim] tile as it lies in memory (the MN-major B operand).
#pragma once
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>

#include "ops.cuh"
#include "tcgen05.cuh"

namespace y2 {
namespace opt {

constexpr int kRows = 128;   // query rows of a side
constexpr int kKeys = 128;   // keys of a K or V tile
constexpr int kTmemCols = 512;
__host__ __device__ constexpr int s_col(int side) { return 128 * side; }  // scores, then weights over them
__host__ __device__ constexpr int o_col(int side) { return 256 + 128 * side; }
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

// One lane of the (converged) warp. The warp that issues products runs its control flow with all
// lanes, so that descriptors stay in uniform registers, and only the instructions with one:
// issued from a branch that one lane had taken, each product cost about 75 cycles.
Y2_DEV bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\tselp.u32 %0, 1, 0, e;\n\t}"
      : "=r"(p));
  return p != 0;
}
// A value that every lane holds, for the compiler to know it.
Y2_DEV uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

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

// S = Q.K^T of one side: Q and K in slabs of [128 rows][64 dims]. 128 keys a product: with 64
// the reads of Q from shared memory (4 KB a product) would hold the tensor cores to 2/3.
template <int D, bool F16>
Y2_DEV void issue_scores(uint32_t tmem_s, uint32_t qs, uint32_t ks) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) {
    const uint32_t off = (kk >> 2) * (kRows * 128) + (kk & 3) * 32;
    tc::mma_bf16(tmem_s, tc::sdesc_sw128(qs + off), tc::sdesc_sw128(ks + off), idesc<F16>(kKeys, false), kk > 0);
  }
}
// O (+)= P.V of one side over the keys [16 k0, 16 k1) of a tile.
template <int D, bool F16>
Y2_DEV void issue_values(uint32_t tmem_o, uint32_t tmem_p, uint32_t vs, int k0, int k1, bool accumulate) {
#pragma unroll
  for (int kk = k0; kk < k1; ++kk)
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
Y2_DEV void store16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
Y2_DEV void wait_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

Y2_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The running statistics of a thread's row: m is the score that the exponent is taken
// relative to (not always the maximum so far, see move_max), l the sum of the weights in parts.
// live: the lane's row is one of the call's (the others hold anything and decide nothing).
struct RowStats {
  float m, l[4];
  bool live;
  Y2_DEV void begin(bool is_live) { m = -INFINITY, l[0] = l[1] = l[2] = l[3] = 0.f, live = is_live; }
  Y2_DEV float total() const { return (l[0] + l[1]) + (l[2] + l[3]); }
};

// Pairs of f32 in one instruction.
Y2_DEV void fma2(float& x, float& y, float ax, float ay, float bx, float by, float cx, float cy) {
  asm("{\n\t.reg .b64 s, t, u;\n\t"
      "mov.b64 s, {%2, %3};\n\tmov.b64 t, {%4, %5};\n\tmov.b64 u, {%6, %7};\n\t"
      "fma.rn.f32x2 s, s, t, u;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "=f"(x), "=f"(y)
      : "f"(ax), "f"(ay), "f"(bx), "f"(by), "f"(cx), "f"(cy));
}
Y2_DEV void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 s, t;\n\t"
      "mov.b64 s, {%0, %1};\n\tmov.b64 t, {%2, %3};\n\t"
      "add.rn.f32x2 s, s, t;\n\tmov.b64 {%0, %1}, s;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}

// The largest of three, NaN if one of them is.
Y2_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x of two values on the FMA units: x = n + f with n the nearest integer and |f| <= 1/2, 2^f by
// a polynomial fitted for the least relative error (degree 3 for bf16 weights: 7.5e-5, degree
// 4 for f16: 2.6e-6; the rounding that follows is off by up to 3.9e-3 and 4.9e-4), and n added to its
// exponent. x is below about 100 and not NaN. From -127 down the result is 0, so that a key whose
// score is -inf adds nothing however large its value is: there n = -127 and f = 0, and since both
// constant terms are below 1 the sum of the exponents is negative, which max() turns into 0. (A
// select on x instead keeps x alive and spilled 40 to 70 bytes a thread.)
template <bool F16>
Y2_DEV void poly_ex2(float& x, float& y) {
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23: adding it leaves n in the low bits
  x = fmaxf(x, -127.f);
  y = fmaxf(y, -127.f);
  float nx = x, ny = y;
  add2(nx, ny, kRound, kRound);
  float rx = nx, ry = ny;
  add2(rx, ry, -kRound, -kRound);
  float fx, fy, px, py;
  fma2(fx, fy, rx, ry, -1.f, -1.f, x, y);
  if constexpr (F16) {
    fma2(px, py, 0x1.399776p-7f, 0x1.399776p-7f, fx, fy, 0x1.ca143ep-5f, 0x1.ca143ep-5f);
    fma2(px, py, px, py, fx, fy, 0x1.ec06dcp-3f, 0x1.ec06dcp-3f);
    fma2(px, py, px, py, fx, fy, 0x1.62e0dcp-1f, 0x1.62e0dcp-1f);
    fma2(px, py, px, py, fx, fy, 0x1.ffffe8p-1f, 0x1.ffffe8p-1f);
  } else {
    fma2(px, py, 0x1.c3f694p-5f, 0x1.c3f694p-5f, fx, fy, 0x1.f0de16p-3f, 0x1.f0de16p-3f);
    fma2(px, py, px, py, fx, fy, 0x1.62f31cp-1f, 0x1.62f31cp-1f);
    fma2(px, py, px, py, fx, fy, 0x1.fff692p-1f, 0x1.fff692p-1f);
  }
  x = __int_as_float(max((int)(__float_as_uint(px) + (__float_as_uint(nx) << 23)), 0));
  y = __int_as_float(max((int)(__float_as_uint(py) + (__float_as_uint(ny) << 23)), 0));
}

// c (a - b), whose difference may pass the end of f32 where the product does not (scores near it, a
// scale near 0). c is at most a quarter of the largest number.
Y2_DEV float apart(float c, float a, float b) { return fmaf(a, 0.25f, -0.25f * b) * (4.0f * c); }

// A new maximum mn of a row (NaN moves m too; a row that has seen nothing yet stays): m moves, and O
// and l are scaled by 2^(c (m_old - m_new)), only when a score exceeds m by more than a factor
// 2^8 of weight: until then the weights are at most 2^8, exact in the f32 sums, and the final
// division by l removes the factor. So most tiles leave O alone. O is settled: the P.V of the
// previous tile was issued before the scores of this one.
template <int D>
Y2_DEV void move_max(uint32_t o_addr, float c, bool first, float mn, RowStats& st) {
  const bool move = first || (st.live && mn != -INFINITY && !(apart(c, mn, st.m) <= 8.0f));
  if (!first && __any_sync(0xffffffffu, move)) {
    const float alpha = move ? ex2(apart(c, st.m, mn)) : 1.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) st.l[i] *= alpha;
#pragma unroll 1
    for (int q = 0; q < D; q += 16) {
      uint32_t o[16];
      tc::tmem_ld16(o_addr + q, o);
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
      store16(o_addr + q, o);
    }
  }
  if (move) st.m = mn;
}

// Exponents of f16 weights are 7 higher: weights reach 2^8 (move_max), so 2^15 at most, and those down
// to 2^-21 of the reference instead of 2^-14 are normal numbers (of several thousand keys, each
// 2^-25 of the largest, nothing was left). The division by l removes it. bf16 has f32's range.
template <bool F16>
constexpr float kLift = F16 ? 7.f : 0.f;
// Whether c s - c m, one FMA, is the exponent of a score s. c m is rounded, so that all weights formed
// relative to this m share a factor of up to 2^(c m 2^-24). The division by l removes it, except
// beside tiles with another m: below 2^12 it is at most 2^(2^-12), a third of half a step of f16. An
// infinite or NaN m is out of range, too.
Y2_DEV bool in_range(float c, float m) { return fabsf(c * m) < 0x1p12f; }
// The exponent of any row: (a s + b) k + kLift. An m of +inf or NaN makes the row NaN; an m of -inf
// (no score above it yet) gives every weight 0.
struct Exponent {
  float a, b, k;
  Y2_DEV Exponent(float c, float m) {
    const bool plain = in_range(c, m) || m == -INFINITY;
    a = plain ? c : 0.25f;
    b = m == -INFINITY ? 0.f : plain ? -c * m : -0.25f * m;
    k = plain ? 1.f : 4.f * c;
  }
};

// A side's softmax over one tile of 128 keys: the scores in TMEM become weights
// p = 2^(c (s - m)), packed over them. c = |scale| log2(e), see weight_scale. Every lane of the
// warp takes part. The maximum first (m starts as the first tile's), then the weights in a second
// pass over the scores in TMEM (reading them again costs less than holding 128 registers). False,
// and nothing done, when a row's maximum is out of range: softmax_masked does the tile. p is
// rounded to 16 bits (relative error of half a step, as the output's own rounding, and for f16 the
// range of kLift; l sums the unrounded weights). kPoly of 16 pairs take the FMA units, the others
// the special-function unit (trees, captured, with 0 / 1 / 2 / 4 of 16: full trees 65.4 / 60.0 /
// 63.9 / 59.1 us, a batch 44.9 / 42.5 / 45.0 / 42.3). In packed attention's softmax_settled they gain
// nothing: 8,192 rows of 24 heads 760 us with none and 773 with 2, prompt pair 30.1 and 29.8.
// part() runs when 96 weights are stored; the caller announces the last 32.
constexpr int kPoly = 1;
template <int D, bool F16, class Part>
Y2_DEV bool softmax_tile(uint32_t s_addr, uint32_t o_addr, float c, bool first, RowStats& st, Part part) {
  uint32_t v[2][32];
  float mx[4] = {st.m, st.m, st.m, st.m};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load32(s_addr + 64 * h, v[0]);
    load32(s_addr + 64 * h + 32, v[1]);
    wait_loads();
    arrived(v[0]);
    arrived(v[1]);
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      mx[0] = max3(mx[0], __uint_as_float(v[0][i]), __uint_as_float(v[0][i + 1]));
      mx[1] = max3(mx[1], __uint_as_float(v[0][i + 2]), __uint_as_float(v[0][i + 3]));
      mx[2] = max3(mx[2], __uint_as_float(v[1][i]), __uint_as_float(v[1][i + 1]));
      mx[3] = max3(mx[3], __uint_as_float(v[1][i + 2]), __uint_as_float(v[1][i + 3]));
    }
  }
  const float mn = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
  if (__any_sync(0xffffffffu, st.live && !in_range(c, mn))) return false;
  load32(s_addr, v[0]);
  move_max<D>(o_addr, c, first, mn, st);
  const float mc = fmaf(-c, st.m, kLift<F16>);
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    uint32_t(&s)[32] = v[q & 1];
    wait_loads();
    arrived(s);
    if (q < 3) load32(s_addr + 32 * (q + 1), v[(q + 1) & 1]);
    uint32_t p[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      fma2(a, b, __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]), c, c, mc, mc);
      if (i % (16 / kPoly) == 16 / kPoly - 1) {
        poly_ex2<F16>(a, b);
      } else {
        a = ex2(a);
        b = ex2(b);
      }
      add2(st.l[2 * (i & 1)], st.l[2 * (i & 1) + 1], a, b);
      p[i] = pack16<F16>(a, b);
    }
    store16(s_addr + 16 * q, p);
    if (q == 2) part();
  }
  return true;
}

// The same where rows do not see every key (bit i of `vis`), the scale is negative, or the others
// turned a tile down. UNROLL 1 keeps it small, as its instructions come from far away (tree attention:
// full trees 65.4 -> 62.6 us; packed attention is as fast with 4).
template <int D, bool F16, int UNROLL, class Part>
Y2_DEV void softmax_masked(uint32_t s_addr, uint32_t o_addr, float c, bool negate, bool first, const uint32_t (&vis)[4],
                           RowStats& st, Part part) {
  const uint32_t sign = negate ? 0x80000000u : 0u;
  uint32_t v[32];
  auto take = [&](int q) {
    const uint32_t bits = vis[q];
    load32(s_addr + 32 * q, v);
    wait_loads();
    arrived(v);
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = bits >> i & 1 ? v[i] ^ sign : 0xff800000u;
  };
  float mx = st.m, my = st.m;
#pragma unroll UNROLL
  for (int q = 0; q < 4; ++q) {
    if (__all_sync(0xffffffffu, vis[q] == 0)) continue;
    take(q);
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      mx = max3(mx, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
      my = max3(my, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
    }
  }
  move_max<D>(o_addr, c, first, max3(mx, my, my), st);
  const Exponent e(c, st.m);
#pragma unroll UNROLL
  for (int q = 0; q < 4; ++q) {
    uint32_t p[16];
    if (__all_sync(0xffffffffu, vis[q] == 0)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = 0;
    } else {
      take(q);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        float a, b;
        fma2(a, b, __uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), e.a, e.a, e.b, e.b);
        fma2(a, b, a, b, e.k, e.k, kLift<F16>, kLift<F16>);
        a = ex2(a);
        b = ex2(b);
        add2(st.l[2 * (i & 1)], st.l[2 * (i & 1) + 1], a, b);
        p[i] = pack16<F16>(a, b);
      }
    }
    store16(s_addr + 16 * q, p);
    if (q == 2) part();
  }
}

// The same for a tile that every row sees whole, with a positive scale, after the first one: the
// weights are formed relative to the m there is, the maximum is found on the way, and only
// when it asks for another m (false: nothing has been written) softmax_masked does the tile.
// The vote also turns down an m out of range: after tiles without any weight (scores of -inf) m is
// -inf, which no weight can be taken relative to.
// Without the first pass the exponentials start as soon as the scores are there (8,192 rows of
// 24 heads, all seen, when this form was added: 756 -> 716 us in bursts). Only long packed
// sequences gain: in tree attention the larger code cost more than the pass (65.2 -> 67.8 us).
template <int D, bool F16, class Part>
Y2_DEV bool softmax_settled(uint32_t s_addr, float c, RowStats& st, Part part) {
  const float mc = in_range(c, st.m) ? fmaf(-c, st.m, kLift<F16>) : NAN;
  uint32_t v[2][32], p[3][16];
  float l[4] = {0.f, 0.f, 0.f, 0.f}, mx = -INFINITY, my = -INFINITY;
  auto weights = [&](float a, float b, int i, float (&sum)[4]) {
    a = ex2(a);
    b = ex2(b);
    add2(sum[2 * (i & 1)], sum[2 * (i & 1) + 1], a, b);
    return pack16<F16>(a, b);
  };
  load32(s_addr, v[0]);
#pragma unroll
  for (int q = 0; q < 3; ++q) {
    uint32_t(&s)[32] = v[q & 1];
    wait_loads();
    arrived(s);
    load32(s_addr + 32 * (q + 1), v[(q + 1) & 1]);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a, b;
      fma2(a, b, __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]), c, c, mc, mc);
      if (i & 1) mx = max3(mx, a, b);
      else my = max3(my, a, b);
      p[q][i] = weights(a, b, i, l);
    }
  }
  uint32_t(&s)[32] = v[1];
  float x[32];
  wait_loads();
  arrived(s);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    fma2(x[2 * i], x[2 * i + 1], __uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]), c, c, mc, mc);
    if (i & 1) mx = max3(mx, x[2 * i], x[2 * i + 1]);
    else my = max3(my, x[2 * i], x[2 * i + 1]);
  }
  if (__any_sync(0xffffffffu, st.live && !(max3(mx, my, my) <= 8.0f + kLift<F16>))) return false;
#pragma unroll
  for (int i = 0; i < 4; ++i) st.l[i] += l[i];
#pragma unroll
  for (int q = 0; q < 3; ++q) store16(s_addr + 16 * q, p[q]);
  part();
#pragma unroll
  for (int i = 0; i < 16; ++i) p[0][i] = weights(x[2 * i], x[2 * i + 1], i, st.l);
  store16(s_addr + 48, p[0]);
  return true;
}

// Key `r` of a V tile in shared memory (slabs of [128][64 dims], 128-byte swizzle), 64 dims of
// it (slab at `vs`), where some row of the side does not see it: a value that is not finite
// would reach those rows as 0 * inf, so it becomes zero here, and *found is set (before, for who
// reads the zero) for the rows that do see it to add it at the end. dead: no row sees the
// key, all of it becomes zero.
template <bool F16>
Y2_DEV void clean_values(unsigned char* vs, int r, bool dead, int* found) {
  if (dead) {
#pragma unroll
    for (int ch = 0; ch < 8; ++ch) *reinterpret_cast<uint4*>(vs + tc::sw128(r, ch)) = make_uint4(0, 0, 0, 0);
    return;
  }
  // x * 0 summed up is NaN when some x is not finite
  uint32_t acc[4] = {0, 0, 0, 0};
#pragma unroll
  for (int ch = 0; ch < 8; ++ch) {
    const uint4 w = *reinterpret_cast<const uint4*>(vs + tc::sw128(r, ch));
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (F16) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(acc[i]) : "r"(x[i]), "r"(0));
      else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(acc[i]) : "r"(x[i]), "r"(0));
    }
  }
  constexpr uint32_t EXP = F16 ? 0x7c00u : 0x7f80u;
  auto bad = [](uint32_t w) { return (w & EXP) == EXP || (w >> 16 & EXP) == EXP; };
  if (!(bad(acc[0]) || bad(acc[1]) || bad(acc[2]) || bad(acc[3]))) return;
  *(volatile int*)found = 1;
  __threadfence_block();
#pragma unroll 1
  for (int ch = 0; ch < 8; ++ch) {
    uint4 w = *reinterpret_cast<uint4*>(vs + tc::sw128(r, ch));
    uint32_t* x = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((x[i] & EXP) == EXP) x[i] &= 0xffff0000u;
      if ((x[i] >> 16 & EXP) == EXP) x[i] &= 0x0000ffffu;
    }
    *reinterpret_cast<uint4*>(vs + tc::sw128(r, ch)) = w;
  }
}

// Four lanes' rows, 64 bytes of each, stored 64 bytes at a time: lane i of the four ends up with
// the i-th 16 bytes of all four rows. (A row a lane, every store would touch 32 lines; the
// output of 256 rows took 7,000 cycles that way.) to[r]: row r of the four, null for none.
Y2_DEV void quad_rows(void* mine, char* (&to)[4]) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    to[r] = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), r, 4));
}
Y2_DEV void quad_store(char* const (&to)[4], int offset, uint4 (&v)[4]) {
  const int lane = threadIdx.x & 3;
#pragma unroll
  for (int d = 1; d < 4; d <<= 1)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & d) continue;
      const bool up = lane & d;
      uint4 s = up ? v[i] : v[i ^ d];
      s.x = __shfl_xor_sync(0xffffffffu, s.x, d);
      s.y = __shfl_xor_sync(0xffffffffu, s.y, d);
      s.z = __shfl_xor_sync(0xffffffffu, s.z, d);
      s.w = __shfl_xor_sync(0xffffffffu, s.w, d);
      if (up) v[i] = s;
      else v[i ^ d] = s;
    }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (to[r]) *reinterpret_cast<uint4*>(to[r] + offset + lane * 16) = v[r];
}
// 32 f32 as 16-bit values, 64 bytes.
template <bool F16>
Y2_DEV void pack32(const float (&f)[32], uint4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    v[i] = make_uint4(pack16<F16>(f[8 * i], f[8 * i + 1]), pack16<F16>(f[8 * i + 2], f[8 * i + 3]),
                      pack16<F16>(f[8 * i + 4], f[8 * i + 5]), pack16<F16>(f[8 * i + 6], f[8 * i + 7]));
}

// Adds the values of a key that are not finite (32 of them at `v`) to a row's outputs.
template <bool F16>
Y2_DEV void add_nonfinite(const uint16_t* v, float (&o)[32]) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    float x[8];
    unpack8<F16>(*reinterpret_cast<const uint4*>(v + i), x);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!isfinite(x[e])) o[i + e] += x[e];
  }
}

// ---- host
// c of the exponents. Not below the smallest normal number: a masked score is -inf, and 0 * -inf is
// not 0. Not above a quarter of the largest: differences of scores are taken in quarters, and
// with a c like that only the largest score has a weight anyway.
inline float weight_scale(float scale) {
  return std::min(std::max(std::fabs(scale) * 1.4426950408889634f, 1.17549435e-38f), 8.5e37f);
}
// Tensor map of 16-bit values [.., dims[1], dims[0]] (strides in bytes of the outer
// dimensions) in boxes of 64 x box1 x box2 values, 128-byte swizzle, zeros beyond the end. The
// driver's encoder is looked up through the runtime, so that the library loads without a driver.
inline bool make_map(CUtensorMap* m, bool f16, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                     cuuint32_t box1, cuuint32_t box2) {
  static std::atomic<void*> found{nullptr};
  void* fn = found.load(std::memory_order_relaxed);
  if (!fn) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return false;
    found.store(fn, std::memory_order_relaxed);
  }
  const cuuint32_t box[3] = {64, box1, box2}, step[3] = {1, 1, 1};
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn)(
             m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
             const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// [rows, heads, dim] values with a row stride in elements, in boxes of [box_rows][box_heads][64].
inline bool make_rows_map(CUtensorMap* m, bool f16, const void* base, uint64_t rows, uint64_t heads, uint64_t dim,
                          uint64_t stride, int box_heads, int box_rows) {
  const cuuint64_t dims[3] = {dim, heads, rows}, strides[2] = {dim * 2, stride * 2};
  return make_map(m, f16, base, 3, dims, strides, (cuuint32_t)box_heads, (cuuint32_t)box_rows);
}

}  // namespace opt
}  // namespace y2
