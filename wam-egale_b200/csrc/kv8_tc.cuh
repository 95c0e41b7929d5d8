// Attention over the E4M3 cache for more than a few query rows, on the
// tcgen05 tensor cores. The mathematics, the rows of a query tile and the
// stream-K line of units are those of kv8_few.cuh, with tiles of 256 rows and
// units of 128 keys.
//
// S = Q K^T reads K's codes as they lie in the cache (kind::f8f6f4, no
// conversion): q 2^-n = hi + lo, hi the nearest E4M3 value and lo the nearest
// E5M2 value of what it leaves, so S = (hi K^T + lo K^T) 2^n costs what one
// bf16 product does. n puts the row's largest magnitude in (224, 448]. From
// 2^-6 on (2^-13.8 of the largest, or less) hi + lo has all eight bits of a bf16 query:
// hi has four, and what it leaves is at most 8 units in the last of the eight,
// which E5M2's three bits hold. Below, hi leaves at most 2^-10 and lo is off by
// half its step, 2^-14 (2^-21 of the row's largest). With E4M3 for lo, whose
// steps end at 2^-9, the error was 2^-10 already from 2^-2 down. The products
// are summed in full fp32 here (measured: 9e-9 relative error against 64 bits
// at K 128, bf16's is 1.2e-7).
// O += P V needs more range than two E4M3 pieces of P hold (a long flat tail
// beside a sharp maximum), so P is f16 as in kv8_few.cuh and V's codes become
// f16 in shared memory, once for 256 rows, by two warps of their own.
//
// One CTA per SM, 384 threads:
//   warps 0..7   softmax, one thread per query row: warps 0-3 on TMEM slot A,
//                warps 4-7 on slot B
//   warp 8       producer: page ids and scales (read four tiles ahead), TMA
//                of the queries' pieces (split once by kv8_split_q_kernel)
//                and of K and V codes, the scales of each 16 keys to a ring
//   warp 9       issues the MMAs
//   warps 10, 11 V codes -> f16
// With more than 128 rows, slot A and slot B hold the tile's two halves and
// meet every key tile; with fewer, both hold the same rows and take the key
// tiles in turn (joined at the end), so that one slot's softmax always runs
// beside the other's products. In both cases the work is a row of steps, step
// s on slot s & 1: S(s + 2) is issued behind PV(s).
// TMEM columns: S/P of A [0,128), of B [128,256), O_A [256,384), O_B [384,512).
//
// Bound by the latency of the chain S -> softmax -> P -> PV of a slot (two softmax
// warps a scheduler; issue active 36%, tensor pipe 41%): a key tile of 256 rows
// takes about 5000 cycles where its MMAs take 2048. 8 x 880 rows over up to 4400 keys of 24 heads (297 GFLOP): 434 us, 0.68
// PFLOP/s, 19 of them the split of the queries; 32 rows of 4 sequences (75 MB
// of cache) 44 us. Slower forms of the same chain, at that size and before the
// last 30 us were taken elsewhere (this one: 468): P through shared memory 549
// to 590 (two or one buffers), PV in two halves 556, scores in 64-key halves
// 753, V's codes read by the converting warps from global memory 505, an eighth
// of the exponentials as a polynomial 510, no register split 758.
#pragma once
#include "attention.cuh"
#include "glue.cuh"
#include "kv8_few.cuh"
#include <type_traits>

namespace wamb {

constexpr int KTC_THREADS = 384, KTC_QR = 256, KTC_TK = 128;
constexpr uint32_t KTC_TILE8 = 128 * 128;      // 128 rows of 128 codes
constexpr int KTC_SCS = 8;     // key tiles whose scales are kept; K, V and f16 V have rings of two

struct KtcSmem {
  static constexpr uint32_t Q_OFF = 0;                                       // slot A hi, lo, slot B hi, lo
  static constexpr uint32_t K_OFF = Q_OFF + 4 * KTC_TILE8;
  static constexpr uint32_t V8_OFF = K_OFF + 2 * KTC_TILE8;
  static constexpr uint32_t V16_OFF = V8_OFF + 2 * KTC_TILE8;
  static constexpr uint32_t STAGE_OFF = V16_OFF + 4 * KTC_TILE8;   // output rows, 4 KB a softmax warp; before them m, l of both slots
  static constexpr uint32_t SC_OFF = STAGE_OFF + 8 * 4096;         // [8 tiles] ks, log2 vs, 1 / vs of 8 groups of 16 keys
  static constexpr uint32_t BAR_OFF = SC_OFF + KTC_SCS * 128;
  static constexpr uint32_t NBARS = 12 + 2 + 2 + 5 + KTC_SCS;
  static constexpr uint32_t SCHED_OFF = BAR_OFF + NBARS * 8;
  static constexpr uint32_t TOTAL = 1024 + SCHED_OFF + sizeof(Kv8SchedSmem) + 16;
  static_assert(TOTAL <= 232448, "shared memory exceeds 227 KB");
};

// kind::f16 instruction descriptor with f16 operands, B MN-major.
__host__ __device__ constexpr uint32_t idesc_f16_mn(int M, int N) {
  return (1u << 4) | (1u << 16) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// Low and high words of the swizzled operand descriptors (sw128_desc): the low
// one moves with the address, the high one is a constant, so that an MMA costs
// its issuing thread one addition.
constexpr uint32_t KTC_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
WAMB_DEV uint32_t ktc_desc_lo(uint32_t addr, uint32_t lbo) { return (addr >> 4) | ((lbo >> 4) << 16); }

// S [128 rows][128 keys] = (hi + lo) K^T: 4 x 32 dims of each piece. The
// instruction descriptor's type fields: A in bits 7-9, B in 10-12, 1 is E5M2.
WAMB_DEV void ktc_issue_s(uint32_t d, uint32_t q, uint32_t k) {
  constexpr uint32_t IDESC = idesc_e4m3(128, 128), IDESC_LO = IDESC | (1u << 7);
  const uint32_t qd = ktc_desc_lo(q, 16), kd = ktc_desc_lo(k, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(qd + (i >> 2) * (KTC_TILE8 >> 4) + (i & 3) * 2), "r"(kd + (i & 3) * 2), "n"(KTC_DESC_HI), "r"(i < 4 ? IDESC : IDESC_LO),
        "r"(i > 0 ? 1u : 0u)
        : "memory");
}
// S^T [128 keys][128 rows] = K (hi + lo)^T.
WAMB_DEV void ktc_issue_st(uint32_t d, uint32_t k, uint32_t q) {
  constexpr uint32_t IDESC = idesc_e4m3(128, 128), IDESC_LO = IDESC | (1u << 10);
  const uint32_t qd = ktc_desc_lo(q, 16), kd = ktc_desc_lo(k, 16);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(kd + (i & 3) * 2), "r"(qd + (i >> 2) * (KTC_TILE8 >> 4) + (i & 3) * 2), "n"(KTC_DESC_HI), "r"(i < 4 ? IDESC : IDESC_LO),
        "r"(i > 0 ? 1u : 0u)
        : "memory");
}
// O [128 rows][128 dims] (+)= P V: P in TMEM, 8 x 16 keys (rows of V past the
// live keys are zero, and so is P).
WAMB_DEV void ktc_issue_pv(uint32_t d, uint32_t pt, uint32_t v, bool accumulate) {
  constexpr uint32_t IDESC = idesc_f16_mn(128, 128);
  const uint32_t vd = ktc_desc_lo(v, KTC_TILE8), acc = accumulate;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(pt + 8 * i), "r"(vd + i * (2048 >> 4)), "n"(KTC_DESC_HI), "n"(IDESC), "r"(i > 0 ? 1u : acc)
        : "memory");
}

// One lane of the converged warp, always the same.
WAMB_DEV bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}

WAMB_DEV void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

WAMB_DEV float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair on the FMA pipe: x clamped to >= -125 (NaN stays), x = n + f
// with |f| <= 1/2 by the 1.5 * 2^23 shifter, 2^f by the polynomial of degree 5
// with the smallest largest relative error (Remez exchange; 1.6e-7 with fp32
// coefficients, recomputed by tests/test_host_exp2_poly5.py), times 2^n put
// together from its exponent bits.
constexpr float KTC_C0 = 1.0000001192092896f;
constexpr float KTC_C1 = 0.6931469440460205f;
constexpr float KTC_C2 = 0.24022120237350464f;
constexpr float KTC_C3 = 0.05550713092088699f;
constexpr float KTC_C4 = 0.009675540961325169f;
constexpr float KTC_C5 = 0.0013276472454890609f;
WAMB_DEV uint64_t ex2_poly5(uint64_t x2) {
  const float2 xv = f2_split(x2);
  const uint64_t x = f2(max3_nan(xv.x, -125.f, -125.f), max3_nan(xv.y, -125.f, -125.f));
  const uint64_t shifter = f2(12582912.f, 12582912.f);
  const uint64_t t = fadd2(x, shifter);
  const uint64_t f = fsub2(x, fsub2(t, shifter));
  uint64_t p = ffma2(f, f2(KTC_C5, KTC_C5), f2(KTC_C4, KTC_C4));
  p = ffma2(p, f, f2(KTC_C3, KTC_C3));
  p = ffma2(p, f, f2(KTC_C2, KTC_C2));
  p = ffma2(p, f, f2(KTC_C1, KTC_C1));
  p = ffma2(p, f, f2(KTC_C0, KTC_C0));
  const float2 tv = f2_split(t);
  return fmul2(p, f2(__int_as_float((__float_as_int(tv.x) << 23) + 0x3f800000),
                     __int_as_float((__float_as_int(tv.y) << 23) + 0x3f800000)));
}

// Four values into their E4M3 code word `h` and the E5M2 word of what it leaves.
WAMB_DEV void split_8bit_x4(const float (&x)[4], uint32_t& h, uint32_t& l) {
  const uint32_t h0 = __nv_cvt_float2_to_fp8x2(make_float2(x[0], x[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t h1 = __nv_cvt_float2_to_fp8x2(make_float2(x[2], x[3]), __NV_SATFINITE, __NV_E4M3);
  const float2 f0 = e4m3x2_to_float2(h0), f1 = e4m3x2_to_float2(h1);
  const uint32_t l0 = __nv_cvt_float2_to_fp8x2(make_float2(x[0] - f0.x, x[1] - f0.y), __NV_SATFINITE, __NV_E5M2);
  const uint32_t l1 = __nv_cvt_float2_to_fp8x2(make_float2(x[2] - f1.x, x[3] - f1.y), __NV_SATFINITE, __NV_E5M2);
  h = h0 | (h1 << 16);
  l = l0 | (l1 << 16);
}
// Exponent n and factor 2^-n that bring a query row's largest magnitude into
// (224, 448]. An infinite query makes its row NaN, as the formula does (a
// saturated one would not).
WAMB_DEV float query_scale(float amax, int& n) {
  const int bits = __float_as_int(fminf(amax, 3.402823466e38f));
  n = max(-118, min(119, (bits >> 23) - 135 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0)));
  return amax <= 3.402823466e38f ? pow2f_exact(-n) : __int_as_float(0x7fffffff);
}

// The queries in two 8-bit pieces, for the tensor-core kernels: row
// (b * heads + h) * rows_pad + r of q8 [., 256] holds hi (128 codes) and lo of
// row r of (sequence b, cached head h), rf its factor 2^n * scale * log2(e);
// rows past the sequence's are zeros. With neg_lse2 (weights): -lse * log2(e),
// -inf for rows that add nothing. Eight lanes hold a row, 16 values each, and
// two rows at once: a warp on a row spent three quarters of its instructions on
// the row's place (45 us for the 169k rows of 8 x 880 tokens x 24 heads, 19 us now).
// Bound by memory (512 B a row) or by the launch.
__global__ void __launch_bounds__(256) kv8_split_q_kernel(const Kv8AttnParams p, const int rows_pad, const int total,
                                                          uint8_t* q8, float* rf, float* neg_lse2) {
  pdl_wait();
  pdl_trigger();   // the kernel behind it finds its work meanwhile (one chunk 92 -> 90 us)
  constexpr int AT_ONCE = 2;
  const int c = threadIdx.x & 7, first = blockIdx.x * (32 * AT_ONCE) + (threadIdx.x >> 3);
  uint4 w[AT_ONCE][2];
  float z[AT_ONCE];
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) {
    const int row = first + 32 * i;
    w[i][0] = w[i][1] = make_uint4(0, 0, 0, 0);
    z[i] = -INFINITY;
    if (row < total) {
      const int bh = row / rows_pad, r = row - bh * rows_pad;
      const int b = bh / p.c.heads, h = bh - b * p.c.heads;
      const int t = r / p.group, hq = h * p.group + r - t * p.group;
      if (t < kv8_count(p.s, b)) {
        const uint4* src = reinterpret_cast<const uint4*>(p.q + b * p.q_sb + t * p.q_st + hq * p.q_sh) + 2 * c;
        w[i][0] = __ldg(src);
        w[i][1] = __ldg(src + 1);
        if (neg_lse2 != nullptr)
          z[i] = __ldg(p.lse_in + (static_cast<long long>(b) * p.s.tokens + t) * (p.c.heads * p.group) + hq);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < AT_ONCE; ++i) {
    const int row = first + 32 * i;
    const uint32_t ws[8] = {w[i][0].x, w[i][0].y, w[i][0].z, w[i][0].w, w[i][1].x, w[i][1].y, w[i][1].z, w[i][1].w};
    float2 v[8];
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = unpack_bf16(ws[k]);
      amax = fmaxf(amax, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    int n;
    const float up = query_scale(amax, n);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x[4] = {v[2 * k].x * up, v[2 * k].y * up, v[2 * k + 1].x * up, v[2 * k + 1].y * up};
      split_8bit_x4(x, hi[k], lo[k]);
    }
    if (row >= total) continue;
    uint4* dst = reinterpret_cast<uint4*>(q8 + static_cast<long long>(row) * 256) + c;
    dst[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    dst[8] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    if (c == 0) {
      rf[row] = pow2f_exact(n) * p.scale_log2;
      if (neg_lse2 != nullptr) neg_lse2[row] = z[i] == -INFINITY ? -INFINITY : z[i] * -1.4426950408889634f;
    }
  }
}

// One CTA's walk over the segments of its share.
template <int QR>
struct KtcWalk {
  Kv8Item it;
  long long u;
  WAMB_DEV bool done(const Kv8Share& sh) const { return u >= sh.u1; }
  WAMB_DEV void next(const Kv8AttnParams& p, const Kv8Share& sh) {
    u = min(sh.u1, it.start + it.n);
    if (u < sh.u1) kv8_seek<QR, KTC_TK>(p, it, u);
  }
};
struct KtcSeg {
  int b, qt, rows;     // sequence, query tile, its rows (1..256)
  int j0, n;           // key tiles [j0, j0 + n)
  int vis;             // keys that the tile's last row sees
  bool two;            // two query halves (rows > 128)
  bool begins, ends;
  WAMB_DEV KtcSeg(const Kv8AttnParams& p, const Kv8Share& sh, const KtcWalk<KTC_QR>& w) {
    b = w.it.e / p.qts;
    qt = w.it.e - b * p.qts;
    rows = min(KTC_QR, Kv8Line<KTC_QR, KTC_TK>::rows(p, b) - qt * KTC_QR);
    j0 = static_cast<int>(w.u - w.it.start);
    n = static_cast<int>(min(sh.u1, w.it.start + w.it.n) - w.u);
    vis = Kv8Line<KTC_QR, KTC_TK>::visible(p, w.it.e);
    two = rows > 128;
    begins = j0 == 0;
    ends = j0 + n == w.it.n;
  }
  WAMB_DEV int live(int j) const { return max(0, min(KTC_TK, vis - (j0 + j) * KTC_TK)); }
};

__global__ void __launch_bounds__(KTC_THREADS, 1)
    kv8_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmQ, const float* q_factor, const int rows_pad, const Kv8AttnParams p) {
  using L = KtcSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = smem_u32(smem);
  const uint32_t sQ = base + L::Q_OFF, sK = base + L::K_OFF, sV8 = base + L::V8_OFF, sV16 = base + L::V16_OFF;
  uint32_t bar = base + L::BAR_OFF;
  auto bars = [&](int n) { const uint32_t b = bar; bar += 8 * n; return b; };
  const uint32_t k_full = bars(2), k_empty = bars(2), v8_full = bars(2), v8_empty = bars(2), v16_full = bars(2), v16_empty = bars(2),
                 s_full = bars(2), p_full = bars(2), q_full = bars(1), q_free = bars(1), o_done = bars(1), o_free = bars(1),
                 drain = bars(1), sc_full = bars(KTC_SCS);
  Kv8SchedSmem& sched = *reinterpret_cast<Kv8SchedSmem*>(smem + L::SCHED_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::SCHED_OFF + sizeof(Kv8SchedSmem));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp: uniform

  // The split of the queries let this kernel start when everything before it
  // was complete: only what it writes is waited for.
  Kv8Share sh;
  KtcWalk<KTC_QR> walk;
  const bool work = kv8_share<KTC_QR, KTC_TK, KTC_THREADS>(p, blockIdx.x, sched, sh, walk.it);
  if (threadIdx.x == 0) kv8_leave_join(p, sh, work, walk.it);
  if (!work) {
    pdl_wait();    // the kernel is not complete before the split is
    return;
  }
  walk.u = sh.u0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
      mbar_init(v8_full + 8 * i, 1);
      mbar_init(v8_empty + 8 * i, 2);     // one arrival per converting warp
      mbar_init(v16_full + 8 * i, 2);
      mbar_init(v16_empty + 8 * i, 1);
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);       // one arrival per softmax warp of the slot
    }
    mbar_init(q_full, 1);
    mbar_init(q_free, 1);
    mbar_init(o_free, 8);
    mbar_init(o_done, 1);
    mbar_init(drain, 1);
    for (int i = 0; i < KTC_SCS; ++i) mbar_init(sc_full + 8 * i, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // The softmax warps hold a whole row of 128 scores: 256 threads x 208 and
  // 128 x 80 registers, within the launch's 384 x 168.
  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
  if (warp == 8) {
    // ---------------------------------------------------------- producer
    // Lane (to, gi) looks after keys [16 gi, +16) of tile `to` of a batch of four.
    const int to = lane >> 3, gi = lane & 7;
    const int box_groups = p.c.page >> 4;   // 16-key groups of one page
    int tiles = 0, queries = 0;             // key tiles and query tiles so far
    int k_loads = 0, v_loads = 0;           // loads issued: tiles, but for the last where a wait ran out
    bool go = true;
    for (int seg = 0; go && !walk.done(sh); walk.next(p, sh), ++seg) {
      const KtcSeg sg(p, sh, walk);
      const int h = walk.it.h;
      // The queries' pieces, once the last segment's scores are made.
      if (seg > 0) go = __all_sync(0xffffffffu, mbar_wait(q_free, (seg - 1) & 1, abort_flag));
      if (!go) break;
      if (lane == 0) {
        const int row = (sg.b * p.c.heads + h) * rows_pad + sg.qt * KTC_QR;
        mbar_arrive_expect_tx(q_full, (sg.two ? 4 : 2) * KTC_TILE8);
        tma_load_2d(sQ, &tmQ, q_full, 0, row);
        tma_load_2d(sQ + KTC_TILE8, &tmQ, q_full, 128, row);
        if (sg.two) {
          tma_load_2d(sQ + 2 * KTC_TILE8, &tmQ, q_full, 0, row + 128);
          tma_load_2d(sQ + 3 * KTC_TILE8, &tmQ, q_full, 128, row + 128);
        }
      }
      ++queries;
      // Page ids are read two batches ahead, scales one, so that no load is
      // waited for.
      struct Ahead { int row; float ks, vs; };   // row < 0: no keys
      auto page_of = [&](int j) {
        const int key = (sg.j0 + j + to) * KTC_TK + gi * 16;
        if (j + to >= sg.n || key >= sg.vis) return -1;
        return max(0, kv8_page(p.s.table, p.s.width, p.c, sg.b, key >> p.c.page_log2));   // a bad id is reported
      };
      auto load = [&](int j, int pid) {
        Ahead a{-1, 1.f, 1.f};
        if (pid >= 0) {
          const int key = (sg.j0 + j + to) * KTC_TK + gi * 16;
          const long long blk = static_cast<long long>(pid) * p.c.heads + h;
          a.row = static_cast<int>((blk << p.c.page_log2) + (key & (p.c.page - 1)));
          a.ks = __ldg(p.c.k_scale + blk);
          a.vs = __ldg(p.c.v_scale + blk);
        }
        return a;
      };
      Ahead now = load(0, page_of(0));
      int pid = page_of(4);
      for (int jb = 0; go && jb < sg.n; jb += 4) {
        const Ahead next = load(jb + 4, pid);
        pid = page_of(jb + 8);
        for (int i = 0; i < 4 && jb + i < sg.n; ++i, ++tiles) {
          const int sc = tiles % KTC_SCS;
          if (to == i) {   // [ks x 8][log2 vs x 8][1 / vs x 8]
            float* at = reinterpret_cast<float*>(smem + L::SC_OFF) + sc * 32 + gi;
            at[0] = now.ks;
            at[8] = log2f(now.vs);
            at[16] = 1.f / now.vs;
          }
          const bool lead = to == i && now.row >= 0 && gi % box_groups == 0;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, lead)) * (p.c.page * 128);
          __syncwarp();
          if (lane == 0) mbar_arrive(sc_full + 8 * sc);
          const int slot = tiles & 1;
          const uint32_t phase = (tiles >> 1) & 1;
          go = __all_sync(0xffffffffu, mbar_wait(k_empty + 8 * slot, phase ^ 1, abort_flag));
          if (!go) break;
          if (lane == 0) mbar_arrive_expect_tx(k_full + 8 * slot, bytes);
          __syncwarp();
          if (lead) tma_load_2d(sK + slot * KTC_TILE8 + gi * 2048, &tmK, k_full + 8 * slot, 0, now.row);
          ++k_loads;
          go = __all_sync(0xffffffffu, mbar_wait(v8_empty + 8 * slot, phase ^ 1, abort_flag));
          if (!go) break;
          if (lane == 0) mbar_arrive_expect_tx(v8_full + 8 * slot, bytes);
          __syncwarp();
          if (lead) tma_load_2d(sV8 + slot * KTC_TILE8 + gi * 2048, &tmV, v8_full + 8 * slot, 0, now.row);
          ++v_loads;
        }
        now = next;
      }
    }
    // Loads still in flight must land before the CTA exits, after a wait that ran out too.
    if (lane == 0) {
      if (queries > 0) mbar_wait_teardown(q_full, (queries - 1) & 1);
      for (int t = max(0, k_loads - 2); t < k_loads; ++t) mbar_wait_teardown(k_full + 8 * (t & 1), (t >> 1) & 1);
      for (int t = max(0, v_loads - 2); t < v_loads; ++t) mbar_wait_teardown(v8_full + 8 * (t & 1), (t >> 1) & 1);
    }
    __syncwarp();
  } else if (warp == 9) {
    // --------------------------------------------------------- MMA issuer
    // The whole warp walks the loop on values that are the same in every lane
    // (so that descriptors are computed in uniform registers) and one lane
    // issues: a lane alone in a divergent branch took ~110 cycles an MMA.
    const bool issuer = elect_one();
    uint32_t kq = 0, kpar = 0;      // K ring: slot and phase of the next score tile
    uint32_t vq = 0, vpar = 0;      // f16 V ring, likewise
    uint32_t ppar = 0;              // bit t: phase of slot t's next P tile
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    bool ok = true;
    for (uint32_t seg = 0; ok && !walk.done(sh); walk.next(p, sh), ++seg) {
      const KtcSeg sg(p, sh, walk);
      const bool two = __shfl_sync(0xffffffffu, sg.two, 0);
      const int tiles = __shfl_sync(0xffffffffu, sg.n, 0);
      const int steps = two ? 2 * tiles : tiles;
      auto wait = [&](uint32_t b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag)) != 0; };
      ok = wait(q_full, seg & 1);
      // Step s: PV of its tile, then the scores of step s + 2 (slot `t` = s & 1).
      auto step = [&](auto slot, int s) {
        constexpr uint32_t t = decltype(slot)::value;
        const bool last = t == 1 || !two;     // of the key tile
        const bool first = t == 0 || !two;
        // What is there long before P is waited for first.
        if (s + 2 < steps && first) ok = wait(k_full + 8 * kq, kpar);
        if (s >= 0) {
          if (s == 0 && seg > 0) ok = ok && wait(o_free, (seg - 1) & 1);   // the last segment's output has left TMEM
          if (first) ok = ok && wait(v16_full + 8 * vq, vpar);
          ok = ok && wait(p_full + 8 * t, (ppar >> t) & 1);
          if (!ok) return;
          ppar ^= 1u << t;
          tc_fence_after();
          if (issuer) {
            ktc_issue_pv(tm + 256 + t * 128, tm + t * 128, sV16 + vq * (2 * KTC_TILE8), s >= 2);
            if (last) umma_commit(v16_empty + 8 * vq);
          }
          if (last && ++vq == 2) { vq = 0; vpar ^= 1; }
        }
        if (s + 2 < steps) {
          if (!ok) return;
          tc_fence_after();
          if (issuer) {
            ktc_issue_s(tm + t * 128, two ? sQ + t * (2 * KTC_TILE8) : sQ, sK + kq * KTC_TILE8);
            umma_commit(s_full + 8 * t);
            if (last) umma_commit(k_empty + 8 * kq);
          }
          if (last && ++kq == 2) { kq = 0; kpar ^= 1; }
        }
      };
      for (int s = -2; ok && s < steps; s += 2) {
        step(std::integral_constant<uint32_t, 0>{}, s);
        if (issuer && s + 3 == steps) umma_commit(q_free);   // the last scores are made
        if (ok && s + 1 < steps) step(std::integral_constant<uint32_t, 1>{}, s + 1);
        if (issuer && s + 4 == steps) umma_commit(q_free);
      }
      if (issuer) umma_commit(o_done);
    }
    if (issuer) {
      umma_commit(drain);
      mbar_wait_teardown(drain, 0);
    }
    __syncwarp();
  } else {
    // --------------------------------------------- V codes -> f16 tiles
    // Warp 10 takes dims [0, 64), warp 11 [64, 128), 16 codes a lane and
    // piece. Eight lanes take rows r and r ^ 5, four pieces each: loads and
    // both stores of a piece then meet every bank once.
    const int sub = lane >> 3, row8 = (lane & 4) ? sub ^ 5 : sub, c4 = lane & 3, half = warp - 10;
    int tiles = 0;
    bool ok = true;
    for (; ok && !walk.done(sh); walk.next(p, sh)) {
      const KtcSeg sg(p, sh, walk);
      for (int j = 0; ok && j < sg.n; ++j, ++tiles) {
        const int slot = tiles & 1, live = sg.live(j);
        const uint32_t phase = (tiles >> 1) & 1;
        ok = mbar_wait(v8_full + 8 * slot, phase, abort_flag) && mbar_wait(v16_empty + 8 * slot, phase ^ 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t src = sV8 + slot * KTC_TILE8, dst = sV16 + slot * 2 * KTC_TILE8 + half * KTC_TILE8;
#pragma unroll 4
        for (int i = 0; i < 16; ++i) {
          const int r = 8 * i + row8;
          uint4 w = lds128(src + r * 128 + (((4 * half + c4) ^ row8) << 4));
          if (r >= live) w = make_uint4(0, 0, 0, 0);   // whatever lies there (NaN codes too) counts for nothing
          const uint32_t at = dst + r * 128;
          sts128(at + (((2 * c4) ^ row8) << 4), make_uint4(e4m3x2_to_f16x2(w.x), e4m3x2_hi_to_f16x2(w.x),
                                                           e4m3x2_to_f16x2(w.y), e4m3x2_hi_to_f16x2(w.y)));
          sts128(at + (((2 * c4 + 1) ^ row8) << 4), make_uint4(e4m3x2_to_f16x2(w.z), e4m3x2_hi_to_f16x2(w.z),
                                                               e4m3x2_to_f16x2(w.w), e4m3x2_hi_to_f16x2(w.w)));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(v16_full + 8 * slot);
          mbar_arrive(v8_empty + 8 * slot);
        }
      }
    }
  }
  } else {
    // ------------------------------------------------ softmax / epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2;          // TMEM slot
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lane_base + t * 128, tO = tmem + lane_base + 256 + t * 128;
    int tile0 = 0, scount = 0;
    bool ok = true;
    for (int seg = 0; !walk.done(sh); walk.next(p, sh), ++seg) {
      const KtcSeg sg(p, sh, walk);
      const int h = walk.it.h;
      const int rr = sg.qt * KTC_QR + (sg.two ? t * 128 : 0) + r;     // row of the (sequence, head)
      const bool valid = rr < sg.qt * KTC_QR + sg.rows;
      const int tok = rr / p.group;
      const float rf = valid ? __ldg(q_factor + (static_cast<long long>(sg.b) * p.c.heads + h) * rows_pad + rr) : 0.f;
      const int len = kv8_len(p.s, p.c, sg.b);
      const int seen = p.causal ? max(0, min(len, len - kv8_count(p.s, sg.b) + tok + 1)) : len;
      float m = -INFINITY, l = 0.f;
      const int mine = sg.two ? sg.n : (sg.n + 1 - t) >> 1;   // key tiles of this slot
      for (int i = 0; ok && i < mine; ++i, ++scount) {
        const int j = sg.two ? i : 2 * i + t;
        const int sc = (tile0 + j) % KTC_SCS;
        // The tile's scales come to registers before its scores are there:
        // shared memory answers slowly while the MMAs read their operands.
        ok = mbar_wait(sc_full + 8 * sc, ((tile0 + j) / KTC_SCS) & 1, abort_flag);
        const float4* scale = reinterpret_cast<const float4*>(smem + L::SC_OFF) + sc * 8;
        float fs[8], lv[8];
        {
          const float4 a = scale[0], b = scale[1], c = scale[2], d = scale[3];
          const float ks[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
          for (int g8 = 0; g8 < 8; ++g8) fs[g8] = fmaxf(rf * ks[g8], 1.17549435e-38f);   // > 0: hidden scores stay -inf
          lv[0] = c.x; lv[1] = c.y; lv[2] = c.z; lv[3] = c.w;
          lv[4] = d.x; lv[5] = d.y; lv[6] = d.z; lv[7] = d.w;
        }
        ok = ok && mbar_wait(s_full + 8 * t, scount & 1, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        const int lim = seen - (sg.j0 + j) * KTC_TK;    // keys of this tile that the row sees
        const bool part = __any_sync(0xffffffffu, lim < KTC_TK);
        if (part) {
          // Hidden scores become -inf where they lie, in a rolled loop: 128
          // selects inside the common path cost it 4% (its code no longer
          // stays in the instruction cache).
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float x[32];
            tmem_ld32(tS + c * 32, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c * 32 + k >= lim) x[k] = -INFINITY;
            tmem_st32(tS + c * 32, x);
          }
          tmem_wait_st();
        }
        float s[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float x[32];
          tmem_ld32(tS + c * 32, x);
#pragma unroll
          for (int k = 0; k < 32; ++k) s[c * 32 + k] = x[k];
        }
        tmem_wait_ld();
        // Maximum of y over the 8 groups of 16 keys; NaN wins (it makes the row NaN).
        float mx = -INFINITY;
#pragma unroll
        for (int g8 = 0; g8 < 8; ++g8) {
          const float* sg8 = s + 16 * g8;
          float a = max3_nan(sg8[0], sg8[1], sg8[2]), b = max3_nan(sg8[3], sg8[4], sg8[5]);
          a = max3_nan(a, sg8[6], sg8[7]);
          b = max3_nan(b, sg8[8], sg8[9]);
          a = max3_nan(a, sg8[10], sg8[11]);
          b = max3_nan(b, sg8[12], sg8[13]);
          a = max3_nan(a, sg8[14], sg8[15]);
          a = max3_nan(a, b, b);
          a = fmaf(a, fs[g8], lv[g8]);
          mx = max3_nan(mx, a, a);
        }
        const bool grow = !(mx <= m + FEW_RESCALE);
        const float m_new = grow ? mx : m;
        const float z = (m_new == -INFINITY ? 0.f : m_new) - FEW_OFFSET;
        const float alpha = grow ? (m == -INFINITY ? 0.f : exp2f(m - m_new)) : 1.f;
        float sums[8];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int gq = 0; gq < 2; ++gq) {
            const float cs = lv[2 * c + gq] - z;
            const uint64_t f2s = f2(fs[2 * c + gq], fs[2 * c + gq]), c2s = f2(cs, cs);
            uint64_t sum2 = f2(0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint64_t x2 = ffma2(f2(s[32 * c + 16 * gq + 2 * k], s[32 * c + 16 * gq + 2 * k + 1]), f2s, c2s);
              const float2 x = f2_split(x2);
              const float a = ex2_mufu(x.x), b = ex2_mufu(x.y);
              sum2 = fadd2(sum2, f2(a, b));
              pk[8 * gq + k] = pack_f16(a, b);
            }
            const float2 sv = f2_split(sum2);
            sums[2 * c + gq] = sv.x + sv.y;
          }
          tmem_st16u(tS + c * 16, pk);
        }
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
          // O is stable: this S was issued behind the slot's last PV and is complete.
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float o[32];
            tmem_ld32(tO + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= alpha;
            tmem_st32(tO + c * 32, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 8 * t);
        {
          const float4 a = scale[4], b = scale[5];
          float sum = sums[0] * a.x;
          sum = fmaf(sums[1], a.y, sum);
          sum = fmaf(sums[2], a.z, sum);
          sum = fmaf(sums[3], a.w, sum);
          sum = fmaf(sums[4], b.x, sum);
          sum = fmaf(sums[5], b.y, sum);
          sum = fmaf(sums[6], b.z, sum);
          sum = fmaf(sums[7], b.w, sum);
          l = fmaf(l, alpha, sum);
        }
        m = m_new;
      }
      tile0 += sg.n;
      if (ok) ok = mbar_wait(o_done, seg & 1, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
      if (!ok) l = 0.f;
      const bool whole = sg.begins && sg.ends;
      float* part = p.part + static_cast<size_t>(2 * blockIdx.x + (sg.begins ? 1 : 0)) * kv8_part_floats<KTC_QR>();
      const int prow = (sg.two ? t * 128 : 0) + r;
      const int hq = h * p.group + rr - tok * p.group;
      float wA = 1.f, wB = 0.f, den = l, M = m;
      if (!sg.two) {
        // Both slots hold the same rows: slot t finishes columns [64 t, +64).
        float* xm = reinterpret_cast<float*>(smem + L::STAGE_OFF);
        xm[t * 256 + r] = m;
        xm[t * 256 + 128 + r] = l;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float m0 = xm[r], l0 = xm[128 + r], m1 = xm[256 + r], l1 = xm[384 + r];
        M = fmaxf(m0, m1);
        wA = m0 == -INFINITY ? 0.f : exp2f(m0 - M);
        wB = m1 == -INFINITY ? 0.f : exp2f(m1 - M);
        den = wA * l0 + wB * l1;
        asm volatile("bar.sync 1, 256;" ::: "memory");
      }
      const float mref = M == -INFINITY ? M : M - FEW_OFFSET;
      const float inv = den == 0.f ? 0.f : 1.f / den;
      const int chunks = sg.two ? 4 : 2;
      const uint32_t src = sg.two ? tO : tmem + lane_base + 256 + t * 64;
      const int col0 = sg.two ? 0 : t * 64;
      // 32 columns at a time go through 4 KB of the warp's own, so that global
      // memory sees whole 128-byte (bf16: 64-byte) pieces of rows. (A thread
      // storing its own row took ~9400 cycles a segment.)
      const uint32_t stage = base + L::STAGE_OFF + warp * 4096;
      const int row0 = sg.qt * KTC_QR + prow - lane;        // first row of the warp
#pragma unroll 1
      for (int c = 0; ok && c < chunks; ++c) {
        float o[32];
        tmem_ld32(src + c * 32, o);
        tmem_wait_ld();
        if (!sg.two) {
          const bool has_b = sg.n > 1;      // slot B met a key tile
          float o1[32];
          if (has_b) {
            tmem_ld32(src + 128 + c * 32, o1);
            tmem_wait_ld();
          }
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = has_b ? o[k] * wA + o1[k] * wB : o[k] * wA;
        }
        __syncwarp();     // the last columns have been read
        const int sub = lane >> 3, c8 = lane & 7;
        if (whole) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            sts128(stage + lane * 128 + ((k ^ (lane & 7)) << 4),
                   make_uint4(pack_bf16(o[8 * k] * inv, o[8 * k + 1] * inv), pack_bf16(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                              pack_bf16(o[8 * k + 4] * inv, o[8 * k + 5] * inv), pack_bf16(o[8 * k + 6] * inv, o[8 * k + 7] * inv)));
          __syncwarp();
          // Four lanes to a row, eight rows at a time.
          for (int i = 0; i < 4; ++i) {
            const int rl = 8 * i + (lane >> 2), row = row0 + rl, k = lane & 3;
            if (row >= sg.qt * KTC_QR + sg.rows) continue;
            const int tk = row / p.group;
            __nv_bfloat16* to = p.out + sg.b * p.o_sb + tk * p.o_st + (h * p.group + row - tk * p.group) * p.o_sh;
            *reinterpret_cast<uint4*>(to + col0 + c * 32 + k * 8) = lds128(stage + rl * 128 + ((k ^ (rl & 7)) << 4));
          }
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            sts128(stage + lane * 128 + ((k ^ (lane & 7)) << 4),
                   make_uint4(__float_as_uint(o[4 * k]), __float_as_uint(o[4 * k + 1]), __float_as_uint(o[4 * k + 2]),
                              __float_as_uint(o[4 * k + 3])));
          __syncwarp();
          for (int i = 0; i < 8; ++i) {
            const int rl = 4 * i + sub, pr = prow - lane + rl;
            if (pr < sg.rows)
              *reinterpret_cast<uint4*>(part + pr * 128 + col0 + c * 32 + c8 * 4) = lds128(stage + rl * 128 + ((c8 ^ (rl & 7)) << 4));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free);
      if (valid && (sg.two || t == 0)) {
        if (!whole) {
          part[KTC_QR * 128 + prow] = mref;
          part[KTC_QR * 129 + prow] = den;
        } else if (p.lse != nullptr) {
          p.lse[(static_cast<long long>(sg.b) * p.s.tokens + tok) * (p.c.heads * p.group) + hq] = kv8_row_lse(mref, den);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ----------------------------------------------------------------- weights
// Attention weights for more than a few query rows: S^T = K Q^T with the keys
// in the lanes (M 128 keys, N 128 query rows), so that a thread owns a key
// and adds up its column of exp(s - lse) with no exchange between threads; the
// rows' factors and log-sum-exps come from shared memory, the same address for
// a whole warp. Units are key tiles (all query rows of the sequence), cut
// evenly over the CTAs; a unit's sums are complete, so there are no partials.
// Two neighbouring key tiles of a head go together: warps 0-3 take the first,
// warps 4-7 the second, each with two score buffers in TMEM, and every query
// tile that is loaded serves both.
// Bound by the exponentials: 128 x 128 of them take the SM's MUFU 1024
// cycles, the products of the two query pieces 512.
// 880 rows over 4400 keys of 24 heads (23.8 GFLOP): 50 us, 7 of them the split
// of the queries; 8 such sequences of up to 4400 keys 271 us, 0.55 PFLOP/s. 17
// rows over 16 k keys of 8 x 8 heads: 47 us (63 with the columns behind the rows).
// 320 threads: warps 0..7 exponentials, warp 8 loads, warp 9 issues the MMAs.
constexpr int KWT_THREADS = 320, KWT_QS = 4, KWT_FS = 8, KWT_SCS = 16, KWT_QR = 1 << 30;
constexpr int KWT_POLY = 2;      // pairs of every eight whose 2^x runs on the FMA pipe: 0, 1, 2, 3, 4 took 58, 52, 50, 50, 52 us (below)

struct KwtSmem {
  static constexpr uint32_t K_OFF = 0;                                     // [2 pairs] 2 tiles of codes
  static constexpr uint32_t Q_OFF = K_OFF + 4 * KTC_TILE8;                 // [4] hi, lo
  static constexpr uint32_t F_OFF = Q_OFF + KWT_QS * 2 * KTC_TILE8;        // [8] factors, -lse2 of 128 rows
  static constexpr uint32_t SC_OFF = F_OFF + KWT_FS * 1024;                // [16 pairs] ks of 16 groups of 16 keys
  static constexpr uint32_t BAR_OFF = SC_OFF + KWT_SCS * 64;
  static constexpr uint32_t NBARS = 4 + 2 * KWT_QS + 2 * KWT_FS + 8 + 1;
  static constexpr uint32_t SCHED_OFF = BAR_OFF + NBARS * 8;
  static constexpr uint32_t TOTAL = 1024 + SCHED_OFF + sizeof(Kv8SchedSmem) + 16;
  static_assert(TOTAL <= 232448, "shared memory exceeds 227 KB");
};

// One or two neighbouring key tiles, and their query tiles [q0, q1).
struct KwtPair {
  int b, h, k0, len, cnt, rows, q0, q1, shift;   // row r sees key j when r >= group * (j - shift)
  WAMB_DEV KwtPair(const Kv8AttnParams& p, const Kv8Share& sh, const KtcWalk<KWT_QR>& w) {
    b = w.it.e;
    h = w.it.h;
    k0 = static_cast<int>(w.u - w.it.start) * KTC_TK;
    cnt = static_cast<int>(min(2ll, min(sh.u1, w.it.start + w.it.n) - w.u));
    len = kv8_len(p.s, p.c, b);
    const int tokens = kv8_count(p.s, b);
    shift = len - tokens;
    rows = tokens * p.group;
    q1 = (rows + 127) / 128;
    q0 = p.causal && k0 > shift ? static_cast<int>(min(q1 - 1ll, static_cast<long long>(k0 - shift) * p.group / 128)) : 0;
  }
  WAMB_DEV void next(const Kv8AttnParams& p, const Kv8Share& sh, KtcWalk<KWT_QR>& w) const {
    w.u += cnt;
    if (w.u < sh.u1) kv8_seek<KWT_QR, KTC_TK>(p, w.it, w.u);
  }
};

__global__ void __launch_bounds__(KWT_THREADS, 1)
    kv8_weights_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ,
                          const float* q_factor, const float* q_neg_lse2, const int rows_pad, const Kv8AttnParams p) {
  using L = KwtSmem;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t base = smem_u32(smem);
  const uint32_t sK = base + L::K_OFF, sQ = base + L::Q_OFF, sF = base + L::F_OFF;
  uint32_t bar = base + L::BAR_OFF;
  auto bars = [&](int n) { const uint32_t b = bar; bar += 8 * n; return b; };
  const uint32_t k_full = bars(2), k_empty = bars(2), q_full = bars(KWT_QS), q_empty = bars(KWT_QS),
                 f_full = bars(KWT_FS), f_free = bars(KWT_FS), s_full = bars(4), s_free = bars(4), drain = bars(1);
  Kv8SchedSmem& sched = *reinterpret_cast<Kv8SchedSmem*>(smem + L::SCHED_OFF);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::SCHED_OFF + sizeof(Kv8SchedSmem));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // warp: uniform

  // As in kv8_tc_kernel, only the split of the queries is waited for.
  kv8_carry_base<KWT_THREADS>(p);
  Kv8Share sh;
  KtcWalk<KWT_QR> walk;
  if (!kv8_share<KWT_QR, KTC_TK, KWT_THREADS>(p, blockIdx.x, sched, sh, walk.it)) {
    pdl_wait();
    return;
  }
  walk.u = sh.u0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) { mbar_init(k_full + 8 * i, 1); mbar_init(k_empty + 8 * i, 1); }
    for (int i = 0; i < KWT_QS; ++i) { mbar_init(q_full + 8 * i, 1); mbar_init(q_empty + 8 * i, 1); }
    for (int i = 0; i < KWT_FS; ++i) { mbar_init(f_full + 8 * i, 1); mbar_init(f_free + 8 * i, 8); }
    for (int i = 0; i < 4; ++i) { mbar_init(s_full + 8 * i, 1); mbar_init(s_free + 8 * i, 4); }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  auto wait = [&](uint32_t b, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(b, parity, abort_flag)) != 0; };

  if (warp == 8) {
    // ---------------------------------------------------------- producer
    // Lane i < 16 looks after keys [16 i, +16) of a pair, one pair ahead.
    const int box_groups = p.c.page >> 4;
    int pairs = 0, tiles = 0;
    bool go = true;
    struct Ahead { int row; float ks; };
    auto look = [&](const KwtPair& n) {
      Ahead a{-1, 1.f};
      const int key = n.k0 + lane * 16;
      if (lane < 8 * n.cnt && key < n.len) {
        const int pid = max(0, kv8_page(p.s.table, p.s.width, p.c, n.b, key >> p.c.page_log2));   // a bad id is reported
        const long long blk = static_cast<long long>(pid) * p.c.heads + n.h;
        a.row = static_cast<int>((blk << p.c.page_log2) + (key & (p.c.page - 1)));
        a.ks = __ldg(p.c.k_scale + blk);
      }
      return a;
    };
    Ahead now = look(KwtPair(p, sh, walk));
    while (go && !walk.done(sh)) {
      const KwtPair n(p, sh, walk);
      n.next(p, sh, walk);
      Ahead next{-1, 1.f};
      if (!walk.done(sh)) next = look(KwtPair(p, sh, walk));
      const int ks = pairs & 1;
      go = wait(k_empty + 8 * ks, ((pairs >> 1) & 1) ^ 1);
      if (!go) break;
      // The pair's scales are published with the factors of its first query
      // tile; sixteen pairs on, the factor ring has long seen them read.
      if (lane < 16) reinterpret_cast<float*>(smem + L::SC_OFF)[(pairs % KWT_SCS) * 16 + lane] = now.ks;
      const bool lead = now.row >= 0 && lane % box_groups == 0;
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, lead)) * (p.c.page * 128);
      __syncwarp();
      if (lane == 0) mbar_arrive_expect_tx(k_full + 8 * ks, bytes);
      __syncwarp();
      if (lead) tma_load_2d(sK + ks * 2 * KTC_TILE8 + lane * 2048, &tmK, k_full + 8 * ks, 0, now.row);
      ++pairs;
      for (int qt = n.q0; qt < n.q1; ++qt, ++tiles) {
        const int qs = tiles % KWT_QS, fs = tiles % KWT_FS;
        go = wait(q_empty + 8 * qs, ((tiles / KWT_QS) & 1) ^ 1) && wait(f_free + 8 * fs, ((tiles / KWT_FS) & 1) ^ 1);
        if (!go) break;
        if (lane == 0) {
          const int row = (n.b * p.c.heads + n.h) * rows_pad + qt * 128;
          const uint32_t at = sQ + qs * 2 * KTC_TILE8, f = sF + fs * 1024;
          mbar_arrive_expect_tx(q_full + 8 * qs, 2 * KTC_TILE8);
          tma_load_2d(at, &tmQ, q_full + 8 * qs, 0, row);
          tma_load_2d(at + KTC_TILE8, &tmQ, q_full + 8 * qs, 128, row);
          mbar_arrive_expect_tx(f_full + 8 * fs, 1024);
          bulk_load(f, q_factor + row, 512, f_full + 8 * fs);
          bulk_load(f + 512, q_neg_lse2 + row, 512, f_full + 8 * fs);
        }
        __syncwarp();
      }
      now = next;
    }
    // Loads still in flight must land before the CTA exits, after a wait that ran out too.
    if (lane == 0) {
      for (int t = max(0, pairs - 2); t < pairs; ++t) mbar_wait_teardown(k_full + 8 * (t & 1), (t >> 1) & 1);
      for (int t = max(0, tiles - KWT_QS); t < tiles; ++t) {
        mbar_wait_teardown(q_full + 8 * (t % KWT_QS), (t / KWT_QS) & 1);
        mbar_wait_teardown(f_full + 8 * (t % KWT_FS), (t / KWT_FS) & 1);
      }
    }
    __syncwarp();
  } else if (warp == 9) {
    // --------------------------------------------------------- MMA issuer
    const bool issuer = elect_one();
    uint32_t pairs = 0, tiles = 0, made[2] = {0, 0};   // score tiles made for each group
    bool ok = true;
    while (ok && !walk.done(sh)) {
      const KwtPair n(p, sh, walk);
      const int nq = __shfl_sync(0xffffffffu, n.q1 - n.q0, 0);
      const bool both = __shfl_sync(0xffffffffu, n.cnt, 0) == 2;
      const uint32_t kt = sK + (pairs & 1) * 2 * KTC_TILE8;
      ok = wait(k_full + 8 * (pairs & 1), (pairs >> 1) & 1);
      for (int i = 0; ok && i < nq; ++i, ++tiles) {
        const uint32_t qs = tiles % KWT_QS;
        ok = wait(q_full + 8 * qs, (tiles / KWT_QS) & 1);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if (g == 1 && !both) break;
          const uint32_t sb = 2 * g + (made[g] & 1);
          ok = ok && wait(s_free + 8 * sb, ((made[g] >> 1) & 1) ^ 1);
          if (!ok) break;
          ++made[g];
          tc_fence_after();
          if (issuer) {
            // Keys are the rows here, the two query pieces the columns.
            ktc_issue_st(tmem + sb * 128, kt + g * KTC_TILE8, sQ + qs * 2 * KTC_TILE8);
            umma_commit(s_full + 8 * sb);
          }
          __syncwarp();
        }
        if (!ok) break;
        if (issuer) {
          umma_commit(q_empty + 8 * qs);
          if (i == nq - 1) umma_commit(k_empty + 8 * (pairs & 1));
        }
        __syncwarp();
      }
      n.next(p, sh, walk);
      ++pairs;
    }
    if (issuer) {
      umma_commit(drain);
      mbar_wait_teardown(drain, 0);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------- exponentials
    const int grp = warp >> 2;
    const int r = (warp & 3) * 32 + lane;     // key within the tile == TMEM lane
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + grp * 256;
    int pairs = 0, tiles = 0;
    uint32_t taken = 0;     // score tiles of this group
    bool ok = true;         // once false, the loop goes on without waiting
    for (; !walk.done(sh); ++pairs) {
      const KwtPair n(p, sh, walk);
      const bool active = grp < n.cnt;
      const int key = n.k0 + grp * KTC_TK + r;
      const bool store = active && key < n.len;
      const long long at = (static_cast<long long>(n.b) * p.c.heads + n.h) * p.w_cap + key;
      const float from = store && p.base != nullptr ? __ldcg(p.base + at) : 0.f;
      const long long first = p.causal ? static_cast<long long>(key - n.shift) * p.group : 0;   // first row that sees the key
      uint64_t ks2 = 0, acc[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
      for (int qt = n.q0; qt < n.q1; ++qt, ++tiles) {
        const int fs = tiles % KWT_FS;
        ok = ok && wait(f_full + 8 * fs, (tiles / KWT_FS) & 1);
        if (active) {
          if (qt == n.q0) {
            const float ks = reinterpret_cast<const float*>(smem + L::SC_OFF)[(pairs % KWT_SCS) * 16 + grp * 8 + (r >> 4)];
            ks2 = f2(ks, ks);
          }
          const uint32_t sb = 2 * grp + (taken & 1), ts = tS + (taken & 1) * 128;
          ok = ok && wait(s_full + 8 * sb, (taken >> 1) & 1);
          ++taken;
          tc_fence_after();
          const float4* f = reinterpret_cast<const float4*>(smem + L::F_OFF + fs * 1024);
          const int lim = static_cast<int>(max(0ll, min(128ll, first - qt * 128ll)));   // rows below it do not see the key
          if (__any_sync(0xffffffffu, lim > 0)) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              float x[32];
              tmem_ld32(ts + c * 32, x);
              tmem_wait_ld();
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (c * 32 + k < lim) x[k] = -INFINITY;
              tmem_st32(ts + c * 32, x);
            }
            tmem_wait_st();
          }
          float sA[32], sB[32];
          auto add = [&](const float (&s)[32], int c) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 rf = f[c * 8 + k], nl = f[32 + c * 8 + k];
#pragma unroll
              for (int u = 0; u < 2; ++u) {
                const uint64_t a = fmul2(f2(s[4 * k + 2 * u], s[4 * k + 2 * u + 1]), ks2);
                const uint64_t x2 = ffma2(a, u ? f2(rf.z, rf.w) : f2(rf.x, rf.y), u ? f2(nl.z, nl.w) : f2(nl.x, nl.y));
                if (2 * (k & 3) + u >= 8 - KWT_POLY) {
                  acc[u] = fadd2(acc[u], ex2_poly5(x2));
                } else {
                  const float2 x = f2_split(x2);
                  acc[u] = fadd2(acc[u], f2(ex2_mufu(x.x), ex2_mufu(x.y)));
                }
              }
            }
          };
          tmem_ld32(ts, sA);
          tmem_wait_ld();
          tmem_ld32(ts + 32, sB);
          // 32 columns that lie behind the rows have nothing to add.
          const int live = n.rows - qt * 128;
          add(sA, 0);
          tmem_wait_ld();
          tmem_ld32(ts + 64, sA);
          if (live > 32) add(sB, 1);
          tmem_wait_ld();
          tmem_ld32(ts + 96, sB);
          if (live > 64) add(sA, 2);
          tmem_wait_ld();
          tc_fence_before();   // the scores are in registers: the buffer is free
          __syncwarp();
          if (lane == 0) mbar_arrive(s_free + 8 * sb);
          if (live > 96) add(sB, 3);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(f_free + 8 * fs);
      }
      const float2 a0 = f2_split(acc[0]), a1 = f2_split(acc[1]);
      const float sum = (a0.x + a0.y) + (a1.x + a1.y);
      // The polynomial gives 2^-125 for a row that does not see the key.
      if (store) p.weights[at] = ok ? from + (sum < 7.9e-31f ? 0.f : sum) : 0.f;
      n.next(p, sh, walk);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace wamb
