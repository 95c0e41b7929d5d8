// Attention and attention weights over the E4M3 cache (kv8.cuh) for few query
// rows: the single-token form and small groups, where the cache's bytes bound
// the call.
//
//   s_ij = scale q_i . (code_j ks_j),  o_i = sum_j softmax_j(s_ij) code'_j vs_j
//   lse_i = ln sum_j exp(s_ij),        w_j = sum_i exp(s_ij - lse_i)
//
// The `group` query heads of one cached head are rows of one tile (row
// r = token * group + head in group), so each cached byte is read once for
// all of them. A warp takes 32 keys at a time, K and V codes (4 KB each) by
// TMA into its own ring, with no barrier between warps until an item ends.
// The codes become f16 in registers (E4M3 is a subset of f16, nothing is
// rounded) and meet the queries in m16n8k16 products with fp32 sums. (The
// E4M3 m16n8k32 form is no shortcut here: with it a step took about twice the
// instructions.) Queries go to f16 scaled per row by a power
// of two that puts the largest magnitude into [2^13, 2^14), which keeps their
// eight bits over 28 binades.
//
// The scales of a block enter the exponent: with y_ij = s_ij log2(e) +
// log2(vs_j) the kernel sums P_ij = 2^(y_ij - M_i) against the codes, M_i a
// running maximum of y (moved only when it grows by more than 2^8), and
// l_i = sum_j P_ij / vs_j. P goes to the product as f16 with an offset of 2^6:
// 11 bits down to 2^-20 of the row's maximum and whole steps of 2^-30 below.
//
// Bound by the latency of a warp's step (load -> convert -> product -> exponential ->
// product, one unit at a time) with twelve to sixteen warps an SM: one token of 8
// sequences of 18 to 32 thousand keys (8 heads, 4 query heads each, 420 MB)
// takes 82 us, 5.1 TB/s, with 35 M warp instructions, half of them the
// conversions of codes and the products, and issue active 44% of the cycles;
// its attention weights (K alone, 227 MB) take 49 us, 4.7 TB/s, at 53%. The smallest calls
// (2 sequences of 500 keys, 12 heads) take 11 us, nearly all of it the latency of two
// launches and of table -> scale -> codes.
#pragma once
#include "attention.cuh"
#include "kv8.cuh"

namespace wamb {

struct Kv8AttnParams {
  Kv8Cache c;
  Kv8Seqs s;
  const __nv_bfloat16* q;
  long long q_sb, q_st, q_sh;      // element strides of (batch, token, head)
  int group, causal;
  float scale_log2;                // softmax scale * log2(e)
  __nv_bfloat16* out;
  long long o_sb, o_st, o_sh;
  float* lse;                      // [batch, tokens, heads * group] or null
  // attention weights
  const float* lse_in;             // like lse
  const float* base;               // [batch, heads, w_cap] or null (zeros)
  float* weights;                  // like base; may be base
  long long w_cap;
  // stream-K: query tiles per sequence, CTAs, partials
  int qts, ctas;
  float* part;
};

// --------------------------------------------------------------- schedule
// The work of a call is a line of units. Entry e = b * qts + qt (a query tile
// of QR rows of sequence b) has n(e) units of TK keys for each cached head;
// entries follow one another, heads within an entry, key tiles within a
// head: an item is one (entry, head). The line is cut into equal shares, one
// per CTA, whatever the lengths, which only the device knows. A CTA finishes
// items that lie in its share and leaves partials (max, sum, O) for the one
// it joins in the middle (slot 0) and the one it leaves unfinished (slot 1).
template <int QR, int TK>
struct Kv8Line {
  WAMB_DEV static int rows(const Kv8AttnParams& p, int b) { return kv8_count(p.s, b) * p.group; }
  // Keys that the last row of the tile sees (every row of it sees no more).
  WAMB_DEV static int visible(const Kv8AttnParams& p, int e) {
    const int b = e / p.qts, qt = e - b * p.qts;
    const int len = kv8_len(p.s, p.c, b);
    if (!p.causal) return len;
    const int t = kv8_count(p.s, b);
    const int last = (min(t * p.group, (qt + 1) * QR) - 1) / p.group;
    return max(0, min(len, len - t + last + 1));
  }
  // Units per head; a tile with rows has one at least (it must be answered).
  WAMB_DEV static int units(const Kv8AttnParams& p, int e) {
    const int b = e / p.qts, qt = e - b * p.qts;
    if (qt * QR >= rows(p, b)) return 0;
    return max(1, (visible(p, e) + TK - 1) / TK);
  }
};

struct Kv8Item {
  int e, h, n;         // entry, head, units
  long long start;     // first unit on the line
};

// Moves `it` forward to the item that holds unit u.
template <int QR, int TK>
WAMB_DEV void kv8_seek(const Kv8AttnParams& p, Kv8Item& it, long long u) {
  long long left = it.start + static_cast<long long>(it.n) * (p.c.heads - it.h);   // end of the entry
  while (u >= left) {
    it.start = left;
    it.h = 0;
    do { ++it.e; it.n = Kv8Line<QR, TK>::units(p, it.e); } while (it.n == 0);
    left = it.start + static_cast<long long>(it.n) * p.c.heads;
  }
  const int skip = static_cast<int>((u - it.start) / it.n);
  it.h += skip;
  it.start += static_cast<long long>(skip) * it.n;
}

struct Kv8SchedSmem {
  long long warp[32];
  long long start;
  int e;
};
struct Kv8Share {
  long long units;     // of the whole line
  int ctas;            // shares
  long long u0, u1;
  WAMB_DEV long long first(int cta) const { return cta * units / ctas; }
};

// The share of `cta` and the item of its first unit; false without work.
// Called by the whole block.
template <int QR, int TK, int THREADS>
WAMB_DEV bool kv8_share(const Kv8AttnParams& p, int cta, Kv8SchedSmem& sm, Kv8Share& sh, Kv8Item& it) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int entries = p.s.batch * p.qts;
  long long sum = 0;
  for (int e = tid; e < entries; e += THREADS) sum += Kv8Line<QR, TK>::units(p, e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sm.warp[warp] = sum;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) total += sm.warp[i];
  sh.units = total * p.c.heads;
  sh.ctas = static_cast<int>(min(static_cast<long long>(p.ctas), max(1ll, sh.units)));   // a unit each at least
  if (sh.units == 0 || cta >= sh.ctas) return false;
  sh.u0 = sh.first(cta);
  sh.u1 = sh.first(cta + 1);
  __syncthreads();
  // The entry of u0: scan the entries' units a block at a time.
  long long run = 0;
  for (int e0 = 0;; e0 += THREADS) {
    const int e = e0 + tid;
    const long long mine = e < entries ? static_cast<long long>(Kv8Line<QR, TK>::units(p, e)) * p.c.heads : 0;
    long long inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sm.warp[warp] = inc;
    __syncthreads();
    long long before = run;
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += sm.warp[i];
      run += sm.warp[i];
    }
    const long long end = before + inc;
    if (end - mine <= sh.u0 && sh.u0 < end) {
      sm.e = e;
      sm.start = end - mine;
    }
    __syncthreads();
    if (sh.u0 < run) break;
  }
  it.e = sm.e;
  it.h = 0;
  it.start = sm.start;
  it.n = Kv8Line<QR, TK>::units(p, it.e);
  kv8_seek<QR, TK>(p, it, sh.u0);
  return true;
}

// Weights past a sequence's keys carry the base over. Pieces of 2048 columns
// go round the CTAs; a thread's 16 loads are in flight together.
template <int THREADS>
WAMB_DEV void kv8_carry_base(const Kv8AttnParams& p) {
  if (p.weights == p.base) return;
  constexpr int PIECE = 2048, EACH = (PIECE + THREADS - 1) / THREADS;
  const long long pieces = (p.w_cap + PIECE - 1) / PIECE, all = pieces * p.s.batch * p.c.heads;
  for (long long i = blockIdx.x; i < all; i += gridDim.x) {
    const long long row = i / pieces;
    const int b = static_cast<int>(row / p.c.heads);
    const int seen = kv8_count(p.s, b) > 0 ? kv8_len(p.s, p.c, b) : 0;
    const long long j0 = (i - row * pieces) * PIECE, j1 = min(p.w_cap, j0 + PIECE);
    if (j1 <= seen) continue;
    float v[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const long long j = j0 + u * THREADS + threadIdx.x;
      v[u] = p.base != nullptr && j >= seen && j < j1 ? __ldcg(p.base + row * p.w_cap + j) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
      const long long j = j0 + u * THREADS + threadIdx.x;
      if (j >= seen && j < j1) p.weights[row * p.w_cap + j] = v[u];
    }
  }
}

// Floats of a partial: O [QR][128] relative to the row's M, then M, l.
template <int QR>
__host__ __device__ constexpr size_t kv8_part_floats() { return static_cast<size_t>(QR) * 130; }

// Final values of a row from its merged (M, l): out = O / l, lse.
WAMB_DEV float kv8_row_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f; }

// What CTA c leaves for the merge: the item that it finished but did not
// begin (first < 0: none), and the CTA that began it.
struct Kv8Join {
  int first, e, h, pad;
};
constexpr size_t KV8_JOIN_BYTES = 1024 * sizeof(Kv8Join);   // in front of the partials
WAMB_DEV Kv8Join* kv8_joins(const Kv8AttnParams& p) { return reinterpret_cast<Kv8Join*>(p.part) - 1024; }
// Called by one thread of every CTA, with the first item of its share.
WAMB_DEV void kv8_leave_join(const Kv8AttnParams& p, const Kv8Share& sh, bool work, const Kv8Item& it) {
  Kv8Join j{-1, 0, 0, 0};
  if (work && it.start < sh.u0 && it.start + it.n <= sh.u1) {
    j.first = static_cast<int>(((it.start + 1) * sh.ctas - 1) / sh.units);
    j.e = it.e;
    j.h = it.h;
  }
  kv8_joins(p)[blockIdx.x] = j;
}

// Joins the partials of items that several CTAs worked on, in CTA order:
// block (c, y) takes rows [y RB, +RB) of the item that CTA c finished. The
// eight warps share a row's partials (every eighth each, so that a hundred of
// them are read in a few round trips) and add their sums in warp order.
template <int QR, int RB>
__global__ void __launch_bounds__(256) kv8_merge_kernel(const Kv8AttnParams p) {
  __shared__ float4 sum[RB][8][32];
  __shared__ float den[RB][8], row_max[RB];
  pdl_wait();
  const int c = blockIdx.x;
  const Kv8Join j = kv8_joins(p)[c];
  if (j.first < 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = j.e / p.qts, qt = j.e - b * p.qts;
  const int rows = min(QR, kv8_count(p.s, b) * p.group - qt * QR);
  constexpr size_t PF = kv8_part_floats<QR>();
  const int cnt = c - j.first + 1;      // two at least
  auto slot = [&](int i) { return p.part + static_cast<size_t>(2 * (j.first + i) + (i == 0 ? 1 : 0)) * PF; };
  // Row `row` of the tile from its sums.
  auto finish = [&](int row, const float4& acc, float l, float m) {
    const int rr = qt * QR + row, t = rr / p.group, hq = j.h * p.group + rr - t * p.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    *reinterpret_cast<uint2*>(p.out + b * p.o_sb + t * p.o_st + hq * p.o_sh + lane * 4) =
        make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
    if (p.lse != nullptr && lane == 0)
      p.lse[(static_cast<long long>(b) * p.s.tokens + t) * (p.c.heads * p.group) + hq] = kv8_row_lse(m, l);
  };
  if constexpr (RB > 1) {
    // Two partials, as where there are more items than CTAs: four rows to a
    // warp, all their loads in flight, by a quarter of the blocks.
    if (cnt == 2) {
      constexpr int EACH = 4;
      const int r0 = (blockIdx.y * 8 + warp) * EACH;
      float4 v[EACH][2];
      float mk[EACH][2], lk[EACH][2];
#pragma unroll
      for (int q = 0; q < EACH; ++q)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          lk[q][i] = 0.f;
          if (r0 + q < rows) {
            v[q][i] = __ldcg(reinterpret_cast<const float4*>(slot(i) + (r0 + q) * 128) + lane);
            mk[q][i] = __ldcg(slot(i) + QR * 128 + r0 + q);
            lk[q][i] = __ldcg(slot(i) + QR * 129 + r0 + q);
          }
        }
#pragma unroll
      for (int q = 0; q < EACH; ++q) {
        if (r0 + q >= rows) continue;
        float m = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (lk[q][i] != 0.f) m = fmaxf(m, mk[q][i]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (lk[q][i] == 0.f) continue;   // no key seen there
          const float w = exp2f(mk[q][i] - m);
          l += w * lk[q][i];
          acc.x += w * v[q][i].x;
          acc.y += w * v[q][i].y;
          acc.z += w * v[q][i].z;
          acc.w += w * v[q][i].w;
        }
        finish(r0 + q, acc, l, m);
      }
      return;
    }
  }
  const int row0 = blockIdx.y * RB;
  if (row0 >= rows) return;
  // Few partials: a warp per row. Many: all warps on each row.
  const int step = cnt > 8 || RB == 1 ? 8 : 1, from = step == 8 ? warp : 0;
  for (int q = step == 8 ? 0 : warp; q < RB; q += step == 8 ? 1 : 8) {
    const int row = row0 + q;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    if (row < rows) {
      float m = -INFINITY;
      if (step == 8) {
        for (int i = lane; i < cnt; i += 32) m = fmaxf(m, __ldcg(slot(i) + QR * 128 + row));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      }
      for (int i0 = from; i0 < cnt; i0 += 8 * step) {
        float4 v[8];
        float mk[8], lk[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int i = i0 + u * step;
          lk[u] = 0.f;
          if (i < cnt) {
            v[u] = __ldcg(reinterpret_cast<const float4*>(slot(i) + row * 128) + lane);
            mk[u] = __ldcg(slot(i) + QR * 128 + row);
            lk[u] = __ldcg(slot(i) + QR * 129 + row);
          }
        }
        if (step == 1) {   // all partials of the row are here
#pragma unroll
          for (int u = 0; u < 8; ++u)
            if (lk[u] != 0.f) m = fmaxf(m, mk[u]);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          if (lk[u] == 0.f) continue;   // no key seen there
          const float w = exp2f(mk[u] - m);
          l += w * lk[u];
          acc.x += w * v[u].x;
          acc.y += w * v[u].y;
          acc.z += w * v[u].z;
          acc.w += w * v[u].w;
        }
      }
      if (step == 1) {
        sum[q][0][lane] = acc;
        if (lane == 0) den[q][0] = l;
      } else {
        sum[q][warp][lane] = acc;
        if (lane == 0) den[q][warp] = l;
      }
      // The row's maximum is the same for all its warps; the first keeps it.
      if (lane == 0 && (step == 1 || warp == 0)) row_max[q] = m;
    }
  }
  __syncthreads();
  const int parts = step == 8 ? 8 : 1;
  for (int q = warp; q < RB; q += 8) {
    if (row0 + q >= rows) continue;
    float4 acc = sum[q][0][lane];
    float l = den[q][0];
    for (int i = 1; i < parts; ++i) {
      const float4 v = sum[q][i][lane];
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
      l += den[q][i];
    }
    finish(row0 + q, acc, l, row_max[q]);
  }
}

// --------------------------------------------------------------- few rows
constexpr int FEW_QR = 16, FEW_TK = 128, FEW_THREADS = 128, FEW_WARPS = 4;
constexpr int FEW_KEYS = 32;          // of a warp in one unit: two halves of 16, each inside one page
constexpr float FEW_RESCALE = 8.f;    // log2 growth of the maximum that moves it
constexpr float FEW_OFFSET = 6.f;     // P is 2^6 at the maximum

// A warp's keys of one unit: where their codes lie and what they are scaled by.
struct FewUnit {
  int row[2];      // first row of each half in the [pages * heads * page, 128] code matrix
  int k0, live;    // first key position, live keys
  float ks[2], lv[2], iv[2];   // scales of K; log2 and reciprocal of the scales of V
  int e, h, last;  // last: the unit ends its item or the CTA's share
  int pad;
};

// Three CTAs fit an SM (four of the weights'): twelve warps, each with 12 KB (10)
// of its keys on their way or in use. (Two CTAs with 16 KB a warp took 104 us
// where this took 89: one token of 8 sequences of 18 to 32 thousand keys.)
template <bool WEIGHTS>
struct FewSmem {
  static constexpr int STAGES = WEIGHTS ? 5 : 3;                              // of 16 keys
  static constexpr uint32_t K_BYTES = 16 * 128;
  static constexpr uint32_t STAGE_BYTES = WEIGHTS ? K_BYTES : 2 * K_BYTES;    // K codes, V codes
  static constexpr uint32_t RING = FEW_WARPS * STAGES * STAGE_BYTES;
  static constexpr uint32_t LD = 132;                               // merge rows, padded
  static constexpr uint32_t MERGE_OFF = RING;
  static constexpr uint32_t MERGE_BYTES = WEIGHTS ? 0 : FEW_QR * LD * 4;
  static constexpr uint32_t ML_OFF = MERGE_OFF + MERGE_BYTES;       // m, l [warps][16]
  static constexpr uint32_t UNIT_OFF = ML_OFF + 2 * FEW_WARPS * FEW_QR * 4;   // [warps][2 batches][16]
  static constexpr uint32_t BAR_OFF = UNIT_OFF + FEW_WARPS * 32 * sizeof(FewUnit);
  static constexpr uint32_t SCHED_OFF = BAR_OFF + FEW_WARPS * STAGES * 8;
  static constexpr uint32_t TOTAL = 1024 + SCHED_OFF + sizeof(Kv8SchedSmem) + 16;
  static_assert(sizeof(FewUnit) == 56 && (WEIGHTS ? 4 : 3) * (TOTAL + 1024) <= 233472, "the CTAs must fit an SM");
};

// fp32 += f16 x f16: 16 rows x 16 x 8.
WAMB_DEV void mma_f16_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
WAMB_DEV uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
WAMB_DEV uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
  return v;
}

// The 16 rows of an (entry, head) as f16 A operands of eight 16-wide steps.
// Thread t = lane & 3 holds dims 16 t .. 16 t + 15 in words 0-3 of a row and
// 64 + 16 t .. in words 4-7; step w takes word w (the same order for queries
// and keys, so the sum over dims is the same).
struct FewQ {
  uint32_t a[8][4];
  float rf[2];        // row factor: (power-of-two row scale) * scale * log2(e); rows g, g + 8
  int seen[2];        // keys each row sees
};

WAMB_DEV void few_load_q(const Kv8AttnParams& p, int e, int h, FewQ& f) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int b = e;   // one query tile per sequence
  const int tokens = kv8_count(p.s, b), len = kv8_len(p.s, p.c, b);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int rr = g + 8 * half;
    const bool ok = rr < tokens * p.group;
    const int t = rr / p.group;
    const __nv_bfloat16* src = p.q + b * p.q_sb + t * p.q_st + (h * p.group + rr - t * p.group) * p.q_sh + 16 * t4;
    float x[8][4];
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint4 w = ok ? __ldg(reinterpret_cast<const uint4*>(src + (i >> 1) * 64 + (i & 1) * 8)) : make_uint4(0, 0, 0, 0);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = unpack_bf16(ws[k]);
        x[2 * i + (k >> 1)][2 * (k & 1)] = v.x;
        x[2 * i + (k >> 1)][2 * (k & 1) + 1] = v.y;
        amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
      }
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int ex = min(max(__float_as_int(amax) >> 23, 14), 254);
    const float up = __int_as_float((267 - ex) << 23);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      f.a[w][half] = pack_f16(x[w][0] * up, x[w][1] * up);
      f.a[w][2 + half] = pack_f16(x[w][2] * up, x[w][3] * up);
    }
    f.rf[half] = __int_as_float((ex - 13) << 23) * p.scale_log2;
    f.seen[half] = ok && p.causal ? max(0, min(len, len - tokens + t + 1)) : len;   // a missing row is never the one that masks
  }
}

// S [16 rows][32 keys] of a warp's keys at its two stages (swizzled rows of 128
// codes; eight lanes meet each bank twice, which costs less than ordering the
// pieces by row did in selects).
WAMB_DEV void few_scores(const uint32_t (&stage)[2], const FewQ& q, float (&s)[4][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t row = stage[j >> 1] + (8 * (j & 1) + g) * 128;
    const uint4 x = lds128(row + ((t4 ^ g) << 4)), y = lds128(row + (((t4 + 4) ^ g) << 4));
    const uint32_t w[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) s[j][i] = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) mma_f16_16816(s[j], q.a[k], e4m3x2_to_f16x2(w[k]), e4m3x2_hi_to_f16x2(w[k]));
  }
}

// Attention (WEIGHTS = false) and attention weights (true; each unit owns its
// keys' sums, so no sum has a racing order).
template <bool WEIGHTS>
__global__ void __launch_bounds__(FEW_THREADS, WEIGHTS ? 4 : 3)
    kv8_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                   const Kv8AttnParams p) {
  using L = FewSmem<WEIGHTS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  Kv8SchedSmem& sched = *reinterpret_cast<Kv8SchedSmem*>(smem + L::SCHED_OFF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::SCHED_OFF + sizeof(Kv8SchedSmem));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const uint32_t ring = smem_u32(smem) + warp * (L::STAGES * L::STAGE_BYTES);
  const uint32_t bars = smem_u32(smem + L::BAR_OFF) + warp * (L::STAGES * 8);
  FewUnit* units = reinterpret_cast<FewUnit*>(smem + L::UNIT_OFF) + warp * 32;
  if (lane == 0)
    for (int i = 0; i < L::STAGES; ++i) mbar_init(bars + 8 * i, 1);
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_barrier_init();
  pdl_wait();
  if constexpr (WEIGHTS) kv8_carry_base<FEW_THREADS>(p);
  Kv8Share sh;
  Kv8Item it;
  const bool work = kv8_share<FEW_QR, FEW_TK, FEW_THREADS>(p, blockIdx.x, sched, sh, it);
  if constexpr (!WEIGHTS) {
    if (threadIdx.x == 0) kv8_leave_join(p, sh, work, it);
  }
  if (!work) return;
  const int count = static_cast<int>(sh.u1 - sh.u0);
  bool began = it.start == sh.u0;      // the current item begins in this share

  // Batches of 16 units: lanes 2 i, 2 i + 1 look up the halves of unit i, a whole
  // batch ahead of its use. `it` moves over the line with them.
  auto load_batch = [&](int j0) {
    const int j = min(j0 + (lane >> 1), count - 1), hf = lane & 1;
    kv8_seek<FEW_QR, FEW_TK>(p, it, sh.u0 + j);
    const int tile = static_cast<int>(sh.u0 + j - it.start);
    const int k0 = tile * FEW_TK + warp * FEW_KEYS;
    const int live = max(0, min(FEW_KEYS, Kv8Line<FEW_QR, FEW_TK>::visible(p, it.e) - k0));
    int row = 0;
    float ks = 1.f, vs = 1.f;
    if (live > 16 * hf) {
      const int k = k0 + 16 * hf;
      int pid = kv8_page(p.s.table, p.s.width, p.c, it.e / p.qts, k >> p.c.page_log2);
      if (pid < 0) pid = 0;   // reported
      const long long blk = static_cast<long long>(pid) * p.c.heads + it.h;
      row = static_cast<int>((blk << p.c.page_log2) + (k & (p.c.page - 1)));
      ks = __ldg(p.c.k_scale + blk);
      if constexpr (!WEIGHTS) vs = __ldg(p.c.v_scale + blk);
    }
    FewUnit& u = units[(j0 & 16) + (lane >> 1)];
    u.row[hf] = row;
    u.ks[hf] = ks;
    u.lv[hf] = log2f(vs);
    u.iv[hf] = 1.f / vs;
    if (hf == 0) {
      u.k0 = k0;
      u.live = live;
      u.e = it.e;
      u.h = it.h;
      u.last = tile == it.n - 1 || j == count - 1;
    }
    it.e = __shfl_sync(0xffffffffu, it.e, 31);
    it.h = __shfl_sync(0xffffffffu, it.h, 31);
    it.n = __shfl_sync(0xffffffffu, it.n, 31);
    it.start = __shfl_sync(0xffffffffu, it.start, 31);
    __syncwarp();
  };
  // Ring loads, 16 keys each: issued and consumed so far; the next half to
  // issue; units looked up.
  uint32_t issued = 0, used = 0;
  int ahead = 0, known = 0;
  auto issue = [&]() {
    while (ahead < 2 * known && issued < used + L::STAGES) {
      const FewUnit& u = units[(ahead >> 1) & 31];
      if (u.live > 16 * (ahead & 1)) {
        if (lane == 0) {
          const uint32_t st = issued % L::STAGES, at = ring + st * L::STAGE_BYTES, bar = bars + 8 * st;
          const int row = u.row[ahead & 1];
          mbar_arrive_expect_tx(bar, L::STAGE_BYTES);
          tma_load_2d(at, &tmK, bar, 0, row);
          if constexpr (!WEIGHTS) tma_load_2d(at + L::K_BYTES, &tmV, bar, 0, row);
        }
        ++issued;
      }
      ++ahead;
    }
  };
  // The first item's queries are asked for before its pages are looked up.
  FewQ q;
  few_load_q(p, it.e, it.h, q);
  bool loaded = true;
  load_batch(0);
  known = min(16, count);
  issue();

  float o[16][4];
  float m[2], l[2];
  auto reset = [&]() {
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
  };
  bool fresh = true;
  bool ok = true;
  for (int j = 0; j < count; ++j) {
    if ((j & 15) == 4 && known < count) {   // the batch before this one is used up: its places take the next
      load_batch(known);
      known = min(known + 16, count);
      issue();
    }
    const FewUnit& u = units[j & 31];
    const int live = u.live, k0 = u.k0, last = u.last;
    if (fresh) {
      if (!loaded) few_load_q(p, u.e, u.h, q);
      loaded = false;
      if constexpr (WEIGHTS) {
        // The rows' log-sum-exp in log2 units; rows that see nothing add nothing.
        const int tokens = kv8_count(p.s, u.e);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int rr = g + 8 * half, t = rr / p.group;
          l[half] = INFINITY;
          if (rr < tokens * p.group) {
            const float x = p.lse_in[(static_cast<long long>(u.e) * p.s.tokens + t) * (p.c.heads * p.group) + u.h * p.group +
                                     rr - t * p.group];
            if (x != -INFINITY) l[half] = x * 1.4426950408889634f;
          }
        }
      } else {
        reset();
      }
      fresh = false;
    }
    if (live > 0) {
      const float ks[2] = {u.ks[0], u.ks[1]};
      [[maybe_unused]] const float lv[2] = {u.lv[0], u.lv[1]}, iv[2] = {u.iv[0], u.iv[1]};
      const uint32_t st0 = used % L::STAGES, st1 = st0 + 1 == L::STAGES ? 0 : st0 + 1;
      const uint32_t stage[2] = {ring + st0 * L::STAGE_BYTES, ring + st1 * L::STAGE_BYTES};
      const bool two = live > 16;
      auto arrived = [&]() {
        ok = mbar_wait(bars + 8 * st0, (used / L::STAGES) & 1, abort_flag) && ok;
        if (two) ok = mbar_wait(bars + 8 * st1, ((used + 1) / L::STAGES) & 1, abort_flag) && ok;
      };
      if constexpr (WEIGHTS) {
        // Lane (g, t) finishes key 8 (g / 2) + 2 t + g % 2.
        const int key = 8 * (g >> 1) + 2 * t4 + (g & 1);
        const long long at = (static_cast<long long>(u.e) * p.c.heads + u.h) * p.w_cap + k0 + key;
        const float base = p.base != nullptr && key < live ? __ldcg(p.base + at) : 0.f;
        arrived();
        float s[4][4];
        few_scores(stage, q, s);
        __syncwarp();
        used += two ? 2 : 1;
        issue();
        float mine = 0.f;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          const float f0 = q.rf[0] * ks[jt >> 1], f1 = q.rf[1] * ks[jt >> 1];
          const int kk = k0 + 8 * jt + 2 * t4;
          float w[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float a = ex2_mufu(fmaf(s[jt][c], f0, -l[0])), d = ex2_mufu(fmaf(s[jt][2 + c], f1, -l[1]));
            w[c] = (kk + c < q.seen[0] ? a : 0.f) + (kk + c < q.seen[1] ? d : 0.f);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) w[c] += __shfl_xor_sync(0xffffffffu, w[c], x);
          }
          if (jt == g >> 1) mine = (g & 1) ? w[1] : w[0];
        }
        if (key < live) p.weights[at] = ok ? base + mine : 0.f;
      } else {
        arrived();
        float s[4][4];
        few_scores(stage, q, s);
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          const float f[2] = {q.rf[0] * ks[jt >> 1], q.rf[1] * ks[jt >> 1]};
#pragma unroll
          for (int c = 0; c < 4; ++c) s[jt][c] = fmaf(s[jt][c], f[c >> 1], lv[jt >> 1]);
        }
        if (__any_sync(0xffffffffu, k0 + FEW_KEYS > min(q.seen[0], q.seen[1]))) {
#pragma unroll
          for (int jt = 0; jt < 4; ++jt)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (k0 + 8 * jt + 2 * t4 + (c & 1) >= q.seen[c >> 1]) s[jt][c] = -INFINITY;
        }
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          mx[0] = fmax3(mx[0], s[jt][0], s[jt][1]);
          mx[1] = fmax3(mx[1], s[jt][2], s[jt][3]);
        }
        if (__any_sync(0xffffffffu, mx[0] > m[0] + FEW_RESCALE || mx[1] > m[1] + FEW_RESCALE)) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float v = mx[half];
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
            v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
            const float nm = fmaxf(m[half], v);
            const float a = m[half] == -INFINITY ? 0.f : exp2f(m[half] - nm);
            m[half] = nm;
            l[half] *= a;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              o[i][2 * half] *= a;
              o[i][2 * half + 1] *= a;
            }
          }
        }
        const float z0 = (m[0] == -INFINITY ? 0.f : m[0]) - FEW_OFFSET, z1 = (m[1] == -INFINITY ? 0.f : m[1]) - FEW_OFFSET;
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
          s[jt][0] = ex2_mufu(s[jt][0] - z0);
          s[jt][1] = ex2_mufu(s[jt][1] - z0);
          s[jt][2] = ex2_mufu(s[jt][2] - z1);
          s[jt][3] = ex2_mufu(s[jt][3] - z1);
          l[0] = fmaf(s[jt][0] + s[jt][1], iv[jt >> 1], l[0]);
          l[1] = fmaf(s[jt][2] + s[jt][3], iv[jt >> 1], l[1]);
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          // V rows 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t of the half, dims [16 g, +16);
          // output column n = g of product i is dim 16 g + i.
          const uint32_t a[4] = {pack_f16(s[2 * kk][0], s[2 * kk][1]), pack_f16(s[2 * kk][2], s[2 * kk][3]),
                                 pack_f16(s[2 * kk + 1][0], s[2 * kk + 1][1]), pack_f16(s[2 * kk + 1][2], s[2 * kk + 1][3])};
          if (kk == 1 && !two) break;     // no keys there
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = (i >> 1) * 8 + 2 * t4 + (i & 1);
            v[i] = lds128(stage[kk] + L::K_BYTES + r * 128 + ((g ^ (r & 7)) << 4));
          }
          if (live < 16 * kk + 16) {      // whatever lies behind the keys (NaN codes too) counts for nothing
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (16 * kk + (i >> 1) * 8 + 2 * t4 + (i & 1) >= live) v[i] = make_uint4(0, 0, 0, 0);
          }
          __syncwarp();
          ++used;
          issue();
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t v0 = w == 0 ? v[0].x : w == 1 ? v[0].y : w == 2 ? v[0].z : v[0].w;
            const uint32_t v1 = w == 0 ? v[1].x : w == 1 ? v[1].y : w == 2 ? v[1].z : v[1].w;
            const uint32_t v2 = w == 0 ? v[2].x : w == 1 ? v[2].y : w == 2 ? v[2].z : v[2].w;
            const uint32_t v3 = w == 0 ? v[3].x : w == 1 ? v[3].y : w == 2 ? v[3].z : v[3].w;
            const uint32_t lo0 = __byte_perm(v0, v1, 0x5140), hi0 = __byte_perm(v0, v1, 0x7362);
            const uint32_t lo1 = __byte_perm(v2, v3, 0x5140), hi1 = __byte_perm(v2, v3, 0x7362);
            mma_f16_16816(o[4 * w], a, e4m3x2_to_f16x2(lo0), e4m3x2_to_f16x2(lo1));
            mma_f16_16816(o[4 * w + 1], a, e4m3x2_hi_to_f16x2(lo0), e4m3x2_hi_to_f16x2(lo1));
            mma_f16_16816(o[4 * w + 2], a, e4m3x2_to_f16x2(hi0), e4m3x2_to_f16x2(hi1));
            mma_f16_16816(o[4 * w + 3], a, e4m3x2_hi_to_f16x2(hi0), e4m3x2_hi_to_f16x2(hi1));
          }
        }
      }
    }
    if (!last) continue;
    fresh = true;
    if constexpr (!WEIGHTS) {
      // The item, or the share, ends: the warps' results meet in shared memory.
      float* wm = reinterpret_cast<float*>(smem + L::ML_OFF);
      float* wl = wm + FEW_WARPS * FEW_QR;
      float* buf = reinterpret_cast<float*>(smem + L::MERGE_OFF);
      const int b = u.e, h = u.h;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
        if (t4 == 0) {
          wm[warp * FEW_QR + g + 8 * half] = m[half];
          wl[warp * FEW_QR + g + 8 * half] = l[half];
        }
      }
      __syncthreads();
      const int rows = min(FEW_QR, kv8_count(p.s, b) * p.group);
      // One warp after another adds its rows, relative to the largest maximum.
      for (int w = 0; w < FEW_WARPS; ++w) {
        if (w == warp) {
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int r = g + 8 * half;
            if (r < rows) {
              float M = -INFINITY;
#pragma unroll
              for (int x = 0; x < FEW_WARPS; ++x) M = fmaxf(M, wm[x * FEW_QR + r]);
              const float f = m[half] == -INFINITY && l[half] == 0.f ? 0.f : exp2f(m[half] - M);
#pragma unroll
              for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                  float4* to = reinterpret_cast<float4*>(buf + r * L::LD + 32 * t4 + 16 * c + i);
                  float4 v = w == 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *to;
                  v.x = fmaf(f, o[i][2 * half + c], v.x);
                  v.y = fmaf(f, o[i + 1][2 * half + c], v.y);
                  v.z = fmaf(f, o[i + 2][2 * half + c], v.z);
                  v.w = fmaf(f, o[i + 3][2 * half + c], v.w);
                  *to = v;
                }
            }
          }
        }
        __syncthreads();
      }
      // Whole only when the share holds the item's first and last unit.
      const int n = max(1, (Kv8Line<FEW_QR, FEW_TK>::visible(p, b) + FEW_TK - 1) / FEW_TK);
      const bool whole = began && (k0 - warp * FEW_KEYS) / FEW_TK == n - 1;
      float* part = p.part + static_cast<size_t>(2 * blockIdx.x + (began ? 1 : 0)) * kv8_part_floats<FEW_QR>();
      for (int i = threadIdx.x; i < rows * 32; i += FEW_THREADS) {
        const int r = i >> 5, c4 = i & 31;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) M = fmaxf(M, wm[w * FEW_QR + r]);
        const float4 acc = *reinterpret_cast<const float4*>(buf + r * L::LD + c4 * 4);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_WARPS; ++w) {
          const float mw = wm[w * FEW_QR + r], lw = wl[w * FEW_QR + r];
          if (lw != 0.f) den += exp2f(mw - M) * lw;
        }
        const float mref = M == -INFINITY ? M : M - FEW_OFFSET;
        if (!ok) den = 0.f;
        if (whole) {
          const int t = r / p.group, hq = h * p.group + r - t * p.group;
          const float inv = den == 0.f ? 0.f : 1.f / den;
          *reinterpret_cast<uint2*>(p.out + b * p.o_sb + t * p.o_st + hq * p.o_sh + c4 * 4) =
              make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
          if (p.lse != nullptr && c4 == 0)
            p.lse[(static_cast<long long>(b) * p.s.tokens + t) * (p.c.heads * p.group) + hq] = kv8_row_lse(mref, den);
        } else {
          reinterpret_cast<float4*>(part + r * 128)[c4] = acc;
          if (c4 == 0) {
            part[FEW_QR * 128 + r] = mref;
            part[FEW_QR * 129 + r] = den;
          }
        }
      }
      __syncthreads();
      began = true;
    }
  }
  // Every load has been waited for, unless a wait ran out or ended early because
  // another warp's did: a CTA must not exit with loads on their way, so it stays
  // for a thousand times the latency of memory. (Counting what is on its way
  // into the loop's end cost 8% of the one-token attention.)
  if (*abort_flag)
    for (const uint64_t t0 = globaltimer(); globaltimer() - t0 < 1000000;) {}
}

}  // namespace wamb
