// A paged KV cache held in E4M3 with one scale for each (page, head), and the
// kernels that write it and shrink it. (Attention over it: kv8_few.cuh,
// kv8_tc.cuh.)
//
// Layout: codes [pages, heads, page, 128] bytes, scale [pages, heads] fp32;
// position p of sequence b is row p % page of page table[b, p / page].
// A scale is a power of two, 2^n with n the smallest whole number in
// [-40, 119] such that the block's largest magnitude is at most 448 * 2^n.
// A power of two makes x / s exact, so that a value is rounded once: by at most
// 2^-4 of itself from 2^-6 s on, by at most 2^-10 s below, where E4M3's steps
// no longer shrink (what is below 2^-10 s becomes 0). Moving a block's codes to a
// larger scale (a later token of the block is larger) rounds again only what
// falls below that normal range: a general scale would add a rounding at every
// growth.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"
#include "host.cuh"

namespace wamb {

constexpr int KV8_EXP_MIN = -40, KV8_EXP_MAX = 119;
constexpr int KV8_DEV_ERROR = 5;   // WAMB_DEV_KV8: page id, length or count out of range

struct Kv8Cache {
  uint8_t* k8;
  uint8_t* v8;
  float* k_scale;
  float* v_scale;
  int pages, heads, page, page_log2;
};

// The sequences of a call.
struct Kv8Seqs {
  const int* table;    // [batch, width] page ids
  const int* lens;     // [batch]
  const int* counts;   // [batch] valid tokens of this call, or null (all)
  int batch, width, tokens;
};

// Cached tokens of sequence b. A length out of range is reported and counts as
// `bad`: none, so that nothing is read, added up or kept by a wrong length.
WAMB_DEV int kv8_len(const Kv8Seqs& s, const Kv8Cache& c, int b, int bad = 0) {
  const int n = __ldg(s.lens + b);
  const long long cap = static_cast<long long>(s.width) << c.page_log2;
  if (n < 0 || n > cap) {
    record_error(KV8_DEV_ERROR);
    return bad;
  }
  return n;
}
// Valid rows of sequence b in this call; none (reported) for a count out of range.
WAMB_DEV int kv8_count(const Kv8Seqs& s, int b) {
  if (s.counts == nullptr) return s.tokens;
  const int n = __ldg(s.counts + b);
  if (n < 0 || n > s.tokens) {
    record_error(KV8_DEV_ERROR);
    return 0;
  }
  return n;
}
// Entry `i` of a page table row; -1 (reported) when it names no page.
WAMB_DEV int kv8_page(const int* table, int width, const Kv8Cache& c, int b, int i) {
  const int pid = __ldg(table + static_cast<long long>(b) * width + i);
  if (pid < 0 || pid >= c.pages) {
    record_error(KV8_DEV_ERROR);
    return -1;
  }
  return pid;
}

WAMB_DEV float pow2f_exact(int n) { return __int_as_float((n + 127) << 23); }   // -126 <= n <= 127

// n of the block scale 2^n for the largest magnitude `amax` (>= 0).
// 448 = 1.75 * 2^8: with amax = 1.m * 2^e, n = e - 8, one more when 1.m > 1.75.
WAMB_DEV int kv8_scale_exp(float amax) {
  const int bits = __float_as_int(fminf(amax, 3.402823466e38f));
  const int n = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return max(KV8_EXP_MIN, min(KV8_EXP_MAX, n));
}

// Two E4M3 codes (low 16 bits) -> f16x2, exact.
WAMB_DEV uint32_t e4m3x2_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
// The same of the high 16 bits.
WAMB_DEV uint32_t e4m3x2_hi_to_f16x2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
WAMB_DEV float2 e4m3x2_to_float2(uint32_t codes) {
  const uint32_t h = e4m3x2_to_f16x2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
WAMB_DEV void e4m3x8_to_float(uint2 w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t u = i < 2 ? w.x : w.y;
    const float2 v = e4m3x2_to_float2((i & 1) ? u >> 16 : u & 0xffffu);
    f[2 * i] = v.x;
    f[2 * i + 1] = v.y;
  }
}

// Largest of a value over the block (fmaxf: NaN loses).
template <int THREADS>
WAMB_DEV float kv8_block_max(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) v = fmaxf(v, red[i]);
  return v;
}

// Threads of a block that holds a page's rows of one head in registers.
__host__ __device__ constexpr int kv8_page_threads(int page) { return page < 128 ? 128 : 256; }

// ------------------------------------------------------------------- write
struct Kv8WriteParams {
  Kv8Cache c;
  Kv8Seqs s;
  const void* x[2];            // K, V
  long long sb[2], st[2], sh[2];   // element strides of (batch, token, head)
};

// One block per (touched page, head, sequence, K or V): the block's new rows
// stay in registers between the amax and the rounding, so each is read once.
// Eight threads hold a row, 16 values each.
// Bound by memory for chunks: 8 x 880 rows of 24 heads (130 MB) take 24.7 us,
// 5.3 TB/s; 27.5 with twice the threads and half the loads of each in flight,
// 28.4 with 8 values a thread. By the launch for single tokens (2.2 us).
template <bool F32, int PAGE>
__global__ void __launch_bounds__(kv8_page_threads(PAGE)) kv8_write_kernel(const Kv8WriteParams p) {
  pdl_wait();
  constexpr int THREADS = kv8_page_threads(PAGE), ROWS = THREADS / 8, PASSES = PAGE / ROWS;
  constexpr int WORDS = F32 ? 4 : 2;      // 16-byte pieces of 16 values
  __shared__ float red[THREADS / 32];
  const int h = blockIdx.y, b = blockIdx.z >> 1, which = blockIdx.z & 1;
  // A sequence with a length or count out of range, or without room in its table
  // for all of its rows, is left as it was: its history must not be written over,
  // nor rounded again to a scale that rows at wrong places would set.
  const int start = kv8_len(p.s, p.c, b, -1);
  if (start < 0) return;
  const int cnt = kv8_count(p.s, b);
  if (start + static_cast<long long>(cnt) > static_cast<long long>(p.s.width) * PAGE) {
    if (threadIdx.x == 0) record_error(KV8_DEV_ERROR);
    return;
  }
  const int pi = start / PAGE + blockIdx.x;
  const int lo = max(start, pi * PAGE);
  const int hi = static_cast<int>(min(static_cast<long long>(start) + cnt, (pi + 1ll) * PAGE));
  if (lo >= hi) return;
  const int pid = kv8_page(p.s.table, p.s.width, p.c, b, pi);
  if (pid < 0) return;
  const int held = lo - pi * PAGE, n = hi - lo;
  const int c16 = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  const long long base = b * p.sb[which] + h * p.sh[which] + (lo - start) * p.st[which] + c16 * 16;

  uint4 raw[PASSES][WORDS];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + ROWS * i;
    const uint4* src = reinterpret_cast<const uint4*>(static_cast<const char*>(p.x[which]) +
                                                      (base + r * p.st[which]) * (F32 ? 4 : 2));
#pragma unroll
    for (int k = 0; k < WORDS; ++k) raw[i][k] = r < n ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
  }
  // Values 8 half .. 8 half + 7 of row i.
  auto value = [&](int i, int half, float (&f)[8]) {
    if constexpr (F32) {
      const uint4 a = raw[i][2 * half], d = raw[i][2 * half + 1];
      f[0] = __uint_as_float(a.x); f[1] = __uint_as_float(a.y); f[2] = __uint_as_float(a.z); f[3] = __uint_as_float(a.w);
      f[4] = __uint_as_float(d.x); f[5] = __uint_as_float(d.y); f[6] = __uint_as_float(d.z); f[7] = __uint_as_float(d.w);
    } else {
      const uint32_t w[4] = {raw[i][half].x, raw[i][half].y, raw[i][half].z, raw[i][half].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = unpack_bf16(w[k]);
        f[2 * k] = v.x;
        f[2 * k + 1] = v.y;
      }
    }
  };
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float f[8];
      value(i, half, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) amax = fmaxf(amax, fabsf(f[k]));
    }
  amax = kv8_block_max<THREADS>(amax, red);
  const long long blk = static_cast<long long>(pid) * p.c.heads + h;
  float* scale = (which ? p.c.v_scale : p.c.k_scale) + blk;
  uint8_t* codes = (which ? p.c.v8 : p.c.k8) + blk * (PAGE * 128) + c16 * 16;
  const float s_old = held > 0 ? *scale : 0.f;
  const float s = fmaxf(pow2f_exact(kv8_scale_exp(amax)), s_old);
  const float inv = 1.f / s;
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int r = r0 + ROWS * i;
    if (r >= n) continue;
    uint2 part[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float f[8];
      value(i, half, f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= inv;
      part[half] = pack_e4m3x8(f);
    }
    *reinterpret_cast<uint4*>(codes + (held + r) * 128) = make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
  }
  if (s > s_old) {   // earlier tokens of the block move to the larger scale
    const float ratio = s_old * inv;
    for (int r = r0; r < held; r += ROWS) {
      uint4* at = reinterpret_cast<uint4*>(codes + r * 128);
      const uint4 was = *at;
      uint2 part[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float f[8];
        e4m3x8_to_float(half ? make_uint2(was.z, was.w) : make_uint2(was.x, was.y), f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] *= ratio;
        part[half] = pack_e4m3x8(f);
      }
      *at = make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
    }
    __syncthreads();   // every thread has read the old scale
    if (threadIdx.x == 0) *scale = s;
  }
}

// ------------------------------------------------------------------ evict
struct Kv8EvictParams {
  Kv8Cache c;
  Kv8Seqs s;                 // counts null
  const float* weights;      // [batch, heads, cap]
  long long cap;             // columns of `weights`
  const int* new_table;      // [batch, new_width]
  int new_width;
  int heavy, recent;
  int* kept;                 // [batch, heads, new_width * page]
  float* new_weights;        // like kept
  int* new_lens;             // [batch]
};

// Order-preserving map of a weight: larger weights have larger keys, NaN
// (either sign) is largest, -0 equals +0.
WAMB_DEV uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.f);
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Kept tokens of sequence b: all of the last `recent`, and `heavy` of the rest.
struct Kv8Kept {
  int len, old, heavy, total;   // positions [0, old) compete for `heavy` places
};
WAMB_DEV Kv8Kept kv8_kept(const Kv8EvictParams& p, int b) {
  Kv8Kept k;
  k.len = kv8_len(p.s, p.c, b);
  const int recent = min(p.recent, k.len);
  k.old = k.len - recent;
  k.heavy = min(p.heavy, k.old);
  k.total = k.heavy + recent;
  // More than the new pages hold (the length is above the caller's max_len):
  // cut, the sequence would lose its latest positions. It keeps nothing.
  if (k.total > static_cast<long long>(p.new_width) << p.c.page_log2) {
    record_error(KV8_DEV_ERROR);
    k.heavy = k.total = 0;
  }
  return k;
}

constexpr int KV8_SEL_THREADS = 1024, KV8_SEL_BINS = 2048, KV8_SEL_COPIES = 4;
constexpr int KV8_SEL_KEYS = 36864;       // keys of one head that shared memory holds
constexpr int KV8_SEL_LIST = 8192;        // keys of one bin that it holds apart
constexpr uint32_t KV8_SEL_SMEM = (KV8_SEL_KEYS + KV8_SEL_LIST) * 4;

struct Kv8SelSmem {
  int hist[KV8_SEL_COPIES][KV8_SEL_BINS];
  uint32_t wsum[32];
  int pick[2], listed;
};

// Exclusive sum over the block's threads of v, and the sum of all.
WAMB_DEV uint32_t kv8_block_scan(Kv8SelSmem& sm, uint32_t v, uint32_t& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += u;
  }
  if (lane == 31) sm.wsum[warp] = inc;
  __syncthreads();
  uint32_t sums = sm.wsum[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, sums, o);
    if (lane >= o) sums += u;
  }
  const uint32_t before = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
  all = __shfl_sync(0xffffffffu, sums, 31);
  return inc - v + (warp > 0 ? before : 0);
}

// The bin, counted from the highest, that holds the `need`-th largest key of
// the histogram, and how many of that bin are needed. Whole block.
WAMB_DEV void kv8_pick_bin(Kv8SelSmem& sm, int need) {
  const int tid = threadIdx.x;
  __syncthreads();
  // Each thread owns two bins, highest first: thread t has bins 2047 - 2t, 2046 - 2t.
  int c[2], mine = 0;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int bin = KV8_SEL_BINS - 1 - 2 * tid - j;
    c[j] = 0;
#pragma unroll
    for (int q = 0; q < KV8_SEL_COPIES; ++q) c[j] += sm.hist[q][bin];
    mine += c[j];
  }
  uint32_t all;
  int above = kv8_block_scan(sm, mine, all);
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    if (above < need && need <= above + c[j]) {
      sm.pick[0] = KV8_SEL_BINS - 1 - 2 * tid - j;
      sm.pick[1] = need - above;
    }
    above += c[j];
  }
  __syncthreads();
}
WAMB_DEV void kv8_clear_hist(Kv8SelSmem& sm) {
  for (int i = threadIdx.x; i < KV8_SEL_COPIES * KV8_SEL_BINS; i += KV8_SEL_THREADS) (&sm.hist[0][0])[i] = 0;
  __syncthreads();
}

// A thread's run of a piece of keys, of an odd length so that the threads of a
// warp meet different banks, and at most 31 so that a word marks its keys.
constexpr int KV8_SEL_PIECE = 31 * KV8_SEL_THREADS;
struct Kv8Run {
  int from, len;
  WAMB_DEV explicit Kv8Run(int n) {
    const int c = (n + KV8_SEL_THREADS - 1) / KV8_SEL_THREADS | 1;
    from = min(n, static_cast<int>(threadIdx.x) * c);
    len = min(n - from, c);
  }
  // Bit j: f(key j of the run).
  template <typename F>
  WAMB_DEV uint32_t mark(const uint32_t* keys, F f) const {
    uint32_t m = 0;
    for (int j0 = 0; j0 < len; j0 += 8) {
      uint32_t part = 0;
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (j0 + u < len && f(keys[from + j0 + u])) part |= 1u << u;
      m |= part << j0;
    }
    return m;
  }
};

// Keeps k.heavy of the positions [0, k.old) and writes them, in order.
// HELD: the keys fit shared memory.
template <bool HELD>
WAMB_DEV void kv8_select_heavy(const Kv8Kept& k, const float* w, Kv8SelSmem& sm, uint32_t* keys, uint32_t* list, int* kept,
                               float* nw) {
  const int tid = threadIdx.x, warp = tid >> 5;
  auto key_at = [&](int i) { return HELD ? keys[i] : weight_key(__ldg(w + i)); };
  const bool select = k.heavy < k.old;
  int* hist = sm.hist[warp & (KV8_SEL_COPIES - 1)];
  uint32_t prefix = 0;             // the threshold's bits fixed so far
  int need = k.heavy;              // places left among keys that match them
  if (select) kv8_clear_hist(sm);
  if (HELD || select)
    for (int i0 = tid; i0 < k.old; i0 += 8 * KV8_SEL_THREADS) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = i0 + u * KV8_SEL_THREADS < k.old ? __ldg(w + i0 + u * KV8_SEL_THREADS) : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * KV8_SEL_THREADS;
        if (i < k.old) {
          const uint32_t key = weight_key(v[u]);
          if (HELD) keys[i] = key;
          if (select) atomicAdd(hist + (key >> 21), 1);
        }
      }
    }
  if (select) {
    kv8_pick_bin(sm, need);
    prefix = static_cast<uint32_t>(sm.pick[0]) << 21;
    need = sm.pick[1];
    // The bin's keys go to a list of their own: the two further digits look at
    // them alone (at all keys again where the list overflows).
    if (tid == 0) sm.listed = 0;
    __syncthreads();
    if (HELD) {          // (atomics on one counter took 7 cycles a key)
      int listed = 0;
      for (int base = 0; base < k.old; base += KV8_SEL_PIECE) {
        const Kv8Run run(min(KV8_SEL_PIECE, k.old - base));
        uint32_t m = run.mark(keys + base, [&](uint32_t key) { return (key ^ prefix) >> 21 == 0; });
        uint32_t all;
        int at = listed + static_cast<int>(kv8_block_scan(sm, __popc(m), all));
        for (; m != 0; m &= m - 1, ++at)
          if (at < KV8_SEL_LIST) list[at] = keys[base + run.from + __ffs(m) - 1];
        listed += static_cast<int>(all);
        __syncthreads();            // the sums are rewritten
      }
      if (tid == 0) sm.listed = listed;
    } else {
      for (int i0 = tid; i0 < k.old; i0 += 8 * KV8_SEL_THREADS) {
        uint32_t key[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) key[u] = i0 + u * KV8_SEL_THREADS < k.old ? key_at(i0 + u * KV8_SEL_THREADS) : ~prefix;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          if ((key[u] ^ prefix) >> 21 == 0) {
            const int at = atomicAdd(&sm.listed, 1);
            if (at < KV8_SEL_LIST) list[at] = key[u];
          }
      }
    }
    __syncthreads();
    const bool short_list = sm.listed <= KV8_SEL_LIST;
    const int n = short_list ? sm.listed : k.old;
#pragma unroll 1
    for (int pass = 1; pass < 3; ++pass) {
      const int shift = pass == 1 ? 10 : 0, above = pass == 1 ? 21 : 10;
      const uint32_t digit = pass == 1 ? 0x7ffu : 0x3ffu;
      kv8_clear_hist(sm);
      for (int i = tid; i < n; i += KV8_SEL_THREADS) {
        const uint32_t key = short_list ? list[i] : key_at(i);
        if ((key ^ prefix) >> above == 0) atomicAdd(hist + ((key >> shift) & digit), 1);
      }
      kv8_pick_bin(sm, need);
      prefix |= static_cast<uint32_t>(sm.pick[0]) << shift;
      need = sm.pick[1];
      __syncthreads();
    }
  }
  // Ordered compaction: keys above the threshold and, of those equal to it, the
  // `need` lowest positions. A thread marks the kept ones of its run; the runs
  // before it tell their places; the positions then lie in shared memory, over
  // the keys, and leave it in order. (Ballots and population counts of a warp's
  // neighbouring keys took twice as long.)
  int done = 0, eq_done = 0;
  for (int base = 0; base < k.old; base += KV8_SEL_PIECE) {
    const int n = min(KV8_SEL_PIECE, k.old - base);
    if (!HELD && select) {
      for (int i = tid; i < n; i += KV8_SEL_THREADS) keys[i] = weight_key(__ldg(w + base + i));
    }
    __syncthreads();
    const Kv8Run run(n);
    const uint32_t* piece = HELD ? keys + base : keys;
    uint32_t keep = select ? run.mark(piece, [&](uint32_t key) { return key > prefix; }) : (1u << run.len) - 1;
    uint32_t equal = select ? run.mark(piece, [&](uint32_t key) { return key == prefix; }) : 0u;
    uint32_t all;
    const uint32_t before = kv8_block_scan(sm, __popc(keep) + (static_cast<uint32_t>(__popc(equal)) << 16), all);
    int e = eq_done + static_cast<int>(before >> 16);
    const int first = done + min(eq_done, need);           // of this piece, among all kept
    int to = done + static_cast<int>(before & 0xffff) + min(e, need) - first;
    for (; equal != 0 && e < need; equal &= equal - 1, ++e) keep |= equal & (0u - equal);
    for (; keep != 0; keep &= keep - 1) keys[to++] = base + run.from + __ffs(keep) - 1;
    done += static_cast<int>(all & 0xffff);
    eq_done += static_cast<int>(all >> 16);
    const int last = done + min(eq_done, need);
    __syncthreads();
    for (int j0 = first + tid; j0 < last; j0 += 4 * KV8_SEL_THREADS) {
      int at[4];
      float v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) at[u] = j0 + u * KV8_SEL_THREADS < last ? keys[j0 + u * KV8_SEL_THREADS - first] : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = at[u] >= 0 ? __ldg(w + at[u]) : 0.f;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (at[u] >= 0) {
          kept[j0 + u * KV8_SEL_THREADS] = at[u];
          nw[j0 + u * KV8_SEL_THREADS] = v[u];
        }
    }
    __syncthreads();        // the sums and the keys are rewritten
  }
}

// One block per (head, sequence). The heavy-th largest key is found by a
// radix select (11, 11 and 10 bits, histograms in shared memory: whole-number
// counts, so the order of the atomics does not matter), then one ordered pass
// writes the kept positions. The weights are read once into shared memory, or
// from L2 in each pass where a head has more than 36864. Bound by that one
// SM's instructions (an instruction a key is 240 cycles at 31k keys): 64 heads
// of 31k weights take 22 us of the 72 that an eviction of 8 x 32k tokens takes,
// 24 heads of 3520 take 10 of 17. A sequence whose new pages overlap its old
// ones, or one another, or do not exist is refused: it keeps nothing.
__global__ void __launch_bounds__(KV8_SEL_THREADS) kv8_select_kernel(const Kv8EvictParams p, const int list_at) {
  pdl_wait();
  extern __shared__ uint32_t keys[];
  __shared__ Kv8SelSmem sm;
  const int tid = threadIdx.x;
  const int h = blockIdx.x, b = blockIdx.y;
  Kv8Kept k = kv8_kept(p, b);
  const float* w = p.weights + (static_cast<long long>(b) * p.c.heads + h) * p.cap;
  const long long out_cap = static_cast<long long>(p.new_width) << p.c.page_log2;
  const long long out0 = (static_cast<long long>(b) * p.c.heads + h) * out_cap;
  int* kept = p.kept + out0;
  float* nw = p.new_weights + out0;

  const int new_pages = (k.total + p.c.page - 1) >> p.c.page_log2, old_pages = (k.len + p.c.page - 1) >> p.c.page_log2;
  const int* fresh = p.new_table + static_cast<long long>(b) * p.new_width;
  // No page may be named twice by the new pages, nor be one of the old. A bit
  // for each page id, modulo their number 262144, tells that none is.
  uint32_t* bits = reinterpret_cast<uint32_t*>(&sm.hist[0][0]);
  constexpr uint32_t WORDS = KV8_SEL_COPIES * KV8_SEL_BINS;
  const int* used = p.s.table + static_cast<long long>(b) * p.s.width;
  kv8_clear_hist(sm);
  bool overlap = false, none = false;      // none: a new page that does not exist (its rows would be lost)
  for (int n = tid; n < new_pages; n += KV8_SEL_THREADS) {
    const uint32_t page = static_cast<uint32_t>(__ldg(fresh + n));
    none |= page >= static_cast<uint32_t>(p.c.pages);
    overlap |= atomicOr(bits + (page >> 5) % WORDS, 1u << (page & 31)) >> (page & 31) & 1;
  }
  __syncthreads();
  for (int o = tid; o < old_pages; o += KV8_SEL_THREADS) {
    const uint32_t page = static_cast<uint32_t>(__ldg(used + o));
    overlap |= bits[(page >> 5) % WORDS] >> (page & 31) & 1;
  }
  if (__syncthreads_or(overlap)) {
    // Where a bit is met twice, each window of 262144 ids has the bits to itself
    // (larger caches: ids that are alike collide). Two passes over the tables a
    // window: for 4096 new pages and 16384 old ones 8 us in three windows, where the
    // comparison of all pairs took 2.1 ms.
    overlap = false;
    for (int from = 0; from < p.c.pages; from += 32 * WORDS) {
      kv8_clear_hist(sm);
      for (int n = tid; n < new_pages; n += KV8_SEL_THREADS) {
        const uint32_t at = static_cast<uint32_t>(__ldg(fresh + n)) - from;
        if (at < 32 * WORDS) overlap |= atomicOr(bits + (at >> 5), 1u << (at & 31)) >> (at & 31) & 1;
      }
      __syncthreads();
      for (int o = tid; o < old_pages; o += KV8_SEL_THREADS) {
        const uint32_t at = static_cast<uint32_t>(__ldg(used + o)) - from;
        if (at < 32 * WORDS) overlap |= bits[at >> 5] >> (at & 31) & 1;
      }
      __syncthreads();       // the bits are cleared
    }
  }
  if (__syncthreads_or(overlap || none)) {
    if (tid == 0) record_error(KV8_DEV_ERROR);
    k.heavy = k.total = 0;
  }
  if (h == 0 && tid == 0) p.new_lens[b] = k.total;
  if (k.heavy > 0) {
    if (k.old <= min(list_at, KV8_SEL_KEYS)) kv8_select_heavy<true>(k, w, sm, keys, keys + list_at, kept, nw);
    else kv8_select_heavy<false>(k, w, sm, keys, keys + list_at, kept, nw);
  }
  for (long long j = k.heavy + tid; j < out_cap; j += KV8_SEL_THREADS) {
    const bool live = j < k.total;
    const int pos = k.old + static_cast<int>(j - k.heavy);
    kept[j] = live ? pos : -1;
    nw[j] = live ? __ldg(w + pos) : 0.f;
  }
}

// One block per (new page, head, sequence): gathers the kept rows of K and V
// into registers, takes the new scales from their values and rounds them once.
// kept lists the rows, -1 behind the last. Eight lanes take 16 bytes each of a
// row, so that a warp's load spans four rows and a thread holds all its loads of
// K and V in flight at once; half as many threads with twice the bytes each
// measured 16 us less at 8 sequences x 8 heads of 32k tokens than 16 lanes of 8.
// Bound by memory: 50 us there, 264 MB, 5.3 TB/s, with nine blocks an SM (six
// took 54, ten and twelve 51 to 55; K and V in blocks of their own 53 to 57).
template <int PAGE>
__global__ void __launch_bounds__(kv8_page_threads(PAGE), PAGE == 128 ? 3 : 9) kv8_gather_kernel(const Kv8EvictParams p) {
  pdl_wait();
  // Eight lanes hold a row, 16 codes each.
  constexpr int THREADS = kv8_page_threads(PAGE), ROWS = THREADS / 8, PASSES = PAGE / ROWS;
  __shared__ float red[2][THREADS / 32];
  const int h = blockIdx.y, b = blockIdx.z;
  const int c16 = threadIdx.x & 7, r0 = threadIdx.x >> 3;
  const int* kept = p.kept + ((static_cast<long long>(b) * p.c.heads + h) * p.new_width + blockIdx.x) * PAGE;
  int pos[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) pos[i] = kept[r0 + ROWS * i];
  const int dst = __ldg(p.new_table + static_cast<long long>(b) * p.new_width + blockIdx.x);
  if (__syncthreads_and(pos[0] < 0)) return;   // the page receives nothing (row 0 is kept first)
  if (dst < 0 || dst >= p.c.pages) {
    if (threadIdx.x == 0) record_error(KV8_DEV_ERROR);
    return;
  }
  const int* table = p.s.table + static_cast<long long>(b) * p.s.width;
  uint4 raw[2][PASSES];
  float sc[2][PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    raw[0][i] = raw[1][i] = make_uint4(0, 0, 0, 0);
    sc[0][i] = sc[1][i] = 0.f;
    if (pos[i] >= 0) {
      const int pid = __ldg(table + pos[i] / PAGE);
      if (pid >= 0 && pid < p.c.pages) {
        const int blk = pid * p.c.heads + h;      // rows of codes are below 2^31
        const long long at = (static_cast<long long>(blk) * PAGE + pos[i] % PAGE) * 128 + c16 * 16;
        raw[0][i] = *reinterpret_cast<const uint4*>(p.c.k8 + at);
        raw[1][i] = *reinterpret_cast<const uint4*>(p.c.v8 + at);
        sc[0][i] = p.c.k_scale[blk];
        sc[1][i] = p.c.v_scale[blk];
      } else {
        record_error(KV8_DEV_ERROR);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      __half2 m = __floats2half2_rn(0.f, 0.f);     // codes are exact in f16; NaN loses
      const uint32_t w[4] = {raw[x][i].x, raw[x][i].y, raw[x][i].z, raw[x][i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t lo = e4m3x2_to_f16x2(w[k]), hi = e4m3x2_hi_to_f16x2(w[k]);
        m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&lo)));
        m = __hmax2(m, __habs2(*reinterpret_cast<const __half2*>(&hi)));
      }
      const float2 v = __half22float2(m);
      amax = fmaxf(amax, fmaxf(v.x, v.y) * sc[x][i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((threadIdx.x & 31) == 0) red[x][threadIdx.x >> 5] = amax;
  }
  __syncthreads();
  const int blk = dst * p.c.heads + h;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    float m = red[x][0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, red[x][i]);
    const float s = pow2f_exact(kv8_scale_exp(m)), inv = 1.f / s;
    uint8_t* to = (x ? p.c.v8 : p.c.k8) + static_cast<long long>(blk) * (PAGE * 128) + c16 * 16;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
      if (pos[i] < 0) continue;
      // inv is a power of two, so the factor is exact (a block of zeros may meet a huge old scale).
      const float factor = fminf(sc[x][i] * inv, 3.402823466e38f);
      uint2 part[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float f[8];
        e4m3x8_to_float(k ? make_uint2(raw[x][i].z, raw[x][i].w) : make_uint2(raw[x][i].x, raw[x][i].y), f);
#pragma unroll
        for (int q = 0; q < 8; ++q) f[q] *= factor;
        part[k] = pack_e4m3x8(f);
      }
      *reinterpret_cast<uint4*>(to + (r0 + ROWS * i) * 128) = make_uint4(part[0].x, part[0].y, part[1].x, part[1].y);
    }
    if (threadIdx.x == 0) (x ? p.c.v_scale : p.c.k_scale)[blk] = s;
  }
}

}  // namespace wamb
