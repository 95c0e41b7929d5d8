// Argument checks and launches of the E4M3 cache operators.
#pragma once
#include "kv8_tc.cuh"

namespace wamb {

inline bool stride8(int64_t s) { return s % 8 == 0; }

inline int kv8_cache_check(const wamb_kv8_cache* c, Kv8Cache* out) {
  WAMB_REQUIRE(c->k8 && c->v8 && c->k_scale && c->v_scale, WAMB_ERR_ARG, "kv8: null cache pointer");
  WAMB_REQUIRE(aligned16(c->k8) && aligned16(c->v8), WAMB_ERR_ALIGN, "kv8: codes must be 16-byte aligned");
  WAMB_REQUIRE(c->page == 16 || c->page == 32 || c->page == 64 || c->page == 128, WAMB_ERR_SHAPE,
               "kv8: page %d (16, 32, 64 or 128 tokens)", c->page);
  WAMB_REQUIRE(c->pages > 0 && c->heads > 0 && c->heads <= 65535, WAMB_ERR_SHAPE, "kv8: pages %d, heads %d", c->pages,
               c->heads);
  // Rows of codes are addressed by a 32-bit coordinate.
  WAMB_REQUIRE(static_cast<int64_t>(c->pages) * c->heads * c->page <= INT32_MAX, WAMB_ERR_SHAPE,
               "kv8: %d pages x %d heads x %d tokens exceed 2^31 - 1 rows", c->pages, c->heads, c->page);
  out->k8 = static_cast<uint8_t*>(c->k8);
  out->v8 = static_cast<uint8_t*>(c->v8);
  out->k_scale = c->k_scale;
  out->v_scale = c->v_scale;
  out->pages = c->pages;
  out->heads = c->heads;
  out->page = c->page;
  out->page_log2 = c->page == 16 ? 4 : c->page == 32 ? 5 : c->page == 64 ? 6 : 7;
  return WAMB_OK;
}

inline int kv8_seqs_check(const wamb_kv8_seqs* s, int page, Kv8Seqs* out) {
  WAMB_REQUIRE(s->batch >= 0 && s->batch <= 32767 && s->tokens >= 0 && s->table_width > 0, WAMB_ERR_SHAPE,
               "kv8: batch %d (0..32767), tokens %d, table_width %d", s->batch, s->tokens, s->table_width);
  // Positions and their tiles' ends stay far from the 32-bit limit.
  WAMB_REQUIRE(static_cast<int64_t>(s->table_width) * page + s->tokens <= (1 << 30), WAMB_ERR_SHAPE,
               "kv8: %d pages of %d tokens and %d new tokens exceed 2^30 positions", s->table_width, page, s->tokens);
  WAMB_REQUIRE(s->batch == 0 || (s->table && s->lens), WAMB_ERR_ARG, "kv8: null table or lens");
  out->table = s->table;
  out->lens = s->lens;
  out->counts = s->counts;
  out->batch = s->batch;
  out->width = s->table_width;
  out->tokens = s->tokens;
  return WAMB_OK;
}

template <bool F32>
inline int kv8_write_launch(const Kv8WriteParams& p, dim3 grid, cudaStream_t s) {
  switch (p.c.page) {
    case 16: return launch_kernel(kv8_write_kernel<F32, 16>, grid, dim3(kv8_page_threads(16)), 0, s, p);
    case 32: return launch_kernel(kv8_write_kernel<F32, 32>, grid, dim3(kv8_page_threads(32)), 0, s, p);
    case 64: return launch_kernel(kv8_write_kernel<F32, 64>, grid, dim3(kv8_page_threads(64)), 0, s, p);
    default: return launch_kernel(kv8_write_kernel<F32, 128>, grid, dim3(kv8_page_threads(128)), 0, s, p);
  }
}

inline int kv8_write_impl(const wamb_kv8_write_args* a, cudaStream_t s) {
  WAMB_REQUIRE(a != nullptr, WAMB_ERR_ARG, "null args");
  Kv8WriteParams p{};
  int rc = kv8_cache_check(&a->cache, &p.c);
  if (rc) return rc;
  rc = kv8_seqs_check(&a->seqs, p.c.page, &p.s);
  if (rc) return rc;
  if (p.s.batch == 0 || p.s.tokens == 0) return WAMB_OK;
  WAMB_REQUIRE(a->x_is_f32 == 0 || a->x_is_f32 == 1, WAMB_ERR_ARG, "x_is_f32 must be 0 or 1");
  WAMB_REQUIRE(a->k && a->v, WAMB_ERR_ARG, "kv8 write: null K or V");
  WAMB_REQUIRE(aligned16(a->k) && aligned16(a->v), WAMB_ERR_ALIGN, "kv8 write: K and V must be 16-byte aligned");
  p.x[0] = a->k;
  p.x[1] = a->v;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? a->v_stride : a->k_stride;
    WAMB_REQUIRE(stride8(st[0]) && stride8(st[1]) && stride8(st[2]), WAMB_ERR_ALIGN,
                 "kv8 write: strides must be multiples of 8 elements");
    p.sb[i] = st[0];
    p.st[i] = st[1];
    p.sh[i] = st[2];
  }
  DeviceInfo di;
  rc = device_info(&di);
  if (rc) return rc;
  const int touched = (p.s.tokens + p.c.page - 2) / p.c.page + 1;   // pages that `tokens` rows can meet
  const dim3 grid(touched, p.c.heads, 2 * p.s.batch);
  return a->x_is_f32 ? kv8_write_launch<true>(p, grid, s) : kv8_write_launch<false>(p, grid, s);
}

template <typename K>
inline int kv8_smem_once(K kern, int bytes, bool* done) {
  int dev = 0;
  WAMB_CHECK_CUDA(cudaGetDevice(&dev));
  if (!done[dev]) {
    WAMB_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done[dev] = true;
  }
  return WAMB_OK;
}

inline int kv8_evict_impl(const wamb_kv8_evict_args* a, cudaStream_t s) {
  WAMB_REQUIRE(a != nullptr, WAMB_ERR_ARG, "null args");
  Kv8EvictParams p{};
  int rc = kv8_cache_check(&a->cache, &p.c);
  if (rc) return rc;
  rc = kv8_seqs_check(&a->seqs, p.c.page, &p.s);
  if (rc) return rc;
  p.s.counts = nullptr;
  WAMB_REQUIRE(a->heavy >= 0 && a->recent >= 0, WAMB_ERR_ARG, "kv8 evict: heavy %d, recent %d", a->heavy, a->recent);
  WAMB_REQUIRE(a->new_width > 0 && static_cast<int64_t>(a->new_width) * p.c.page <= (1 << 30), WAMB_ERR_SHAPE,
               "kv8 evict: new_width %d", a->new_width);
  const int64_t cap = static_cast<int64_t>(p.s.width) * p.c.page;
  const int64_t most = std::min<int64_t>(static_cast<int64_t>(a->heavy) + a->recent, a->max_len);
  WAMB_REQUIRE(a->max_len >= 0 && a->max_len <= cap, WAMB_ERR_SHAPE, "kv8 evict: max_len %lld", (long long)a->max_len);
  WAMB_REQUIRE(most <= static_cast<int64_t>(a->new_width) * p.c.page, WAMB_ERR_SHAPE,
               "kv8 evict: %lld kept tokens do not fit %d pages", (long long)most, a->new_width);
  if (p.s.batch == 0) return WAMB_OK;
  WAMB_REQUIRE(a->weights && a->new_table && a->kept && a->new_weights && a->new_lens, WAMB_ERR_ARG,
               "kv8 evict: null pointer");
  WAMB_REQUIRE(a->new_weights != a->weights, WAMB_ERR_ARG, "kv8 evict: new_weights must not be weights");
  WAMB_REQUIRE(a->weights_cap >= cap, WAMB_ERR_SHAPE, "kv8 evict: weights hold %lld of %lld positions",
               (long long)a->weights_cap, (long long)cap);
  DeviceInfo di;
  rc = device_info(&di);
  if (rc) return rc;
  p.weights = a->weights;
  p.cap = a->weights_cap;
  p.new_table = a->new_table;
  p.new_width = a->new_width;
  p.heavy = a->heavy;
  p.recent = a->recent;
  p.kept = a->kept;
  p.new_weights = a->new_weights;
  p.new_lens = a->new_lens;
  static bool done[64] = {};
  rc = kv8_smem_once(kv8_select_kernel, KV8_SEL_SMEM, done);
  if (rc) return rc;
  // Shared memory for the keys that the tables can hold, so that short heads leave room for more blocks.
  const int hold = static_cast<int>(std::min<int64_t>(cap, KV8_SEL_KEYS)), list = std::min(hold, KV8_SEL_LIST);
  rc = launch_kernel(kv8_select_kernel, dim3(p.c.heads, p.s.batch), dim3(KV8_SEL_THREADS),
                     static_cast<size_t>(hold + list) * 4, s, p, hold);
  if (rc) return rc;
  const dim3 grid(p.new_width, p.c.heads, p.s.batch);
  switch (p.c.page) {
    case 16: return launch_kernel(kv8_gather_kernel<16>, grid, dim3(kv8_page_threads(16)), 0, s, p);
    case 32: return launch_kernel(kv8_gather_kernel<32>, grid, dim3(kv8_page_threads(32)), 0, s, p);
    case 64: return launch_kernel(kv8_gather_kernel<64>, grid, dim3(kv8_page_threads(64)), 0, s, p);
    default: return launch_kernel(kv8_gather_kernel<128>, grid, dim3(kv8_page_threads(128)), 0, s, p);
  }
}

// Three CTAs of the few-row attention fit an SM, four of its weights', one of
// the tensor-core kernels.
inline int kv8_few_ctas(const DeviceInfo& di, bool weights = false) { return (weights ? 4 : 3) * di.sms; }

// A tile of 16 rows is one m16n8k16 operand; more rows go to the tcgen05
// kernel, which reads each key once for 256 of them. Two tiles of 16 measured
// slower: 17 rows over 16k keys 93 us against 85, 32 rows of 4 sequences 59
// against 48 (only short caches gain: 32 rows over 2000 keys 24 against 33).
inline bool kv8_is_few(int64_t rows) { return rows <= FEW_QR; }

// Query rows of a sequence and cached head.
inline int64_t kv8_rows(const wamb_kv8_attention_args* a) {
  return a->cache.heads > 0 ? static_cast<int64_t>(a->seqs.tokens) * (a->q_heads / a->cache.heads) : 0;
}
// The split queries of the tensor-core kernels: rows of 256 bytes, a factor
// and (weights) a log-sum-exp each.
struct Kv8SplitQ {
  int rows_pad = 0;
  long long total = 0;
  size_t bytes(bool weights) const { return static_cast<size_t>(total) * (256 + (weights ? 8 : 4)); }
};
inline Kv8SplitQ kv8_split_q(int64_t batch, int64_t heads, int64_t rows) {
  Kv8SplitQ q;
  q.rows_pad = static_cast<int>((rows + 127) / 128 * 128);
  q.total = batch * heads * q.rows_pad;
  return q;
}
// Joins and two partials for each CTA, then the split queries.
inline size_t kv8_part_bytes(bool few, const DeviceInfo& di) {
  const size_t floats = few ? kv8_few_ctas(di) * kv8_part_floats<FEW_QR>() : di.sms * kv8_part_floats<KTC_QR>();
  return (KV8_JOIN_BYTES + 2 * floats * sizeof(float) + 255) / 256 * 256;
}
inline size_t kv8_workspace(const wamb_kv8_attention_args* a, bool weights, const DeviceInfo& di) {
  const int64_t rows = kv8_rows(a);
  const bool few = kv8_is_few(rows);
  return (weights ? 0 : kv8_part_bytes(few, di)) +
         (few ? 0 : kv8_split_q(a->seqs.batch, a->cache.heads, rows).bytes(weights));
}
// Splits the queries into `at`; returns the map of its rows and the factors.
inline int kv8_split_launch(const Kv8AttnParams& p, const Kv8SplitQ& sq, uint8_t* at, bool weights, CUtensorMap* map,
                            float** factor, float** neg_lse2, cudaStream_t s) {
  WAMB_REQUIRE(sq.total <= INT32_MAX - 64, WAMB_ERR_SHAPE, "kv8: %lld query rows", sq.total);
  *factor = reinterpret_cast<float*>(at + sq.total * 256);
  *neg_lse2 = weights ? *factor + sq.total : nullptr;
  int rc = make_tmap_2d(map, at, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, sq.total, 256, 256, 128, 128);
  if (rc) return rc;
  return launch_kernel(kv8_split_q_kernel, dim3(static_cast<unsigned>((sq.total + 63) / 64)), dim3(256), 0, s, p,
                       sq.rows_pad, static_cast<int>(sq.total), at, *factor, *neg_lse2);
}

inline int kv8_attention_impl(const wamb_kv8_attention_args* a, bool weights, cudaStream_t s) {
  WAMB_REQUIRE(a != nullptr, WAMB_ERR_ARG, "null args");
  Kv8AttnParams p{};
  int rc = kv8_cache_check(&a->cache, &p.c);
  if (rc) return rc;
  rc = kv8_seqs_check(&a->seqs, p.c.page, &p.s);
  if (rc) return rc;
  WAMB_REQUIRE(a->q_heads > 0 && a->q_heads % p.c.heads == 0, WAMB_ERR_SHAPE,
               "kv8: %d query heads are no multiple of %d cached heads", a->q_heads, p.c.heads);
  WAMB_REQUIRE(a->causal == 0 || a->causal == 1, WAMB_ERR_ARG, "causal must be 0 or 1");
  WAMB_REQUIRE(a->scale > 0.f && std::isfinite(a->scale), WAMB_ERR_ARG, "kv8: scale must be positive and finite");
  p.group = a->q_heads / p.c.heads;
  WAMB_REQUIRE(static_cast<int64_t>(p.s.tokens) * p.group <= (1 << 29), WAMB_ERR_SHAPE, "kv8: %d x %d query rows",
               p.s.tokens, p.group);
  const int rows = p.s.tokens * p.group;
  const bool few = kv8_is_few(rows);
  p.qts = weights || few ? 1 : (rows + KTC_QR - 1) / KTC_QR;
  WAMB_REQUIRE(static_cast<int64_t>(p.s.batch) * std::max(1, p.qts) <= (1 << 30), WAMB_ERR_SHAPE, "kv8: too many query tiles");
  if (p.s.batch == 0 || (p.s.tokens == 0 && !weights)) return WAMB_OK;
  WAMB_REQUIRE(p.s.tokens == 0 || a->q, WAMB_ERR_ARG, "kv8: null q");
  WAMB_REQUIRE(aligned16(a->q), WAMB_ERR_ALIGN, "kv8: q must be 16-byte aligned");
  WAMB_REQUIRE(stride8(a->q_stride[0]) && stride8(a->q_stride[1]) && stride8(a->q_stride[2]), WAMB_ERR_ALIGN,
               "kv8: q strides must be multiples of 8 elements");
  p.q = static_cast<const __nv_bfloat16*>(a->q);
  p.q_sb = a->q_stride[0];
  p.q_st = a->q_stride[1];
  p.q_sh = a->q_stride[2];
  p.causal = a->causal;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  const int64_t cap = static_cast<int64_t>(p.s.width) * p.c.page;
  if (weights) {
    WAMB_REQUIRE(a->weights && (a->lse || p.s.tokens == 0), WAMB_ERR_ARG, "kv8 weights: null lse or weights");
    WAMB_REQUIRE(a->weights_cap >= cap, WAMB_ERR_SHAPE, "kv8 weights: %lld columns for %lld positions",
                 (long long)a->weights_cap, (long long)cap);
    p.lse_in = a->lse;
    p.base = a->base;
    p.weights = a->weights;
    p.w_cap = a->weights_cap;
  } else {
    WAMB_REQUIRE(a->out, WAMB_ERR_ARG, "kv8 attention: null out");
    WAMB_REQUIRE(aligned16(a->out), WAMB_ERR_ALIGN, "kv8 attention: out must be 16-byte aligned");
    WAMB_REQUIRE(stride8(a->out_stride[0]) && stride8(a->out_stride[1]) && stride8(a->out_stride[2]), WAMB_ERR_ALIGN,
                 "kv8 attention: out strides must be multiples of 8 elements");
    p.out = static_cast<__nv_bfloat16*>(a->out);
    p.o_sb = a->out_stride[0];
    p.o_st = a->out_stride[1];
    p.o_sh = a->out_stride[2];
    p.lse = a->lse;
  }
  DeviceInfo di;
  rc = device_info(&di);
  if (rc) return rc;
  WAMB_REQUIRE(kv8_few_ctas(di) <= static_cast<int>(KV8_JOIN_BYTES / sizeof(Kv8Join)), WAMB_ERR_DEVICE, "kv8: %d SMs",
               di.sms);
  const size_t need = kv8_workspace(a, weights, di);
  if (need > 0) {
    WAMB_REQUIRE(a->workspace && a->workspace_bytes >= need, WAMB_ERR_WORKSPACE, "kv8: workspace of %zu bytes, needs %zu",
                 a->workspace ? a->workspace_bytes : size_t{0}, need);
    WAMB_REQUIRE(reinterpret_cast<uintptr_t>(a->workspace) % 256 == 0, WAMB_ERR_ALIGN,
                 "kv8: workspace must be 256-byte aligned");
  }
  uint8_t* ws = static_cast<uint8_t*>(a->workspace);
  if (!weights) p.part = reinterpret_cast<float*>(ws + KV8_JOIN_BYTES);
  const uint64_t code_rows = static_cast<uint64_t>(p.c.pages) * p.c.heads * p.c.page;
  // Boxes of the TMA loads: the few-row kernel takes 16 keys, the other whole pages.
  const uint32_t box = few ? 16 : p.c.page;
  CUtensorMap tmK, tmV;
  rc = make_tmap_2d(&tmK, p.c.k8, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, code_rows, 128, 128, box, 128);
  if (rc) return rc;
  rc = make_tmap_2d(&tmV, p.c.v8, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, code_rows, 128, 128, box, 128);
  if (rc) return rc;
  p.ctas = kv8_few_ctas(di, weights);
  if (weights && few) {
    static bool done[64] = {};
    rc = kv8_smem_once(kv8_few_kernel<true>, FewSmem<true>::TOTAL, done);
    if (rc) return rc;
    return launch_kernel(kv8_few_kernel<true>, dim3(p.ctas), dim3(FEW_THREADS), FewSmem<true>::TOTAL, s, tmK, tmV, p);
  }
  if (few) {
    static bool done[64] = {};
    rc = kv8_smem_once(kv8_few_kernel<false>, FewSmem<false>::TOTAL, done);
    if (rc) return rc;
    rc = launch_kernel(kv8_few_kernel<false>, dim3(p.ctas), dim3(FEW_THREADS), FewSmem<false>::TOTAL, s, tmK, tmV, p);
    if (rc) return rc;
    if (cap <= FEW_TK) return WAMB_OK;   // one unit per item: nothing is ever shared
    return launch_kernel(kv8_merge_kernel<FEW_QR, 1>, dim3(p.ctas, rows), dim3(256), 0, s, p);
  }
  p.ctas = di.sms;
  CUtensorMap tmQ;
  float *factor = nullptr, *neg_lse2 = nullptr;
  const Kv8SplitQ sq = kv8_split_q(p.s.batch, p.c.heads, rows);
  rc = kv8_split_launch(p, sq, weights ? ws : ws + kv8_part_bytes(false, di), weights, &tmQ, &factor, &neg_lse2, s);
  if (rc) return rc;
  if (weights) {
    static bool done[64] = {};
    rc = kv8_smem_once(kv8_weights_tc_kernel, KwtSmem::TOTAL, done);
    if (rc) return rc;
    return launch_kernel(kv8_weights_tc_kernel, dim3(p.ctas), dim3(KWT_THREADS), KwtSmem::TOTAL, s, tmK, tmQ,
                         static_cast<const float*>(factor), static_cast<const float*>(neg_lse2), sq.rows_pad, p);
  }
  static bool done[64] = {};
  rc = kv8_smem_once(kv8_tc_kernel, KtcSmem::TOTAL, done);
  if (rc) return rc;
  rc = launch_kernel(kv8_tc_kernel, dim3(p.ctas), dim3(KTC_THREADS), KtcSmem::TOTAL, s, tmK, tmV, tmQ,
                     static_cast<const float*>(factor), sq.rows_pad, p);
  if (rc) return rc;
  if (cap <= KTC_TK) return WAMB_OK;
  return launch_kernel(kv8_merge_kernel<KTC_QR, 8>, dim3(p.ctas, (std::min(rows, KTC_QR) + 7) / 8), dim3(256), 0, s, p);
}

}  // namespace wamb
