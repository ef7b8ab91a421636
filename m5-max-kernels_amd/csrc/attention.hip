// C entries of attention over dense keys and values and over a paged cache (kernels: attention_core.h).
#include "attention_core.h"

namespace m5k {
namespace attn {
// Each in a translation unit of its own.
template <> int launch_typed<DENSE, false, NO_CODES>(Args&, int, int, hipStream_t);
template <> int launch_typed<DENSE, true, NO_CODES>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES16, false, NO_CODES>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES16, true, NO_CODES>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES, false, NO_CODES>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES, true, NO_CODES>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES16, false, E4M3>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES16, true, E4M3>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES16, false, INT8>(Args&, int, int, hipStream_t);
template <> int launch_typed<PAGES16, true, INT8>(Args&, int, int, hipStream_t);

template <int DT, int D>
static int launch_join_of(const Args& a, hipStream_t st) {
  const int64_t rows = int64_t{a.tokens} * a.heads;
  if (a.splits > JOINED_TOGETHER)
    launch_kernel(attention_join<DT, D, 4>, dim3(static_cast<uint32_t>(rows)), dim3(256), st, a);
  else
    launch_kernel(attention_join<DT, D, 1>, dim3(static_cast<uint32_t>((rows + 3) / 4)), dim3(256), st, a);
  return launch_status("attention join");
}

int launch_join(const Args& a, int dtype, int head_dim, hipStream_t st) {
  const bool bf16 = dtype == M5K_BF16;
  if (head_dim == 64) return bf16 ? launch_join_of<M5K_BF16, 64>(a, st) : launch_join_of<M5K_F16, 64>(a, st);
  return bf16 ? launch_join_of<M5K_BF16, 128>(a, st) : launch_join_of<M5K_F16, 128>(a, st);
}
}  // namespace attn
}  // namespace m5k

namespace {

using m5k::attn::Args;

// Fields that both entries share, checked.
int common(Args& a, const void* q, int dtype, int64_t tokens, int64_t heads, int64_t kv_heads, int head_dim,
           int64_t q_head, int64_t q_token, float scale, int64_t window, int64_t sinks, float softcap,
           const float* slopes, const int32_t* prefix, void* out, int splits, float* workspace,
           int64_t workspace_elems) {
  M5K_REQUIRE(q && out, "attention: null pointer");
  M5K_REQUIRE(dtype == M5K_BF16 || dtype == M5K_F16, "attention: dtype must be bf16 or f16");
  M5K_REQUIRE(head_dim == 64 || head_dim == 128, "attention: head_dim must be 64 or 128");
  M5K_REQUIRE(tokens > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
              "attention: heads must be a positive multiple of kv_heads, tokens positive");
  M5K_REQUIRE(tokens <= (1 << 24) && heads <= (1 << 16) && tokens * heads < (int64_t{1} << 30),
              "attention: too many tokens");
  M5K_REQUIRE(q_head % 8 == 0 && q_token % 8 == 0 && m5k::aligned16(q) && m5k::aligned16(out),
              "attention: q and out rows must be 16-byte aligned");
  M5K_REQUIRE(scale >= 0x1p-126f && scale < 1e30f && softcap >= 0.0f && softcap < 1e30f,
              "attention: scale must be positive, softcap nonnegative, both finite");
  // A subnormal cap and an infinite quotient turn scores of 0 into NaN.
  M5K_REQUIRE(softcap == 0.0f || (softcap >= 0x1p-126f && scale / softcap <= 1.0001e37f),
              "attention: softcap must be 0 or a normal number, scale / softcap at most 1e37");
  M5K_REQUIRE(window >= 0 && window < (1 << 30), "attention: bad window");
  M5K_REQUIRE(!(window && prefix), "attention: a window and a prefix cannot be combined");
  M5K_REQUIRE(sinks >= 0 && sinks < (1 << 30) && (!sinks || window), "attention: sinks need a window");
  M5K_REQUIRE(splits >= 1 && splits <= 64, "attention: splits must be in [1, 64]");
  M5K_REQUIRE(splits == 1 || (workspace && m5k::aligned16(workspace) &&
                              workspace_elems >= splits * tokens * heads * (int64_t{head_dim} + 2)),
              "attention: the workspace must hold splits * tokens * heads * (head_dim + 2) floats, 16-byte aligned");
  a.q = static_cast<const uint16_t*>(q);
  a.out = static_cast<uint16_t*>(out);
  a.q_head = q_head;
  a.q_token = q_token;
  a.slopes = slopes;
  a.prefix = prefix;
  a.tokens = static_cast<int>(tokens);
  a.heads = static_cast<int>(heads);
  a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(heads / kv_heads);
  a.window = static_cast<int>(window);
  a.sinks = static_cast<int>(sinks);
  a.scale = scale;
  a.softcap = softcap;
  a.splits = splits;
  a.part_o = workspace;
  a.part_ml = workspace ? workspace + splits * tokens * heads * head_dim : nullptr;
  m5k::magic_of(static_cast<uint32_t>(a.group), a.group_magic, a.group_shift);
  return M5K_OK;
}

// Keys that the plan counts a row to see: with first keys, no more than those, the window and a tile.
int64_t reach(int64_t keys, int64_t window, int64_t sinks, bool causal) {
  const int64_t seen = (causal ? 1 : 2) * window + sinks + 64;
  return sinks && seen < keys ? seen : keys;
}

}  // namespace

extern "C" int m5k_attention_plan(int paged, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t sequences,
                                  int64_t keys, int cus, int* splits, int* few) {
  m5k::clear_error();
  M5K_REQUIRE(paged == 0 || paged == 1 || (paged > 1 && paged < 32 && ((paged & 7) == 2 || (paged & 7) == 4)),
              "attention_plan: bad paged");
  M5K_REQUIRE(splits && tokens > 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && sequences >= 0 && keys >= 0,
              "attention_plan: bad sizes");
  if (cus <= 0) cus = m5k::device_cus();
  if (cus <= 0) cus = 256;
  const int group = static_cast<int>(heads / kv_heads), kvh = static_cast<int>(kv_heads);
  *splits = m5k::attn::plan_splits(paged, tokens, group, kvh, sequences, keys, cus);
  if (few) *few = m5k::attn::plan(paged, tokens, group, kvh, sequences, keys, cus).few;
  return M5K_OK;
}

extern "C" int m5k_attention_sinks(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim,
                                   int64_t q_head, int64_t q_token, const void* k, int64_t k_head, int64_t k_key,
                                   const void* v, int64_t v_head, int64_t v_key, int64_t keys, int64_t kv_heads,
                                   float scale, int causal, int64_t window, int64_t sinks, float softcap,
                                   const float* slopes, const int32_t* document_starts, int64_t documents,
                                   const int32_t* prefix_lengths, void* out, int splits, float* workspace,
                                   int64_t workspace_elems, void* stream) {
  m5k::clear_error();
  Args a = {};
  if (int rc = common(a, q, dtype, tokens, heads, kv_heads, head_dim, q_head, q_token, scale, window, sinks, softcap,
                      slopes, prefix_lengths, out, splits, workspace, workspace_elems))
    return rc;
  M5K_REQUIRE(keys >= 0 && keys <= (1 << 24) && (keys == 0 || (k && v)), "attention: bad keys");
  M5K_REQUIRE(m5k::aligned16(k) && m5k::aligned16(v) && k_head % 8 == 0 && k_key % 8 == 0 && v_head % 8 == 0 &&
                  v_key % 8 == 0,
              "attention: k and v rows must be 16-byte aligned");
  constexpr int64_t kRowMax = 1 << 23;
  M5K_REQUIRE(keys <= 1 || (k_key >= head_dim && v_key >= head_dim && k_key <= kRowMax && v_key <= kRowMax),
              "attention: rows of k and v must be head_dim to 2^23 elements apart");
  M5K_REQUIRE(!document_starts || (documents > 0 && documents <= (1 << 24) && tokens == keys),
              "attention: documents need as many keys as tokens");
  M5K_REQUIRE(!prefix_lengths || causal, "attention: a prefix needs a causal mask");
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.k_head = k_head;
  a.k_row = keys == 1 ? head_dim : k_key;
  a.v_head = v_head;
  a.v_row = keys == 1 ? head_dim : v_key;
  a.keys = static_cast<int>(keys);
  a.causal = causal != 0;
  a.starts = document_starts;
  a.sequences = static_cast<int>(documents);
  a.reach = reach(keys, window, sinks, causal != 0);
  const auto run = sinks ? m5k::attn::launch_typed<m5k::attn::DENSE, true, m5k::attn::NO_CODES>
                         : m5k::attn::launch_typed<m5k::attn::DENSE, false, m5k::attn::NO_CODES>;
  return run(a, dtype, head_dim, m5k::as_stream(stream));
}

extern "C" int m5k_attention(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head,
                             int64_t q_token, const void* k, int64_t k_head, int64_t k_key, const void* v,
                             int64_t v_head, int64_t v_key, int64_t keys, int64_t kv_heads, float scale, int causal,
                             int64_t window, float softcap, const float* slopes, const int32_t* document_starts,
                             int64_t documents, const int32_t* prefix_lengths, void* out, int splits,
                             float* workspace, int64_t workspace_elems, void* stream) {
  return m5k_attention_sinks(q, dtype, tokens, heads, head_dim, q_head, q_token, k, k_head, k_key, v, v_head, v_key,
                             keys, kv_heads, scale, causal, window, 0, softcap, slopes, document_starts, documents,
                             prefix_lengths, out, splits, workspace, workspace_elems, stream);
}

namespace {

// Fields of the paged entries, checked; `unit` elements of a cache row lie in 16 bytes.
int paged(Args& a, const void* k_cache, int64_t k_page, int64_t k_head, int64_t k_slot, const void* v_cache,
          int64_t v_page, int64_t v_head, int64_t v_slot, int unit, int64_t pages, int64_t page_size,
          const int32_t* page_table, int64_t table_width, int64_t sequences, const int32_t* query_starts,
          const int32_t* context_lengths) {
  M5K_REQUIRE(k_cache && v_cache && page_table && query_starts && context_lengths, "paged_attention: null pointer");
  M5K_REQUIRE(pages > 0 && pages <= INT32_MAX && page_size > 0 && page_size <= (1 << 20) && table_width > 0 &&
                  table_width * page_size <= (1 << 30),
              "paged_attention: a sequence may have up to 2^30 keys in pages of up to 2^20");
  M5K_REQUIRE(sequences > 0 && sequences <= (1 << 24), "paged_attention: bad number of sequences");
  M5K_REQUIRE(m5k::aligned16(k_cache) && m5k::aligned16(v_cache) && k_page % unit == 0 && k_head % unit == 0 &&
                  k_slot % unit == 0 && v_page % unit == 0 && v_head % unit == 0 && v_slot % unit == 0,
              "paged_attention: cache rows must be 16-byte aligned");
  a.k = static_cast<const uint16_t*>(k_cache);
  a.v = static_cast<const uint16_t*>(v_cache);
  a.k_page = k_page;
  a.k_head = k_head;
  a.k_row = k_slot;
  a.v_page = v_page;
  a.v_head = v_head;
  a.v_row = v_slot;
  a.pages = static_cast<int>(pages);
  a.page_size = static_cast<int>(page_size);
  a.table = page_table;
  a.table_width = table_width;
  a.starts = query_starts;
  a.context = context_lengths;
  a.sequences = static_cast<int>(sequences);
  a.keys = static_cast<int>(table_width * page_size);
  a.reach = reach(a.keys, a.window, a.sinks, true);
  a.causal = 1;
  m5k::magic_of(static_cast<uint32_t>(page_size), a.page_magic, a.page_shift);
  return M5K_OK;
}

}  // namespace

extern "C" int m5k_paged_attention_sinks(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim,
                                         int64_t q_head, int64_t q_token, const void* k_cache, int64_t k_page,
                                         int64_t k_head, int64_t k_slot, const void* v_cache, int64_t v_page,
                                         int64_t v_head, int64_t v_slot, int64_t pages, int64_t page_size,
                                         int64_t kv_heads, const int32_t* page_table, int64_t table_width,
                                         int64_t sequences, const int32_t* query_starts,
                                         const int32_t* context_lengths, float scale, int64_t window, int64_t sinks,
                                         float softcap, const float* slopes, const int32_t* prefix_lengths, void* out,
                                         int splits, float* workspace, int64_t workspace_elems, void* stream) {
  m5k::clear_error();
  Args a = {};
  if (int rc = common(a, q, dtype, tokens, heads, kv_heads, head_dim, q_head, q_token, scale, window, sinks, softcap,
                      slopes, prefix_lengths, out, splits, workspace, workspace_elems))
    return rc;
  if (int rc = paged(a, k_cache, k_page, k_head, k_slot, v_cache, v_page, v_head, v_slot, 8, pages, page_size,
                     page_table, table_width, sequences, query_starts, context_lengths))
    return rc;
  using namespace m5k::attn;
  const bool whole = page_size % 16 == 0 && k_slot >= head_dim && v_slot >= head_dim && k_slot <= (1 << 23) &&
                     v_slot <= (1 << 23);
  const auto run = whole ? (sinks ? launch_typed<PAGES16, true, NO_CODES> : launch_typed<PAGES16, false, NO_CODES>)
                         : (sinks ? launch_typed<PAGES, true, NO_CODES> : launch_typed<PAGES, false, NO_CODES>);
  return run(a, dtype, head_dim, m5k::as_stream(stream));
}

extern "C" int m5k_paged_attention(const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim,
                                   int64_t q_head, int64_t q_token, const void* k_cache, int64_t k_page,
                                   int64_t k_head, int64_t k_slot, const void* v_cache, int64_t v_page, int64_t v_head,
                                   int64_t v_slot, int64_t pages, int64_t page_size, int64_t kv_heads,
                                   const int32_t* page_table, int64_t table_width, int64_t sequences,
                                   const int32_t* query_starts, const int32_t* context_lengths, float scale,
                                   int64_t window, float softcap, const float* slopes, const int32_t* prefix_lengths,
                                   void* out, int splits, float* workspace, int64_t workspace_elems, void* stream) {
  return m5k_paged_attention_sinks(q, dtype, tokens, heads, head_dim, q_head, q_token, k_cache, k_page, k_head, k_slot,
                                   v_cache, v_page, v_head, v_slot, pages, page_size, kv_heads, page_table, table_width,
                                   sequences, query_starts, context_lengths, scale, window, 0, softcap, slopes,
                                   prefix_lengths, out, splits, workspace, workspace_elems, stream);
}

extern "C" int m5k_paged_attention_codes(
    const void* q, int dtype, int64_t tokens, int64_t heads, int head_dim, int64_t q_head, int64_t q_token, int mode,
    const void* k_codes, int64_t k_page, int64_t k_head, int64_t k_slot, const uint8_t* k_exponents, int64_t ke_page,
    int64_t ke_head, const void* v_codes, int64_t v_page, int64_t v_head, int64_t v_slot, const uint8_t* v_exponents,
    int64_t ve_page, int64_t ve_head, int64_t block, int64_t pages, int64_t page_size, int64_t kv_heads,
    const int32_t* page_table, int64_t table_width, int64_t sequences, const int32_t* query_starts,
    const int32_t* context_lengths, float scale, int64_t window, int64_t sinks, float softcap, const float* slopes,
    const int32_t* prefix_lengths, void* out, int splits, float* workspace, int64_t workspace_elems, void* stream) {
  m5k::clear_error();
  Args a = {};
  if (int rc = common(a, q, dtype, tokens, heads, kv_heads, head_dim, q_head, q_token, scale, window, sinks, softcap,
                      slopes, prefix_lengths, out, splits, workspace, workspace_elems))
    return rc;
  if (int rc = paged(a, k_codes, k_page, k_head, k_slot, v_codes, v_page, v_head, v_slot, 16, pages, page_size,
                     page_table, table_width, sequences, query_starts, context_lengths))
    return rc;
  M5K_REQUIRE(mode == M5K_QUANT_FP8 || mode == M5K_QUANT_INT8, "paged_attention: codes must be FP8 or INT8");
  M5K_REQUIRE(k_exponents && v_exponents, "paged_attention: null exponents");
  M5K_REQUIRE(block > 0 && block % 16 == 0 && page_size % block == 0,
              "paged_attention: a block must be a multiple of 16 tokens and divide the page");
  constexpr int64_t kRowMax = 1 << 23;
  M5K_REQUIRE(k_slot >= head_dim && v_slot >= head_dim && k_slot <= kRowMax && v_slot <= kRowMax,
              "paged_attention: rows of codes must be head_dim to 2^23 bytes apart");
  a.k_exp = k_exponents;
  a.v_exp = v_exponents;
  a.ke_page = ke_page;
  a.ke_head = ke_head;
  a.ve_page = ve_page;
  a.ve_head = ve_head;
  m5k::magic_of(static_cast<uint32_t>(block), a.block_magic, a.block_shift);
  using namespace m5k::attn;
  const auto run = mode == M5K_QUANT_FP8
                       ? (sinks ? launch_typed<PAGES16, true, E4M3> : launch_typed<PAGES16, false, E4M3>)
                       : (sinks ? launch_typed<PAGES16, true, INT8> : launch_typed<PAGES16, false, INT8>);
  return run(a, dtype, head_dim, m5k::as_stream(stream));
}
