// Attention of the new tokens of a ragged batch over a paged KV cache: how a
// call is cut, the C entries, and the bfloat16 kernels (varlen_kernels.h).
#include "varlen_kernels.h"

namespace dk {
namespace varlen {

template hipError_t launch<Bf16>(const KParams&, const Plan&, int, bool, hipStream_t);

Plan make_plan(const dk_varlen_attn_params* a, int d, int max_query_len, int max_len, int window) {
  Plan plan;
  const int group = a->num_q_heads / a->num_kv_heads;
  const int64_t hkv = a->num_kv_heads, rows = static_cast<int64_t>(a->num_tokens) * group;
  const int64_t most_rows = static_cast<int64_t>(std::min(max_query_len, a->num_tokens)) * group;
  // Keys that a token may see, as far as the host knows.
  const int64_t keys = a->prefix_lens != nullptr ? max_len : std::min<int64_t>(max_len, static_cast<int64_t>(window) + std::max(max_query_len, 32));
  // 32 rows where that takes in every sequence (speculation: 48 of up to 4 tokens,
  // 28 / 4 heads, 62.9 us, and 87.7 as row tiles past 16 rows); beside prompts the others
  // mostly bring one token.
  plan.short_rows = most_rows > 16 && most_rows <= 32 && d <= kWideRows ? 32 : 16;
  if (most_rows > plan.short_rows) {
    // At most this many row tiles: full ones, and one more a sequence, of at least 17 rows each.
    const int64_t tiles = rows / tile_rows(d) + std::min<int64_t>(a->num_seqs, rows / (plan.short_rows + 1));
    plan.tile_groups = tiles * hkv;
    // Few tiles for the 256 CUs: spread (how far, the GPU decides from the lengths;
    // a 512-token chunk on 16000 keys, 128 tiles: 178 us, 400 whole).
    constexpr int most = 512;
    if (rows / tile_rows(d) * hkv < most / 2 && keys > kMinPart * (d <= 128 ? tile_keys<128>() : tile_keys<256>())) {
      plan.split_items = most;
      plan.joins = std::min<int64_t>(plan.tile_groups, most / 2);
      plan.tile_groups = std::max<int64_t>(plan.tile_groups, most);
      plan.tile_ws = static_cast<int64_t>(most) * tile_rows(d);
    }
  }
  plan.row_groups = a->num_seqs * hkv;
  const bool many = a->num_seqs * hkv >= kManyPairs;
  if (keys > (many ? kWholeKeysMany : kWholeKeys)) {
    const int64_t resident = d <= 64 ? 768 : d <= 128 ? 512 : 256;  // workgroups of row_work on 256 CUs
    plan.shares = static_cast<int>(std::max<int64_t>(resident / hkv, 1));
    plan.row_groups = plan.shares * hkv;
    plan.slot_rows = static_cast<int>(std::min<int64_t>(most_rows, plan.short_rows));
    plan.slots = (plan.shares + static_cast<int64_t>(a->num_seqs)) * hkv;
  }
  // One workspace: the tiles' sums and their maxima, then the rows', in floats.
  if (plan.tile_ws > 0 || plan.slots > 0) {
    plan.tile_ml_at = plan.tile_ws * d;
    plan.row_at = plan.tile_ml_at + plan.tile_ws * 2;
    plan.ml_at = plan.row_at + plan.slots * plan.slot_rows * d;
    plan.first_at = plan.ml_at + plan.slots * plan.slot_rows * 2;
    plan.ws_bytes = 4 * (plan.first_at + (plan.slots > 0 ? 2 * a->num_seqs * hkv : 0));
  }
  return plan;
}

// The plan without a workspace: nothing is cut.
Plan whole_plan(const dk_varlen_attn_params* a, int d, const Plan& with) {
  Plan plan;
  plan.tile_groups = with.tile_groups;
  if (with.split_items > 0) {
    const int64_t group = a->num_q_heads / a->num_kv_heads, rows = a->num_tokens * group;
    plan.tile_groups = (rows / tile_rows(d) + std::min<int64_t>(a->num_seqs, rows / (with.short_rows + 1))) * a->num_kv_heads;
  }
  plan.short_rows = with.short_rows;
  plan.row_groups = static_cast<int64_t>(a->num_seqs) * a->num_kv_heads;
  return plan;
}

// No length goes past the caller's bound and what the block tables hold.
int length_bound(const dk_varlen_attn_params* a, int max_seq_len) {
  const int64_t held = static_cast<int64_t>(a->max_blocks) * a->block_size;
  return a->num_blocks == 0 ? 0 : static_cast<int>(std::min<int64_t>(held, max_seq_len));
}

int window_bound(const dk_varlen_attn_params* a, int max_len) {
  return a->window == 0 || a->window > max_len ? std::max(max_len, 1) : a->window;
}

int run(const char* op, const dk_varlen_attn_params* a, int dtype, int head_dim, int max_query_len, int max_seq_len,
        bool fp8, float k_scale, float v_scale, void* workspace, int64_t workspace_bytes, void* stream) {
  clear_error();
  if (a == nullptr) return fail("%s: params must not be NULL", op);
  if (dtype != DK_FLOAT16 && dtype != DK_BFLOAT16) return fail("%s: expected float16 or bfloat16, got dtype code %d", op, dtype);
  const bool dim_ok = head_dim == 64 || head_dim == 128 || head_dim == 192 || head_dim == 256 || (head_dim == 96 && !fp8);
  if (!dim_ok) return fail("%s: head_dim must be 64, 96 (not with an fp8 cache), 128, 192 or 256, got %d", op, head_dim);
  if (a->num_tokens < 0 || a->num_seqs < 0 || a->num_blocks < 0 || a->max_blocks < 0 || max_query_len < 0 || max_seq_len < 0)
    return fail("%s: sizes must be non-negative", op);
  if (a->num_kv_heads <= 0 || a->num_q_heads <= 0 || a->num_q_heads % a->num_kv_heads != 0)
    return fail("%s: num_q_heads must be a multiple of num_kv_heads", op);
  if (a->num_q_heads / a->num_kv_heads > DK_MAX_GQA_GROUP)
    return fail("%s: GQA group size above %d is not supported", op, DK_MAX_GQA_GROUP);
  if (a->block_size <= 0) return fail("%s: block_size must be positive", op);
  if (a->window < 0) return fail("%s: window must be non-negative (0: none)", op);
  if (!(a->softcap >= 0.0f && a->softcap < INFINITY)) return fail("%s: softcap must be non-negative and finite (0: none)", op);
  if (!(std::fabs(a->scale) < INFINITY)) return fail("%s: scale must be finite", op);
  if (fp8 && !(k_scale > 0.0f && v_scale > 0.0f && k_scale < INFINITY && v_scale < INFINITY))
    return fail("%s: k_scale and v_scale must be positive and finite", op);
  if (static_cast<int64_t>(a->num_tokens) * a->num_q_heads > 0x7fffffff || a->num_seqs > (1 << 30))
    return fail("%s: too many tokens x heads or sequences", op);
  if (a->num_tokens == 0 || a->num_seqs == 0) return hipSuccess;
  if (a->out == nullptr || a->q == nullptr || a->seq_lens == nullptr || a->query_start_loc == nullptr)
    return fail("%s: out, q, seq_lens and query_start_loc must not be NULL", op);
  const int max_len = length_bound(a, max_seq_len);
  if (max_len > 0 && (a->k_cache == nullptr || a->v_cache == nullptr || a->block_tables == nullptr))
    return fail("%s: k_cache, v_cache and block_tables must not be NULL", op);
  for (const int64_t stride :
       {a->q_stride_token, a->q_stride_head, a->out_stride_token, a->out_stride_head, a->k_stride_block, a->k_stride_token,
        a->k_stride_head, a->v_stride_block, a->v_stride_token, a->v_stride_head, a->bt_stride}) {
    if (stride < 0 || stride > 0x7fffffff) return fail("%s: strides must be non-negative and below 2^31", op);
  }
  const int elt = fp8 ? 1 : 2;
  const bool rows16 = aligned_to(a->k_cache, 16) && aligned_to(a->v_cache, 16) && a->k_stride_block * elt % 16 == 0 &&
                      a->k_stride_token * elt % 16 == 0 && a->k_stride_head * elt % 16 == 0 &&
                      a->v_stride_block * elt % 16 == 0 && a->v_stride_token * elt % 16 == 0 &&
                      a->v_stride_head * elt % 16 == 0;
  if (!rows16) return fail("%s: KV-cache pointers and strides must be multiples of 16 bytes", op);
  KParams kp{};
  kp.out = static_cast<uint16_t*>(a->out);
  kp.q = static_cast<const uint16_t*>(a->q);
  kp.k = a->k_cache;
  kp.v = a->v_cache;
  kp.tables = a->block_tables;
  kp.lens = a->seq_lens;
  kp.starts = a->query_start_loc;
  kp.prefix = a->prefix_lens;
  kp.slopes = a->alibi_slopes;
  kp.biased = a->alibi_slopes != nullptr;
  kp.q_st = static_cast<int32_t>(a->q_stride_token);
  kp.q_sh = static_cast<int32_t>(a->q_stride_head);
  kp.o_st = static_cast<int32_t>(a->out_stride_token);
  kp.o_sh = static_cast<int32_t>(a->out_stride_head);
  kp.k_sb = static_cast<int32_t>(a->k_stride_block);
  kp.k_st = static_cast<int32_t>(a->k_stride_token);
  kp.k_sh = static_cast<int32_t>(a->k_stride_head);
  kp.v_sb = static_cast<int32_t>(a->v_stride_block);
  kp.v_st = static_cast<int32_t>(a->v_stride_token);
  kp.v_sh = static_cast<int32_t>(a->v_stride_head);
  kp.bt_stride = static_cast<int32_t>(a->bt_stride);
  kp.num_tokens = a->num_tokens;
  kp.num_seqs = a->num_seqs;
  kp.hq = a->num_q_heads;
  kp.group = a->num_q_heads / a->num_kv_heads;
  kp.block_size = a->block_size;
  kp.num_blocks = a->num_blocks;
  kp.max_len = max_len;
  kp.window = window_bound(a, max_len);
  kp.v_scale = v_scale;
  kp.hkv = a->num_kv_heads;
  Plan plan = make_plan(a, head_dim, max_query_len, max_len, kp.window);
  if (plan.ws_bytes > 0 && (workspace == nullptr || workspace_bytes < plan.ws_bytes)) plan = whole_plan(a, head_dim, plan);
  if (plan.ws_bytes > 0 && !aligned_to(workspace, 16)) return fail("%s: workspace must be 16-byte aligned", op);
  if (plan.tile_groups + plan.row_groups > 0x7fffffff || static_cast<int64_t>(a->num_seqs) * a->num_kv_heads > 0x7fffffff)
    return fail("%s: too many sequences x heads", op);
  kp.tile_groups = static_cast<int>(plan.tile_groups);
  kp.shares = plan.shares;
  kp.short_rows = plan.short_rows;
  kp.slot_rows = plan.slot_rows;
  kp.split_items = plan.split_items;
  float* ws = static_cast<float*>(workspace);
  kp.tile_ws = ws;
  kp.tile_ml = ws + plan.tile_ml_at;
  kp.ws = ws + plan.row_at;
  kp.ws_ml = ws + plan.ml_at;
  kp.ws_first = reinterpret_cast<int32_t*>(ws + plan.first_at);
  // floor(j / b) = (j * ceil(2^k / b)) >> k for j < 2^31 with k = 31 + ceil(log2 b):
  // the factor is off by less than 1, the product by less than 2^31 <= 2^k / b.
  int k = 31;
  while ((int64_t{1} << (k - 31)) < a->block_size) ++k;
  kp.bs_shift = k;
  kp.bs_mul = static_cast<uint32_t>(((uint64_t{1} << k) + a->block_size - 1) / a->block_size);
  const float c = a->scale * k_scale;
  kp.q_sign = c < 0.0f ? 0x80008000u : 0u;
  kp.cap2 = a->softcap * kLog2e;
  kp.scale2 = std::fabs(c) * kLog2e * (a->softcap > 0.0f ? 2.0f / a->softcap : 1.0f);
  if (!(kp.scale2 < INFINITY)) return fail("%s: scale / softcap is past fp32's range", op);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return static_cast<int>(dtype == DK_BFLOAT16 ? launch<Bf16>(kp, plan, head_dim, fp8, s)
                                               : launch<F16>(kp, plan, head_dim, fp8, s));
}

}  // namespace varlen
}  // namespace dk

extern "C" int64_t dk_paged_attention_varlen_workspace_bytes(const dk_varlen_attn_params* a, int head_dim,
                                                             int max_query_len, int max_seq_len) {
  using namespace dk::varlen;
  if (a == nullptr || a->num_kv_heads <= 0 || a->num_q_heads < a->num_kv_heads ||
      a->num_q_heads % a->num_kv_heads != 0 || a->num_q_heads / a->num_kv_heads > DK_MAX_GQA_GROUP || head_dim > 256 ||
      a->num_tokens <= 0 || a->num_seqs <= 0 ||
      max_query_len < 0 || max_seq_len < 0 || a->num_blocks < 0 || a->max_blocks < 0 || a->block_size <= 0 || head_dim <= 0)
    return 0;  // nothing to do, or refused by the call
  const int max_len = length_bound(a, max_seq_len);
  return make_plan(a, head_dim, max_query_len, max_len, window_bound(a, max_len)).ws_bytes;
}

extern "C" int dk_paged_attention_varlen(const dk_varlen_attn_params* a, int dtype, int head_dim, int max_query_len,
                                         int max_seq_len, void* workspace, int64_t workspace_bytes, void* stream) {
  return dk::varlen::run("paged_attention_varlen", a, dtype, head_dim, max_query_len, max_seq_len, false, 1.0f, 1.0f,
                         workspace, workspace_bytes, stream);
}

extern "C" int dk_paged_attention_varlen_fp8(const dk_varlen_attn_params* a, int dtype, int head_dim, int max_query_len,
                                             int max_seq_len, float k_scale, float v_scale, void* workspace,
                                             int64_t workspace_bytes, void* stream) {
  return dk::varlen::run("paged_attention_varlen_fp8", a, dtype, head_dim, max_query_len, max_seq_len, true, k_scale,
                         v_scale, workspace, workspace_bytes, stream);
}
