// Attention of the new tokens of a ragged batch over a paged KV cache (gfx950):
// sequence s brings query tokens [start[s], start[s + 1]), the last ones of its
// seq_lens[s] cached tokens, one of them (decode) or thousands (a prompt).
//
//   x_ij = scale * q_i . k_j,  capped to  cap * tanh(x_ij / cap),
//   less slope_h * |i - j|,  over the keys j that token i sees:
//   j <= i and j > i - window, or j < prefix_s;
//   out_i = sum_j softmax_j(x_ij) v_j,  zeros where it sees no key.
#include <cmath>
#include <cstdint>

#include "../../include/decodekernels_amd.h"
#include "dk_device.h"
#include "dk_host.h"

namespace dk {
namespace varlen {

constexpr float kLog2e = 1.4426950408889634f;

struct KParams {
  uint16_t* out;
  const uint16_t* q;
  const void* k;
  const void* v;
  const int32_t* tables;
  const int32_t* lens;
  const int32_t* starts;
  const int32_t* prefix;   // nullptr: none
  const float* slopes;     // nullptr: none
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int64_t bt_stride;
  int num_tokens, num_seqs, hq, group, block_size, num_blocks;
  int max_len;             // no length goes past it: the caller's bound, and what the tables can hold
  int window;              // keys a token sees, itself included; max_len where it sees all before it
  float scale, softcap, k_scale, v_scale;
};

// The sequence that owns token t: how many end at or before it (num_seqs: none
// does). The lanes count side by side.
__device__ __forceinline__ int find_seq(const KParams& p, int t, int lane) {
  int s = 0;
  for (int i = lane; i < p.num_seqs; i += kWave) s += p.starts[i + 1] <= t ? 1 : 0;
#pragma unroll
  for (int off = kWave / 2; off > 0; off >>= 1) s += __shfl_xor(s, off, kWave);
  return s;
}

template <typename E, bool FP8>
__device__ __forceinline__ float element(const void* base, int64_t i) {
  if constexpr (FP8) {
    return __builtin_amdgcn_cvt_f32_fp8(static_cast<const uint8_t*>(base)[i], 0);
  } else {
    return E::to_float(static_cast<const uint16_t*>(base)[i]);
  }
}

// One wave per (token, query head): scores of 64 keys at a time, a key per
// lane, then the weighted sum with the columns over the lanes.
template <typename E, bool FP8>
__global__ __launch_bounds__(kWave) void simple_kernel(const KParams p, int d) {
  __shared__ float q[256];
  __shared__ float weight[kWave];
  const int lane = threadIdx.x;
  const int t = blockIdx.x / p.hq;
  const int h = blockIdx.x - t * p.hq;
  const int kvh = h / p.group;
  const int s = find_seq(p, t, lane);
  if (s >= p.num_seqs) return;  // a row behind the last sequence
  const int first = max(p.starts[s], 0);
  const int n = min(p.starts[s + 1], p.num_tokens) - first;
  const int len = max(min(p.lens[s], p.max_len), 0);
  const int pos = len - n + (t - first);
  const int pre = p.prefix != nullptr ? min(max(p.prefix[s], 0), len) : 0;
  for (int i = lane; i < d; i += kWave) q[i] = E::to_float(p.q[t * p.q_st + h * p.q_sh + i]);
  __syncthreads();
  const float slope = p.slopes != nullptr ? p.slopes[h] : 0.0f;
  float top = -__builtin_huge_valf(), total = 0.0f;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int low = max(pos - p.window + 1, 0);
  const int end = max(pre, pos + 1);
  for (int j0 = 0; j0 < end; j0 += kWave) {
    if (j0 >= pre && j0 + kWave <= low) continue;
    const int j = j0 + lane;
    const bool sees = j < pre || (j <= pos && j >= low);
    float x = -__builtin_huge_valf();
    int64_t at = 0;
    if (sees) {
      const int page = min(max(p.tables[s * p.bt_stride + j / p.block_size], 0), p.num_blocks - 1);
      const int64_t row = page * p.k_sb + (j % p.block_size) * p.k_st + kvh * p.k_sh;
      at = page * p.v_sb + (j % p.block_size) * p.v_st + kvh * p.v_sh;
      float dot = 0.0f;
      for (int i = 0; i < d; ++i) dot += q[i] * element<E, FP8>(p.k, row + i);
      x = dot * p.scale * p.k_scale;
      if (p.softcap > 0.0f) x = p.softcap * tanhf(x / p.softcap);
      x -= slope * static_cast<float>(pos > j ? pos - j : j - pos);
    }
    const float new_top = fmaxf(top, wave_max(x));
    const float ref = new_top == -__builtin_huge_valf() ? 0.0f : new_top;
    const float w = sees ? __builtin_amdgcn_exp2f((x - ref) * kLog2e) : 0.0f;
    const float alpha = __builtin_amdgcn_exp2f((top - ref) * kLog2e);
    total = total * alpha + wave_sum(w);
    top = new_top;
    __syncthreads();
    weight[lane] = w;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 4; ++c) acc[c] *= alpha;
    const uint64_t seen = __ballot(sees);
    for (int jj = 0; jj < kWave; ++jj) {
      if (!((seen >> jj) & 1)) continue;  // never a product with a hidden value
      const int64_t row = __shfl(at, jj, kWave);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + c * kWave < d) acc[c] += weight[jj] * element<E, FP8>(p.v, row + lane + c * kWave);
    }
  }
  uint16_t* out = p.out + t * p.o_st + h * p.o_sh;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + c * kWave < d) out[lane + c * kWave] = E::from_float(total == 0.0f ? 0.0f : acc[c] / total * p.v_scale);
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
  const int64_t held = static_cast<int64_t>(a->max_blocks) * a->block_size;
  const int max_len = a->num_blocks == 0 ? 0 : static_cast<int>(held < max_seq_len ? held : max_seq_len);
  if (max_len > 0 && (a->k_cache == nullptr || a->v_cache == nullptr || a->block_tables == nullptr))
    return fail("%s: k_cache, v_cache and block_tables must not be NULL", op);
  if (a->q_stride_token < 0 || a->q_stride_head < 0 || a->k_stride_block < 0 || a->k_stride_token < 0 ||
      a->k_stride_head < 0 || a->v_stride_block < 0 || a->v_stride_token < 0 || a->v_stride_head < 0 || a->bt_stride < 0 ||
      a->out_stride_token < 0 || a->out_stride_head < 0)
    return fail("%s: strides must be non-negative", op);
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
  kp.q_st = a->q_stride_token;
  kp.q_sh = a->q_stride_head;
  kp.o_st = a->out_stride_token;
  kp.o_sh = a->out_stride_head;
  kp.k_sb = a->k_stride_block;
  kp.k_st = a->k_stride_token;
  kp.k_sh = a->k_stride_head;
  kp.v_sb = a->v_stride_block;
  kp.v_st = a->v_stride_token;
  kp.v_sh = a->v_stride_head;
  kp.bt_stride = a->bt_stride;
  kp.num_tokens = a->num_tokens;
  kp.num_seqs = a->num_seqs;
  kp.hq = a->num_q_heads;
  kp.group = a->num_q_heads / a->num_kv_heads;
  kp.block_size = a->block_size;
  kp.num_blocks = a->num_blocks;
  kp.max_len = max_len;
  kp.window = a->window == 0 || a->window > max_len ? (max_len > 0 ? max_len : 1) : a->window;
  kp.scale = a->scale;
  kp.softcap = a->softcap;
  kp.k_scale = k_scale;
  kp.v_scale = v_scale;
  (void)workspace, (void)workspace_bytes;
  const dim3 grid(static_cast<unsigned>(a->num_tokens * a->num_q_heads)), block(kWave);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == DK_BFLOAT16) {
    if (fp8) hipLaunchKernelGGL((simple_kernel<Bf16, true>), grid, block, 0, s, kp, head_dim);
    else hipLaunchKernelGGL((simple_kernel<Bf16, false>), grid, block, 0, s, kp, head_dim);
  } else {
    if (fp8) hipLaunchKernelGGL((simple_kernel<F16, true>), grid, block, 0, s, kp, head_dim);
    else hipLaunchKernelGGL((simple_kernel<F16, false>), grid, block, 0, s, kp, head_dim);
  }
  return static_cast<int>(hipGetLastError());
}

}  // namespace varlen
}  // namespace dk

extern "C" int64_t dk_paged_attention_varlen_workspace_bytes(const dk_varlen_attn_params* a, int head_dim,
                                                             int max_query_len, int max_seq_len) {
  (void)a, (void)head_dim, (void)max_query_len, (void)max_seq_len;
  return 0;
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
