// RMS norm of every query and key head, the rotation by the token's position
// and the write into the paged cache, in one pass (gfx950):
//
//   y = x / sqrt(mean(x^2) + eps) * w                 (per head, w of head_size)
//   (a, b) -> (a cos - b sin, b cos + a sin)          (first rot_dim columns)
//
// with cos / sin of the token's position from a [max_position, rot_dim] table,
// NeoX pairs (i, i + rot_dim / 2) or GPT-J pairs (2 i, 2 i + 1). Everything is
// fp32 between the one read and the one write of each element: the norm is not
// rounded before the rotation, and a value is rounded once, to the model dtype
// or straight to the cache's e4m3fn. A token whose position lies outside the
// table is no token (padding): its rows and its cache slot are left as they
// were.
#include <cmath>
#include <type_traits>

#include "../../include/decodekernels_amd.h"
#include "dk_device.h"
#include "dk_host.h"

namespace dk {
namespace qk_norm {

constexpr int kThreads = 256;

struct KParams {
  const int64_t* positions;
  const uint16_t* q;
  const uint16_t* k;
  const uint16_t* v;     // nullptr: no cache
  uint16_t* q_out;
  uint16_t* k_out;       // nullptr with a cache
  const uint16_t* q_w;
  const uint16_t* k_w;
  const void* table;
  void* kc;
  void* vc;
  const int64_t* slots;
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh, qo_st, qo_sh, ko_st, ko_sh, table_stride;
  int64_t kc_sb, kc_st, kc_sh, vc_sb, vc_st, vc_sh;
  int num_tokens, hq, hkv, d, rot_dim, max_position, block_size, num_blocks, neox;
  float eps, k_scale, v_scale;
};

template <typename E, typename CT>
__device__ __forceinline__ float table_at(const void* base, int64_t i) {
  if constexpr (sizeof(CT) == 4) return static_cast<const float*>(base)[i];
  else return E::to_float(static_cast<const uint16_t*>(base)[i]);
}

// x / scale saturated to the largest finite e4m3fn (NaN stays NaN).
__device__ __forceinline__ float e4m3_range(float x, float scale) {
  const float y = x / scale;
  return y != y ? y : fminf(fmaxf(y, -448.0f), 448.0f);
}

// Where a wave's head goes: rows of E, or of e4m3fn bytes.
template <typename E, bool FP8>
__device__ __forceinline__ void put(void* row, int i, float x, float scale) {
  if constexpr (FP8) {
    static_cast<uint8_t*>(row)[i] =
        static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(x, scale), 0.0f, 0, false) & 0xff);
  } else {
    static_cast<uint16_t*>(row)[i] = E::from_float(x);
  }
}

// One wave per (token, head): any head size, strides and alignment. Each lane
// owns whole pairs, and the sum of squares has been taken before the first
// write, so the rows may be rewritten in place.
template <typename E, typename CT, bool FP8>
__global__ __launch_bounds__(kThreads) void norm_rotate_kernel(const KParams p) {
  const int lane = threadIdx.x % kWave;
  const int heads = p.hq + (p.v != nullptr ? 2 : 1) * p.hkv;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + threadIdx.x / kWave;
  const int64_t t = item / heads;
  int h = static_cast<int>(item - t * heads);
  if (t >= p.num_tokens) return;
  const int64_t pos = p.positions[t];
  if (pos < 0 || pos >= p.max_position) return;
  int64_t blk = 0, off = 0;
  if (h >= p.hq && p.v != nullptr) {
    const int64_t slot = p.slots[t];
    if (slot < 0) return;
    blk = slot / p.block_size;
    off = slot - blk * p.block_size;
    if (blk >= p.num_blocks) return;
  }
  constexpr int kCacheElt = FP8 ? 1 : 2;
  if (h >= p.hq + p.hkv) {  // value: copied
    h -= p.hq + p.hkv;
    const uint16_t* src = p.v + t * p.v_st + h * p.v_sh;
    void* dst = static_cast<char*>(p.vc) + kCacheElt * (blk * p.vc_sb + off * p.vc_st + h * p.vc_sh);
    for (int i = lane; i < p.d; i += kWave) {
      if constexpr (FP8) put<E, true>(dst, i, E::to_float(src[i]), p.v_scale);
      else static_cast<uint16_t*>(dst)[i] = src[i];
    }
    return;
  }
  const bool is_q = h < p.hq;
  if (!is_q) h -= p.hq;
  const uint16_t* x = is_q ? p.q + t * p.q_st + h * p.q_sh : p.k + t * p.k_st + h * p.k_sh;
  const uint16_t* w = is_q ? p.q_w : p.k_w;
  const bool cached = !is_q && p.v != nullptr;
  void* dst = is_q ? static_cast<void*>(p.q_out + t * p.qo_st + h * p.qo_sh)
              : !cached
                  ? static_cast<void*>(p.k_out + t * p.ko_st + h * p.ko_sh)
                  : static_cast<void*>(static_cast<char*>(p.kc) + kCacheElt * (blk * p.kc_sb + off * p.kc_st + h * p.kc_sh));
  float ss = 0.0f;
  for (int i = lane; i < p.d; i += kWave) {
    const float a = E::to_float(x[i]);
    ss += a * a;
  }
  const float inv = 1.0f / __fsqrt_rn(wave_sum(ss) / static_cast<float>(p.d) + p.eps);
  const int half = p.rot_dim / 2;
  auto store = [&](int i, float y) {
    if (cached) put<E, FP8>(dst, i, y, p.k_scale);
    else put<E, false>(dst, i, y, 1.0f);
  };
  const int64_t row = pos * p.table_stride;
  for (int i = lane; i < half; i += kWave) {
    const float c = table_at<E, CT>(p.table, row + i), s = table_at<E, CT>(p.table, row + half + i);
    const int ia = p.neox ? i : 2 * i, ib = p.neox ? i + half : 2 * i + 1;
    const float a = E::to_float(x[ia]) * inv * E::to_float(w[ia]);
    const float b = E::to_float(x[ib]) * inv * E::to_float(w[ib]);
    store(ia, a * c - b * s);
    store(ib, b * c + a * s);
  }
  for (int i = p.rot_dim + lane; i < p.d; i += kWave) store(i, E::to_float(x[i]) * inv * E::to_float(w[i]));
}

template <typename E, typename CT, bool FP8>
hipError_t launch(const KParams& kp, hipStream_t s) {
  const int64_t items = static_cast<int64_t>(kp.num_tokens) * (kp.hq + (kp.v != nullptr ? 2 : 1) * kp.hkv);
  const dim3 grid(static_cast<unsigned>(ceil_div64(items, kThreads / kWave))), block(kThreads);
  hipLaunchKernelGGL((norm_rotate_kernel<E, CT, FP8>), grid, block, 0, s, kp);
  return hipGetLastError();
}

template <typename E>
hipError_t launch_dtype(const KParams& kp, int table_dtype, bool fp8, hipStream_t s) {
  if (table_dtype == DK_FLOAT32) return fp8 ? launch<E, float, true>(kp, s) : launch<E, float, false>(kp, s);
  return fp8 ? launch<E, uint16_t, true>(kp, s) : launch<E, uint16_t, false>(kp, s);
}

// Argument checks, then the launch; c == nullptr: no cache.
int run(const char* op, const dk_rotary_params* r, const dk_qk_norm_params* n, const dk_cache_write_params* c, int dtype,
        bool with_cache, bool fp8, float k_scale, float v_scale, void* stream) {
  clear_error();
  if (r == nullptr || n == nullptr || (with_cache && c == nullptr)) return fail("%s: params must not be NULL", op);
  if (dtype != DK_FLOAT16 && dtype != DK_BFLOAT16) return fail("%s: expected float16 or bfloat16, got dtype code %d", op, dtype);
  if (r->cache_dtype != dtype && r->cache_dtype != DK_FLOAT32)
    return fail("%s: cos_sin_cache must be float32 or the query dtype", op);
  if (r->num_tokens < 0 || r->num_q_heads < 0 || r->num_kv_heads < 0 || r->max_position < 0)
    return fail("%s: sizes must be non-negative", op);
  if (r->head_size <= 0) return fail("%s: head_size must be positive", op);
  if (r->rot_dim <= 0 || r->rot_dim % 2 != 0 || r->rot_dim > r->head_size)
    return fail("%s: rot_dim must be even and at most head_size", op);
  if (!(n->eps >= 0.0f && n->eps < INFINITY)) return fail("%s: eps must be non-negative and finite", op);
  if (with_cache) {
    if (c->num_tokens != r->num_tokens) return fail("%s: the rotary and cache token counts differ", op);
    if (c->num_kv_heads != r->num_kv_heads || c->head_size != r->head_size)
      return fail("%s: the rotary and cache head counts / sizes differ", op);
    if (r->key != c->key || r->k_stride_token != c->k_stride_token || r->k_stride_head != c->k_stride_head)
      return fail("%s: the rotated key and the cached key must be the same tensor", op);
    if (c->block_size <= 0 || c->num_blocks < 0) return fail("%s: block_size must be positive", op);
    if (fp8 && !(k_scale > 0.0f && v_scale > 0.0f && k_scale < INFINITY && v_scale < INFINITY))
      return fail("%s: k_scale and v_scale must be positive and finite", op);
  }
  const int64_t items = static_cast<int64_t>(r->num_tokens) * (static_cast<int64_t>(r->num_q_heads) + 2ll * r->num_kv_heads);
  if (items == 0) return hipSuccess;
  if (items > 0x7fffffff) return fail("%s: too many tokens x heads", op);
  if (r->positions == nullptr || r->cos_sin_cache == nullptr) return fail("%s: positions and cos_sin_cache must not be NULL", op);
  if (r->num_q_heads > 0 && (r->query == nullptr || n->query_out == nullptr || n->q_weight == nullptr))
    return fail("%s: query, query_out and q_weight must not be NULL", op);
  if (r->num_kv_heads > 0) {
    if (r->key == nullptr || n->k_weight == nullptr) return fail("%s: key and k_weight must not be NULL", op);
    if (!with_cache && n->key_out == nullptr) return fail("%s: key_out must not be NULL", op);
    if (with_cache && (c->value == nullptr || c->key_cache == nullptr || c->value_cache == nullptr || c->slot_mapping == nullptr))
      return fail("%s: value, caches and slot_mapping must not be NULL", op);
  }
  KParams kp{};
  kp.positions = r->positions;
  kp.q = static_cast<const uint16_t*>(r->query);
  kp.k = static_cast<const uint16_t*>(r->key);
  kp.q_out = static_cast<uint16_t*>(n->query_out);
  kp.k_out = static_cast<uint16_t*>(n->key_out);
  kp.q_w = static_cast<const uint16_t*>(n->q_weight);
  kp.k_w = static_cast<const uint16_t*>(n->k_weight);
  kp.table = r->cos_sin_cache;
  kp.q_st = r->q_stride_token;
  kp.q_sh = r->q_stride_head;
  kp.k_st = r->k_stride_token;
  kp.k_sh = r->k_stride_head;
  kp.qo_st = n->qo_stride_token;
  kp.qo_sh = n->qo_stride_head;
  kp.ko_st = n->ko_stride_token;
  kp.ko_sh = n->ko_stride_head;
  kp.table_stride = r->cache_stride;
  kp.num_tokens = r->num_tokens;
  kp.hq = r->num_q_heads;
  kp.hkv = r->num_kv_heads;
  kp.d = r->head_size;
  kp.rot_dim = r->rot_dim;
  kp.max_position = r->max_position;
  kp.neox = r->is_neox != 0;
  kp.eps = n->eps;
  kp.k_scale = k_scale;
  kp.v_scale = v_scale;
  if (with_cache) {
    kp.v = static_cast<const uint16_t*>(c->value);
    kp.kc = c->key_cache;
    kp.vc = c->value_cache;
    kp.slots = c->slot_mapping;
    kp.v_st = c->v_stride_token;
    kp.v_sh = c->v_stride_head;
    kp.kc_sb = c->kc_stride_block;
    kp.kc_st = c->kc_stride_token;
    kp.kc_sh = c->kc_stride_head;
    kp.vc_sb = c->vc_stride_block;
    kp.vc_st = c->vc_stride_token;
    kp.vc_sh = c->vc_stride_head;
    kp.block_size = c->block_size;
    kp.num_blocks = c->num_blocks;
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  return static_cast<int>(dtype == DK_BFLOAT16 ? launch_dtype<Bf16>(kp, r->cache_dtype, fp8, s)
                                               : launch_dtype<F16>(kp, r->cache_dtype, fp8, s));
}

}  // namespace qk_norm
}  // namespace dk

extern "C" int dk_qk_norm_rotary_embedding(const dk_rotary_params* r, const dk_qk_norm_params* n, int dtype,
                                           void* stream) {
  return dk::qk_norm::run("qk_norm_rotary_embedding", r, n, nullptr, dtype, false, false, 1.0f, 1.0f, stream);
}

extern "C" int dk_qk_norm_rotary_embedding_and_cache(const dk_rotary_params* r, const dk_qk_norm_params* n,
                                                     const dk_cache_write_params* c, int dtype, void* stream) {
  return dk::qk_norm::run("qk_norm_rotary_embedding_and_cache", r, n, c, dtype, true, false, 1.0f, 1.0f, stream);
}

extern "C" int dk_qk_norm_rotary_embedding_and_cache_fp8(const dk_rotary_params* r, const dk_qk_norm_params* n,
                                                         const dk_cache_write_params* c, int dtype, float k_scale,
                                                         float v_scale, void* stream) {
  return dk::qk_norm::run("qk_norm_rotary_embedding_and_cache_fp8", r, n, c, dtype, true, true, k_scale, v_scale, stream);
}
