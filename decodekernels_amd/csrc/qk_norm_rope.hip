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
// Tokens up to which a token's heads are spread over workgroups (32 / 8 heads of
// 128 with the cache, cold, spread and not: 64 tokens 7.2 and 8.3 us, 512 9.5 and
// 10.0, 1024 13.7 and 12.8, 4096 33.8 and 31.9).
constexpr int kFewTokens = 512;

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

// 8 values from 16 bytes of E.
template <typename E>
__device__ __forceinline__ void widen(u32x4 w, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = E::lo(w[i]), x[2 * i + 1] = E::hi(w[i]);
}

// 4 (N = 4) or 8 entries of a table row, 16-byte (16-bit tables: 8-byte) aligned.
template <typename E, typename CT, int N>
__device__ __forceinline__ void table_row(const void* base, int64_t i, float* out) {
  if constexpr (sizeof(CT) == 4) {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + i + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) out[j + e] = v[e];
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 4) {
      const u32x2 v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(base) + i + j);
      out[j] = E::lo(v[0]), out[j + 1] = E::hi(v[0]), out[j + 2] = E::lo(v[1]), out[j + 3] = E::hi(v[1]);
    }
  }
}

// 8 values, rounded once, to 16 bytes of E or 8 of e4m3fn.
template <typename E, bool FP8>
__device__ __forceinline__ void put8(void* dst, const float (&y)[8], float scale) {
  if constexpr (FP8) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(y[4 * i], scale), e4m3_range(y[4 * i + 1], scale), 0, false);
      v = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(y[4 * i + 2], scale), e4m3_range(y[4 * i + 3], scale), v, true);
      w[i] = static_cast<uint32_t>(v);
    }
    *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
  } else {
    *reinterpret_cast<u32x4*>(dst) =
        u32x4{pack2<E>(y[0], y[1]), pack2<E>(y[2], y[3]), pack2<E>(y[4], y[5]), pack2<E>(y[6], y[7])};
  }
}

// The same with 16-byte accesses. LP lanes take a head, two chunks of 8 columns
// each that hold the two halves of 8 pairs (NeoX: a chunk of the first half of
// the rotated columns and its partner; GPT-J, and columns past rot_dim: two
// neighbours), so no pair crosses lanes. A workgroup takes one token, and the
// lanes keep its cos / sin and the weights while they go through the heads.
// Bound by memory: 16384 tokens of 32/8 heads of 128 with the cache write are
// 407 MB, 74 us, 5.5 TB/s; 1003 tokens of 28 / 4 heads into fp8 (18 MB) 8.2 us;
// 8 tokens 3.8 us, a launch and two dependent reads.
template <typename E, typename CT, bool NEOX, bool FP8, int LP>
__global__ __launch_bounds__(kThreads) void norm_rotate_vec_kernel(const KParams p) {
  constexpr int kHeads = kThreads / LP;  // side by side
  constexpr int kElt = FP8 ? 1 : 2;      // of the cache
  const int c = threadIdx.x % LP;
  const int heads = p.hq + (p.v != nullptr ? 2 : 1) * p.hkv;
  const int64_t t = blockIdx.x;
  const int64_t pos = p.positions[t];
  if (pos < 0 || pos >= p.max_position) return;
  const int64_t slot = p.v != nullptr ? p.slots[t] : 0;
  const int64_t blk = slot >= 0 ? slot / p.block_size : p.num_blocks;
  const int64_t off = slot - blk * p.block_size;
  const bool put_cache = p.v == nullptr || blk < p.num_blocks;
  const bool mine = 16 * c < p.d;
  const int half = p.rot_dim / 2;
  // This lane's columns, and the first of its 8 pairs.
  const bool pairs = NEOX && 8 * c < half;
  const int col0 = pairs ? 8 * c : 16 * c;  // past the rotated ones: pairs' chunks end at rot_dim = 16 (half / 8)
  const int col1 = pairs ? half + 8 * c : 16 * c + 8;
  float cs[8], sn[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) cs[j] = 1.0f, sn[j] = 0.0f;
  if (mine) {
    const int64_t row = pos * p.table_stride;
    if constexpr (NEOX) {
      if (pairs) {
        table_row<E, CT, 8>(p.table, row + 8 * c, cs);
        table_row<E, CT, 8>(p.table, row + half + 8 * c, sn);
      }
    } else {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        if (16 * c + 8 * x < p.rot_dim) {
          table_row<E, CT, 4>(p.table, row + 8 * c + 4 * x, cs + 4 * x);
          table_row<E, CT, 4>(p.table, row + half + 8 * c + 4 * x, sn + 4 * x);
        }
      }
    }
  }
  const int first = static_cast<int>(blockIdx.y) * kHeads + static_cast<int>(threadIdx.x) / LP;
  for (int h = first; h < heads; h += kHeads * static_cast<int>(gridDim.y)) {
    const bool is_q = h < p.hq, is_v = h >= p.hq + p.hkv;
    const int kh = is_q ? h : is_v ? h - p.hq - p.hkv : h - p.hq;
    const uint16_t* src = is_q ? p.q + t * p.q_st + kh * p.q_sh : is_v ? p.v + t * p.v_st + kh * p.v_sh : p.k + t * p.k_st + kh * p.k_sh;
    u32x4 r0 = {0u, 0u, 0u, 0u}, r1 = {0u, 0u, 0u, 0u};
    if (mine) {
      r0 = *reinterpret_cast<const u32x4*>(src + col0);
      r1 = *reinterpret_cast<const u32x4*>(src + col1);
    }
    float x0[8], x1[8];
    widen<E>(r0, x0);
    widen<E>(r1, x1);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x0[j] * x0[j] + x1[j] * x1[j];
#pragma unroll
    for (int o = 1; o < LP; o <<= 1) ss += __shfl_xor(ss, o, kWave);
    if (!mine || (!is_q && !put_cache)) continue;
    if (is_v) {
      char* dst = static_cast<char*>(p.vc) + kElt * (blk * p.vc_sb + off * p.vc_st + kh * p.vc_sh);
      if constexpr (FP8) {
        put8<E, true>(dst + col0, x0, p.v_scale);
        put8<E, true>(dst + col1, x1, p.v_scale);
      } else {
        *reinterpret_cast<u32x4*>(dst + 2 * col0) = r0;
        *reinterpret_cast<u32x4*>(dst + 2 * col1) = r1;
      }
      continue;
    }
    const float inv = 1.0f / __fsqrt_rn(ss / static_cast<float>(p.d) + p.eps);
    const uint16_t* w = is_q ? p.q_w : p.k_w;
    float w0[8], w1[8];
    widen<E>(*reinterpret_cast<const u32x4*>(w + col0), w0);
    widen<E>(*reinterpret_cast<const u32x4*>(w + col1), w1);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x0[j] = x0[j] * inv * w0[j];
      x1[j] = x1[j] * inv * w1[j];
    }
    float y0[8], y1[8];
    if constexpr (NEOX) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y0[j] = x0[j] * cs[j] - x1[j] * sn[j];
        y1[j] = x1[j] * cs[j] + x0[j] * sn[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        y0[2 * j] = x0[2 * j] * cs[j] - x0[2 * j + 1] * sn[j];
        y0[2 * j + 1] = x0[2 * j + 1] * cs[j] + x0[2 * j] * sn[j];
        y1[2 * j] = x1[2 * j] * cs[4 + j] - x1[2 * j + 1] * sn[4 + j];
        y1[2 * j + 1] = x1[2 * j + 1] * cs[4 + j] + x1[2 * j] * sn[4 + j];
      }
    }
    if (is_q || p.v == nullptr) {
      uint16_t* dst = is_q ? p.q_out + t * p.qo_st + kh * p.qo_sh : p.k_out + t * p.ko_st + kh * p.ko_sh;
      put8<E, false>(dst + col0, y0, 1.0f);
      put8<E, false>(dst + col1, y1, 1.0f);
    } else {
      char* dst = static_cast<char*>(p.kc) + kElt * (blk * p.kc_sb + off * p.kc_st + kh * p.kc_sh);
      put8<E, FP8>(dst + kElt * col0, y0, p.k_scale);
      put8<E, FP8>(dst + kElt * col1, y1, p.k_scale);
    }
  }
}

// 16-byte accesses everywhere, and whole chunks on either side of rot_dim.
template <typename CT>
bool vectorizable(const KParams& p, bool fp8) {
  const int half = p.rot_dim / 2;
  auto rows = [](const void* b, int64_t st, int64_t sh) { return aligned_to(b, 16) && st % 8 == 0 && sh % 8 == 0; };
  bool ok = p.d % 16 == 0 && p.d <= 256 && p.rot_dim % (p.neox ? 16 : 8) == 0 &&
            (p.hq == 0 || (rows(p.q, p.q_st, p.q_sh) && rows(p.q_out, p.qo_st, p.qo_sh) && aligned_to(p.q_w, 16))) &&
            (p.hkv == 0 || (rows(p.k, p.k_st, p.k_sh) && aligned_to(p.k_w, 16)));
  ok = ok && (sizeof(CT) == 4 ? aligned_to(p.table, 16) && p.table_stride % 4 == 0 && half % 4 == 0
                              : aligned_to(p.table, 8) && p.table_stride % 4 == 0 && half % 4 == 0);
  if (p.v == nullptr) return ok && (p.hkv == 0 || rows(p.k_out, p.ko_st, p.ko_sh));
  const int bytes = fp8 ? 8 : 16;  // of 8 elements: strides are multiples of 8 elements either way
  return ok && rows(p.v, p.v_st, p.v_sh) && aligned_to(p.kc, bytes) && aligned_to(p.vc, bytes) && p.kc_sb % 8 == 0 &&
         p.kc_st % 8 == 0 && p.kc_sh % 8 == 0 && p.vc_sb % 8 == 0 && p.vc_st % 8 == 0 && p.vc_sh % 8 == 0;
}

template <typename E, typename CT, bool FP8, int LP>
hipError_t launch_vec(const KParams& kp, hipStream_t s) {
  const int heads = kp.hq + (kp.v != nullptr ? 2 : 1) * kp.hkv;
  const int passes = (heads + kThreads / LP - 1) / (kThreads / LP);
  // A token's heads over several workgroups where there are few tokens.
  const int split = kp.num_tokens <= kFewTokens ? passes : 1;
  const dim3 grid(static_cast<unsigned>(kp.num_tokens), static_cast<unsigned>(split)), block(kThreads);
  if (kp.neox) hipLaunchKernelGGL((norm_rotate_vec_kernel<E, CT, true, FP8, LP>), grid, block, 0, s, kp);
  else hipLaunchKernelGGL((norm_rotate_vec_kernel<E, CT, false, FP8, LP>), grid, block, 0, s, kp);
  return hipGetLastError();
}

template <typename E, typename CT, bool FP8>
hipError_t launch(const KParams& kp, hipStream_t s) {
  if (vectorizable<CT>(kp, FP8)) {
    if (kp.d <= 64) return launch_vec<E, CT, FP8, 4>(kp, s);
    if (kp.d <= 128) return launch_vec<E, CT, FP8, 8>(kp, s);
    return launch_vec<E, CT, FP8, 16>(kp, s);
  }
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
