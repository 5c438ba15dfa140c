// Attention of the new tokens of a ragged batch over a paged KV cache (gfx950):
// sequence s brings query tokens [start[s], start[s + 1]), the last ones of its
// seq_lens[s] cached tokens, one of them (decode) or thousands (a prompt).
//
//   x_ij = scale * q_i . k_j,  capped to  cap * tanh(x_ij / cap),
//   less slope_h * |i - j|,  over the keys j that token i sees:
//   j <= i and j > i - window, or j < prefix_s;
//   out_i = sum_j softmax_j(x_ij) v_j,  zeros where it sees no key.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <type_traits>

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
  // Element strides, each below 2^31 (checked by the host): as 32-bit arguments
  // they take half the scalar registers. Addresses are formed in 64 bits.
  int32_t q_st, q_sh, o_st, o_sh;
  int32_t k_sb, k_st, k_sh, v_sb, v_st, v_sh;
  int32_t bt_stride;
  int num_tokens, num_seqs, hq, group, block_size, num_blocks;
  int max_len;             // no length goes past it: the caller's bound, and what the tables can hold
  int window;              // keys a token sees, itself included; max_len where it sees all before it
  int hkv, rows_short;     // sequences of more than rows_short rows a KV head run in tiles (tile_kernel)
  int split_items;         // workgroups that the tiles of a call may be split over; 0: never split
  float* ws;               // partial results
  uint32_t bs_mul;         // j / block_size = (j * bs_mul) >> bs_shift, for j < 2^31
  int bs_shift;
  float scale, softcap, k_scale, v_scale;
  // In log2 units: the factor of q.k (positive: its sign goes to q), the cap
  // and, for its tanh, exp(2 y) = 2^(cap_in s).
  float scale2, cap2, cap_in;
  uint32_t q_sign;
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

// 8 e4m3fn bytes as 8 elements of E, exactly.
template <typename E>
__device__ __forceinline__ u32x4 fp8x8_to(u32x2 w) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w[0], false);
  const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(w[0], true);
  const auto c = __builtin_amdgcn_cvt_pk_f32_fp8(w[1], false);
  const auto d = __builtin_amdgcn_cvt_pk_f32_fp8(w[1], true);
  return u32x4{pack2<E>(a[0], a[1]), pack2<E>(b[0], b[1]), pack2<E>(c[0], c[1]), pack2<E>(d[0], d[1])};
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
  if (static_cast<int64_t>(n) * p.group > p.rows_short) return;
  const int pre = p.prefix != nullptr ? min(max(p.prefix[s], 0), len) : 0;
  for (int i = lane; i < d; i += kWave) q[i] = E::to_float(p.q[static_cast<int64_t>(t) * p.q_st + static_cast<int64_t>(h) * p.q_sh + i]);
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
      const int64_t page = min(max(p.tables[static_cast<int64_t>(s) * p.bt_stride + j / p.block_size], 0), p.num_blocks - 1);
      const int64_t off = j % p.block_size;
      const int64_t row = page * p.k_sb + off * p.k_st + static_cast<int64_t>(kvh) * p.k_sh;
      at = page * p.v_sb + off * p.v_st + static_cast<int64_t>(kvh) * p.v_sh;
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
  uint16_t* out = p.out + static_cast<int64_t>(t) * p.o_st + static_cast<int64_t>(h) * p.o_sh;
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + c * kWave < d) out[lane + c * kWave] = E::from_float(total == 0.0f ? 0.0f : acc[c] / total * p.v_scale);
}


typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename E>
__device__ __forceinline__ f32x16 mfma_32x32x16(u32x4 a, u32x4 b, f32x16 c);
template <>
__device__ __forceinline__ f32x16 mfma_32x32x16<Bf16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16 mfma_32x32x16<F16>(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr int kTileWaves = 4;
constexpr int kTileThreads = kTileWaves * kWave;
constexpr int kTileRows = 32 * kTileWaves;  // (token, query head of the group) rows of a workgroup
constexpr int kRsrcWord3 = 0x00020000;      // word 3 of a gfx9-family buffer resource for raw loads
constexpr int kSeqsPerThread = 4;

// Infinities and NaN of the dtype: the exponent bits of an element, and the
// lowest of them.
template <typename E>
constexpr uint32_t kExpBits = std::is_same<E, Bf16>::value ? 0x7f80u : 0x7c00u;
template <typename E>
constexpr uint32_t kExpUnit = std::is_same<E, Bf16>::value ? 0x80u : 0x400u;

// Folds 8 elements into `open`, whose halves stay non-zero while every element
// is finite (packed minima instead of 8 comparisons, whose lane masks would
// crowd the scalar registers).
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
template <typename E>
__device__ __forceinline__ u16x2 fold_finite(u16x2 open, u32x4 v) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    open = __builtin_elementwise_min(open, __builtin_bit_cast(u16x2, ~v[i] & (kExpBits<E> * 0x10001u)));
  return open;
}

// Takes the infinities and NaN out of 8 elements (0 in their places) and says
// where they were: bit e of up for infinity, of down for minus infinity, of
// both for NaN.
template <typename E>
__device__ __forceinline__ u32x4 take_out(u32x4 v, uint32_t& up, uint32_t& down) {
  constexpr uint32_t kUnit = kExpUnit<E>;
  up = down = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t x = (v[e / 2] >> (16 * (e % 2))) & 0xffffu;
    const uint32_t out = ((x & kExpBits<E>) + kUnit) >> 15;                  // 1: all exponent bits set
    const uint32_t nan = ((x & (kUnit - 1)) + (kUnit - 1)) / kUnit;          // 1: a fraction
    const uint32_t minus = x >> 15;
    up |= (out & (nan | (minus ^ 1u))) << e;
    down |= (out & (nan | minus)) << e;
    v[e / 2] &= ~((out * 0xffffu) << (16 * (e % 2)));
  }
  return v;
}

// Tokens of a key tile: half as many where a head is wide, for LDS and registers.
template <int D>
constexpr int tile_keys() {
  return D <= 128 ? 64 : 32;
}

// Barrier for data exchanged through LDS only: global loads stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// A uniform int32 through the scalar cache (data of earlier kernels only).
__device__ __forceinline__ int scalar_load(const int32_t* base, int64_t i) {
  return ((const __attribute__((address_space(4))) int32_t*)base)[i];
}

__device__ __forceinline__ int div_block(const KParams& p, int j) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(j)) * p.bs_mul) >> p.bs_shift);
}

// What a sequence brings to this call.
struct Seq {
  int first, n, len, pre;
};

__device__ __forceinline__ Seq make_seq(const KParams& p, int start, int end, int len, int pre) {
  Seq q;
  q.first = min(max(start, 0), p.num_tokens);
  q.n = max(min(end, p.num_tokens) - q.first, 0);
  q.len = max(min(len, p.max_len), 0);
  q.pre = min(max(pre, 0), q.len);
  return q;
}

struct LocateSmem {
  int wave_total[kTileWaves];
  int seq, local;
};

// Row tiles of a sequence: none where its few rows run in the other kernel.
__device__ __forceinline__ int row_tiles(const KParams& p, int start, int end) {
  const int first = min(max(start, 0), p.num_tokens);
  const int64_t rows = static_cast<int64_t>(max(min(end, p.num_tokens) - first, 0)) * p.group;
  return rows > p.rows_short ? static_cast<int>((rows + kTileRows - 1) / kTileRows) : 0;
}

// The sequence and its tile that hold tile `target` of all, and the number of
// tiles in all; seq = -1 past it. The whole workgroup counts, 4 sequences a
// thread and step.
__device__ __forceinline__ int locate_tile(const KParams& p, int target, LocateSmem& sm, int& seq, int& local) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  if (tid == 0) sm.seq = -1;
  int base = 0;
  for (int s0 = 0; s0 < p.num_seqs; s0 += kTileThreads * kSeqsPerThread) {
    int st[kSeqsPerThread + 1], w[kSeqsPerThread], sum = 0;
    const int s = s0 + tid * kSeqsPerThread;
#pragma unroll
    for (int i = 0; i <= kSeqsPerThread; ++i) st[i] = p.starts[min(s + i, p.num_seqs)];
#pragma unroll
    for (int i = 0; i < kSeqsPerThread; ++i) {
      w[i] = s + i < p.num_seqs ? row_tiles(p, st[i], st[i + 1]) : 0;
      sum += w[i];
    }
    int scan = sum;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int v = __shfl_up(scan, off, kWave);
      if (lane >= off) scan += v;
    }
    if (lane == kWave - 1) sm.wave_total[wave] = scan;
    lds_barrier();
    int before = base + scan - sum;
    for (int i = 0; i < kTileWaves; ++i) {
      if (i < wave) before += sm.wave_total[i];
      base += sm.wave_total[i];
    }
#pragma unroll
    for (int i = 0; i < kSeqsPerThread; ++i) {
      if (target >= before && target < before + w[i]) {
        sm.seq = s + i;
        sm.local = target - before;
      }
      before += w[i];
    }
    lds_barrier();
  }
  seq = __builtin_amdgcn_readfirstlane(sm.seq);
  local = __builtin_amdgcn_readfirstlane(sm.local);
  return base;
}

// The key tiles that some row of a workgroup sees: those of the prefix, then
// those from the window's first key on.
struct KeyTiles {
  int prefix, skip, count;  // tiles of the prefix; tiles left out behind them; tiles in all
  __device__ __forceinline__ int index(int n) const { return n < prefix ? n : n + skip; }
};

template <int TK>
__device__ __forceinline__ KeyTiles key_tiles(int pre, int lo, int hi) {
  KeyTiles k;
  k.prefix = (pre + TK - 1) / TK;
  const int first = max(k.prefix, lo / TK);
  k.skip = first - k.prefix;
  k.count = k.prefix + max((hi + TK - 1) / TK - first, 0);
  return k;
}

template <int D>
struct TileSmem {
  static constexpr int TK = tile_keys<D>();
  static constexpr int KP = D + 8;   // row pitches in elements: K rows 4 banks apart, for 16-byte reads of 16 rows;
  static constexpr int VP = D + 32;  // V rows 16 banks apart, for transpose reads of 64 bytes of 4 rows
  struct __attribute__((aligned(16))) Stage {
    uint16_t k[TK * KP];
    uint16_t v[TK * VP];
  } stage[2];
  // Infinities and NaN taken out of a stage's V rows: whether a wave's rows had
  // any, and then a bit for each column (infinity or NaN; minus infinity or NaN).
  int bad[2][kTileWaves];
  uint32_t up[2][TK][D / 32], down[2][TK][D / 32];
};

// Prompts: a workgroup takes 128 rows of one KV head, (token, query head of the
// group) pairs of one sequence, 32 a wave, and all key tiles that they see (or
// an equal part of them). Scores are formed transposed, S^T = K Q^T on
// 32x32x16 MFMAs, so that a lane holds 16 of 32 keys of one row (row l % 32,
// keys 8 (i / 4) + 4 (l / 32) + i % 4): the maximum and sum of a row need one
// exchange between two lanes, and the weights are, rounded to the dtype, the B
// operand of O^T = V^T P^T as they stand, with V^T read transposed from LDS.
// O^T has its row in the same lane again, so rescaling is a multiplication.
template <typename E, int D, bool FP8, bool BS16>
__global__ __launch_bounds__(kTileThreads) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1, D <= 128 ? 2 : 1)))
void tile_kernel(const KParams p) {
  using Smem = TileSmem<D>;
  constexpr int TK = Smem::TK, KP = Smem::KP, VP = Smem::VP;
  constexpr int KB = TK / 32;        // 32-key blocks of a tile
  constexpr int NB = D / 32;         // 32-column blocks of the output
  constexpr int KS = D / 16;         // column steps of Q.K^T
  constexpr int RW = TK / kTileWaves;  // key rows that a wave loads
  constexpr int CPR = D / 8;         // 8-element chunks of a row
  constexpr int NI = RW * CPR / kWave;
  constexpr int ELT = FP8 ? 1 : 2;
  using Chunk = typename std::conditional<FP8, u32x2, u32x4>::type;
  __shared__ Smem sm;
  __shared__ LocateSmem loc;
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int l32 = lane % 32, half = lane / 32;

  // Later tiles (long ones under a causal mask) first; the KV heads of a tile
  // next to one another, so that with 8 of them each XCD's L2 holds one head.
  const int item = static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x);
  int seq, local, parts = 1, part = 0, kv_head, total;
  if (p.split_items == 0) {
    kv_head = p.hkv - 1 - item % p.hkv;
    total = locate_tile(p, item / p.hkv, loc, seq, local);
  } else {
    // Few tiles: each over as many workgroups as make split_items in all. How
    // many tiles there are is known only now.
    total = locate_tile(p, -1, loc, seq, local);
    if (total == 0) return;
    parts = max(p.split_items / (total * p.hkv), 1);
    kv_head = p.hkv - 1 - item % p.hkv;
    part = (item / p.hkv) % parts;
    lds_barrier();
    locate_tile(p, item / p.hkv / parts, loc, seq, local);
  }
  if (seq < 0) return;
  const Seq sq = make_seq(p, scalar_load(p.starts, seq), scalar_load(p.starts, seq + 1), scalar_load(p.lens, seq),
                          p.prefix != nullptr ? scalar_load(p.prefix, seq) : 0);
  const int row0 = local * kTileRows;
  const int rows = min(sq.n * p.group - row0, kTileRows);
  // Positions of the workgroup's first and last row, and of this wave's.
  const int pos0 = sq.len - sq.n + row0 / p.group;
  const int pos1 = sq.len - sq.n + (row0 + rows - 1) / p.group;
  const int wave_row0 = min(32 * wave, rows - 1), wave_row1 = min(32 * wave + 31, rows - 1);
  const bool wave_live = 32 * wave < rows;
  const int wpos0 = sq.len - sq.n + (row0 + wave_row0) / p.group;
  const int wpos1 = sq.len - sq.n + (row0 + wave_row1) / p.group;
  const int lo = max(pos0 - p.window + 1, 0), hi = max(pos1 + 1, 0);
  const KeyTiles tiles = key_tiles<TK>(sq.pre, lo, hi);
  // This part's tiles: at least 4, but for the last one's.
  const int per = parts > 1 ? max((tiles.count + parts - 1) / parts, 4) : tiles.count;
  const int n0 = min(part * per, tiles.count), n1 = min(n0 + per, tiles.count);

  // This lane's row; rows past the last one repeat it and are not stored.
  const int row = row0 + min(32 * wave + l32, rows - 1);
  const int tok = row / p.group;
  const int q_head = kv_head * p.group + (row - tok * p.group);
  const int pos = sq.len - sq.n + tok;
  const int64_t token = sq.first + tok;
  u32x4 qf[KS];  // B operand: row l32, columns 16 s + 8 half ...
  {
    const uint16_t* src = p.q + token * p.q_st + static_cast<int64_t>(q_head) * p.q_sh + 8 * half;
    const bool wide = (reinterpret_cast<uintptr_t>(p.q) % 16 == 0) && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (wide) {
        qf[s] = *reinterpret_cast<const u32x4*>(src + 16 * s);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[s][e] = static_cast<uint32_t>(src[16 * s + 2 * e]) | static_cast<uint32_t>(src[16 * s + 2 * e + 1]) << 16;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[s][e] ^= p.q_sign;
    }
  }
  const float slope2 = p.slopes != nullptr ? p.slopes[q_head] * kLog2e : 0.0f;

  // Row and column of this lane's chunks in the wave's RW key rows.
  auto chunk_row = [&](int i) { return kWave % CPR == 0 ? lane / CPR + i * (kWave / CPR) : (lane + kWave * i) / CPR; };
  auto chunk_col = [&](int i) { return 8 * (kWave % CPR == 0 ? lane % CPR : (lane + kWave * i) % CPR); };
  Chunk rk[NI], rv[NI];

  const char* kbase = static_cast<const char*>(p.k) + ELT * (static_cast<int64_t>(kv_head) * p.k_sh);
  const char* vbase = static_cast<const char*>(p.v) + ELT * (static_cast<int64_t>(kv_head) * p.v_sh);
  const int64_t table_row = static_cast<int64_t>(seq) * p.bt_stride;
  // A key that some row of the workgroup sees.
  auto used = [&](int j) { return j < sq.pre || (j >= lo && j < hi); };
  auto page_of = [&](int t) { return min(max(t, 0), p.num_blocks - 1); };

  auto load = [&](int n) {
    const int t0 = tiles.index(n) * TK;
    const int r0 = t0 + RW * wave;
    const bool inner = t0 + TK <= sq.pre || (t0 >= lo && t0 + TK <= hi);
    if constexpr (BS16) {
      // The wave's rows lie in one cache block: one scalar table entry, one
      // resource each for K and V. Rows that no one sees read as zeros.
      const int g0 = r0 & ~15;
      const bool any = g0 < sq.pre || (g0 + 16 > lo && g0 < hi);
      const int blk = div_block(p, r0);
      const int64_t page = any ? page_of(scalar_load(p.tables, table_row + blk)) : 0;
      const int64_t off = r0 - blk * p.block_size;
      const char* kt = kbase + ELT * (page * p.k_sb + off * p.k_st);
      const char* vt = vbase + ELT * (page * p.v_sb + off * p.v_st);
      const int nrec = any ? 0x7fffffff : 0;
      const auto brk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kt), 0, nrec, kRsrcWord3);
      const auto brv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vt), 0, nrec, kRsrcWord3);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        int ko = ELT * (chunk_row(i) * p.k_st + chunk_col(i));
        int vo = ELT * (chunk_row(i) * p.v_st + chunk_col(i));
        if (!inner && !used(r0 + chunk_row(i))) ko = vo = -1;  // past num_records
        if constexpr (FP8) {
          rk[i] = __builtin_amdgcn_raw_buffer_load_b64(brk, ko, 0, 0);
          rv[i] = __builtin_amdgcn_raw_buffer_load_b64(brv, vo, 0, 0);
        } else {
          rk[i] = __builtin_amdgcn_raw_buffer_load_b128(brk, ko, 0, 0);
          rv[i] = __builtin_amdgcn_raw_buffer_load_b128(brv, vo, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int j = r0 + chunk_row(i);
        rk[i] = rv[i] = Chunk{};
        if (used(j)) {
          const int blk = div_block(p, j);
          const int64_t page = page_of(p.tables[table_row + blk]);
          const int64_t off = j - blk * p.block_size;
          rk[i] = *reinterpret_cast<const Chunk*>(kbase + ELT * (page * p.k_sb + off * p.k_st + chunk_col(i)));
          rv[i] = *reinterpret_cast<const Chunk*>(vbase + ELT * (page * p.v_sb + off * p.v_st + chunk_col(i)));
        }
      }
    }
  };
  // Every row of the workgroup sees all keys of the tile.
  auto all_see = [&](int t0) { return t0 + TK <= sq.pre || (t0 + TK - 1 <= pos0 && t0 > pos1 - p.window); };
  auto store = [&](int n, int st) {
    u32x4 v[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (FP8) v[i] = fp8x8_to<E>(rv[i]);
      else v[i] = rv[i];
    }
    if (!all_see(tiles.index(n) * TK)) {
      u16x2 open = {0xffff, 0xffff};
#pragma unroll
      for (int i = 0; i < NI; ++i) open = fold_finite<E>(open, v[i]);
      const bool bad = __any(open[0] == 0 || open[1] == 0);
      if (lane == 0) sm.bad[st][wave] = bad;
      if (bad) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          uint32_t up, down;
          v[i] = take_out<E>(v[i], up, down);
          const int r = RW * wave + chunk_row(i);
          reinterpret_cast<uint8_t*>(sm.up[st][r])[chunk_col(i) / 8] = static_cast<uint8_t>(up);
          reinterpret_cast<uint8_t*>(sm.down[st][r])[chunk_col(i) / 8] = static_cast<uint8_t>(down);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = RW * wave + chunk_row(i);
      u32x4* k = reinterpret_cast<u32x4*>(sm.stage[st].k + r * KP + chunk_col(i));
      if constexpr (FP8) *k = fp8x8_to<E>(rk[i]);
      else *k = rk[i];
      *reinterpret_cast<u32x4*>(sm.stage[st].v + r * VP + chunk_col(i)) = v[i];
    }
  };

  f32x16 acc[NB];  // O^T: row l32, columns 32 b + 8 (i / 4) + 4 half + i % 4
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = f32x16{};
  float m_ref = -__builtin_huge_valf();  // log2 units
  float l_run = 0.0f;                    // this lane's share of the row's sum

  auto compute = [&](int n, int st) {
    const int t0 = tiles.index(n) * TK;
    // Seen by no row of this wave / by all of them.
    if (!wave_live || (t0 >= sq.pre && (t0 > wpos1 || t0 + TK <= wpos0 - p.window + 1))) return;
    const bool full = t0 + TK <= sq.pre || (t0 + TK - 1 <= wpos0 && t0 > wpos1 - p.window);
    f32x16 s[KB];
    const uint16_t* kt = sm.stage[st].k + l32 * KP + 8 * half;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      s[b] = f32x16{};
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        const u32x4 ka = *reinterpret_cast<const u32x4*>(kt + 32 * b * KP + 16 * c);
        s[b] = mfma_32x32x16<E>(ka, qf[c], s[b]);
      }
    }
    float factor = p.scale2;
    if (p.softcap > 0.0f) {
      // tanh y = 1 - 2 / (e^(2y) + 1): -1 and 1 at the ends, absolute error of
      // an fp32 step of 1 near 0.
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[b][i] = p.cap2 - 2.0f * p.cap2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(s[b][i] * p.cap_in) + 1.0f);
      factor = 1.0f;
    }
    if (p.slopes != nullptr) {
      const int away0 = fresh_vgpr(pos - t0 - 4 * half);
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[b][i] = s[b][i] * factor - slope2 * static_cast<float>(abs(away0 - (32 * b + 8 * (i / 4) + i % 4)));
      factor = 1.0f;
    }
    if (!full) {
      // Past a prefix, key j is seen where 0 <= pos - j < window.
      // (fresh_vgpr: formed here, not 32 differences kept in registers across the tiles)
      const int away0 = fresh_vgpr(pos - t0 - 4 * half), to_prefix = fresh_vgpr(sq.pre - t0 - 4 * half);
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int at = 32 * b + 8 * (i / 4) + i % 4;
          const bool sees = static_cast<uint32_t>(away0 - at) < static_cast<uint32_t>(p.window) || at < to_prefix;
          s[b][i] = sees ? s[b][i] * factor : -__builtin_huge_valf();
          if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // few lane masks at a time
        }
      factor = 1.0f;
    }
    float top = -__builtin_huge_valf();
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
    {
      const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    }
    top *= factor;
    // The reference maximum follows only when a tile passes it by 2^8.
    if (__any(top > m_ref + 8.0f)) {
      const float m_new = fmaxf(m_ref, top);
      const float alpha = __builtin_amdgcn_exp2f(m_ref - (m_new == -__builtin_huge_valf() ? 0.0f : m_new));
      m_ref = m_new;
      l_run *= alpha;
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= alpha;
    }
    const float ref = m_ref == -__builtin_huge_valf() ? 0.0f : m_ref;  // nothing seen yet
    u32x4 pk[2 * KB];  // B operand: row l32, 16 keys a step
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float x = __builtin_amdgcn_exp2f(s[b][i] * factor - ref);
        const float y = __builtin_amdgcn_exp2f(s[b][i + 1] * factor - ref);
        l_run += x + y;
        pk[2 * b + i / 8][(i % 8) / 2] = pack2<E>(x, y);
      }
    const uint16_t* vt = sm.stage[st].v + (4 * half + (lane % 16) / 4) * VP + 16 * ((lane / 16) % 2) + 4 * (lane % 4);
    // A operand of O^T: columns 32 b + l32, the 16 keys of step c in the order of pk[c].
    auto v_operand = [&](int c, int b) {
      using lds_v4i16 = __attribute__((address_space(3))) s16x4;
      const u32x2 x = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + 16 * c * VP + 32 * b)));
      const u32x2 y = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + (16 * c + 8) * VP + 32 * b)));
      return u32x4{x[0], x[1], y[0], y[1]};
    };
#pragma unroll
    for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = mfma_32x32x16<E>(v_operand(c, b), pk[c], acc[b]);
    if (all_see(t0)) return;
    int bad = 0;
#pragma unroll
    for (int w = 0; w < kTileWaves; ++w) bad |= sm.bad[st][w];
    if (__builtin_amdgcn_readfirstlane(bad) == 0) return;
    // Infinities and NaN among values that not every row sees: a row takes
    // those whose key has a weight there (0 x infinity would be NaN). Key
    // 8 (e / 4) + 4 half + e % 4 of a 16-key step is element e of its half.
    uint32_t up[NB] = {}, down[NB] = {};
#pragma unroll 1
    for (int j = 0; j < TK; ++j) {
      if (__builtin_amdgcn_readfirstlane(sm.bad[st][j / RW]) == 0) continue;
      const int e = j % 4 + 4 * ((j % 16) / 8);
      uint32_t word = 0;
#pragma unroll
      for (int c = 0; c < 2 * KB; ++c) {
        if (c != j / 16) continue;
#pragma unroll
        for (int w = 0; w < 4; ++w) word |= w == e / 2 ? pk[c][w] : 0u;
      }
      word = e % 2 != 0 ? word >> 16 : word & 0xffffu;
      const uint32_t takes = __shfl(word, l32 + 32 * ((j / 4) % 2), kWave) != 0 ? 0xffffffffu : 0u;
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        up[b] |= sm.up[st][j][b] & takes;
        down[b] |= sm.down[st][j][b] & takes;
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int u = static_cast<int>(up[b] >> (4 * half)), d = static_cast<int>(down[b] >> (4 * half));
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        constexpr int kInf = 0x7f800000;
        const int at = 31 - (8 * (i / 4) + i % 4);
        acc[b][i] += __int_as_float(((u << at) >> 31) & kInf);
        acc[b][i] -= __int_as_float(((d << at) >> 31) & kInf);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  if (n0 < n1) {
    load(n0);
    store(n0, 0);
    lds_barrier();
    for (int n = n0; n < n1; ++n) {
      const int st = (n - n0) & 1;
      if (n + 1 < n1) load(n + 1);
      compute(n, st);
      if (n + 1 < n1) store(n + 1, st ^ 1);
      lds_barrier();
    }
  }

  {
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
    l_run = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
  if (32 * wave + l32 >= rows) return;
  if (parts > 1) {
    // Partial results: sums against m_ref, joined by tile_join_kernel.
    const int64_t slot = ((static_cast<int64_t>(item / p.hkv / parts) * p.hkv + kv_head) * parts + part) * kTileRows +
                         32 * wave + l32;
    float* dst = p.ws + slot * (D + 2);
    if (half == 0) {
      dst[D] = m_ref;
      dst[D + 1] = l_run;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) dst[32 * b + 8 * (i / 4) + 4 * half + i % 4] = acc[b][i];
    return;
  }
  const float inv = l_run == 0.0f ? 0.0f : p.v_scale / l_run;
  uint16_t* dst = p.out + token * p.o_st + static_cast<int64_t>(q_head) * p.o_sh + 4 * half;
  const bool wide = (reinterpret_cast<uintptr_t>(p.out) % 8 == 0) && p.o_st % 4 == 0 && p.o_sh % 4 == 0;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = l_run == 0.0f ? 0.0f : acc[b][4 * g + i] * inv;
      if (wide) {
        *reinterpret_cast<u32x2*>(dst + 32 * b + 8 * g) = u32x2{pack2<E>(y[0], y[1]), pack2<E>(y[2], y[3])};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[32 * b + 8 * g + i] = E::from_float(y[i]);
      }
    }
}

template <typename E, int D, bool FP8>
hipError_t launch_tiles(const KParams& kp, hipStream_t s) {
  // At most this many row tiles: full ones, and one more a sequence (at least 17 rows each).
  const int64_t rows = static_cast<int64_t>(kp.num_tokens) * kp.group;
  const int64_t more = std::min<int64_t>(kp.num_seqs, rows / (kp.rows_short + 1));
  const int64_t bound = rows / kTileRows + more;
  const dim3 grid(static_cast<unsigned>(bound * kp.hkv)), block(kTileThreads);
  const int64_t reach = int64_t{16} * 2 * std::max(kp.k_st, kp.v_st);
  if (kp.block_size % 16 == 0 && reach < (int64_t{1} << 31))
    hipLaunchKernelGGL((tile_kernel<E, D, FP8, true>), grid, block, 0, s, kp);
  else hipLaunchKernelGGL((tile_kernel<E, D, FP8, false>), grid, block, 0, s, kp);
  return hipGetLastError();
}

template <typename E>
hipError_t launch(const KParams& kp, int d, int max_query_len, bool fp8, hipStream_t s) {
  if (static_cast<int64_t>(max_query_len) * kp.group > kp.rows_short) {
    hipError_t e = hipSuccess;
    if (fp8) {
      switch (d) {
        case 64: e = launch_tiles<E, 64, true>(kp, s); break;
        case 128: e = launch_tiles<E, 128, true>(kp, s); break;
        case 192: e = launch_tiles<E, 192, true>(kp, s); break;
        default: e = launch_tiles<E, 256, true>(kp, s); break;
      }
    } else {
      switch (d) {
        case 64: e = launch_tiles<E, 64, false>(kp, s); break;
        case 96: e = launch_tiles<E, 96, false>(kp, s); break;
        case 128: e = launch_tiles<E, 128, false>(kp, s); break;
        case 192: e = launch_tiles<E, 192, false>(kp, s); break;
        default: e = launch_tiles<E, 256, false>(kp, s); break;
      }
    }
    if (e != hipSuccess) return e;
  }
  const dim3 grid(static_cast<unsigned>(kp.num_tokens * kp.hq)), block(kWave);
  if (fp8) hipLaunchKernelGGL((simple_kernel<E, true>), grid, block, 0, s, kp, d);
  else hipLaunchKernelGGL((simple_kernel<E, false>), grid, block, 0, s, kp, d);
  return hipGetLastError();
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
  kp.window = a->window == 0 || a->window > max_len ? (max_len > 0 ? max_len : 1) : a->window;
  kp.scale = a->scale;
  kp.softcap = a->softcap;
  kp.k_scale = k_scale;
  kp.v_scale = v_scale;
  (void)workspace, (void)workspace_bytes;
  kp.hkv = a->num_kv_heads;
  kp.rows_short = 16;
  // floor(j / b) = (j * ceil(2^k / b)) >> k for j < 2^31 with k = 31 + ceil(log2 b):
  // the factor is off by less than 1, the product by less than 2^31 <= 2^k / b.
  int k = 31;
  while ((int64_t{1} << (k - 31)) < a->block_size) ++k;
  kp.bs_shift = k;
  kp.bs_mul = static_cast<uint32_t>(((uint64_t{1} << k) + a->block_size - 1) / a->block_size);
  const float c = kp.scale * kp.k_scale;
  kp.q_sign = c < 0.0f ? 0x80008000u : 0u;
  kp.scale2 = std::fabs(c) * kLog2e;
  kp.cap2 = kp.softcap * kLog2e;
  kp.cap_in = kp.softcap > 0.0f ? 2.0f * kLog2e * std::fabs(c) / kp.softcap : 0.0f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return static_cast<int>(dtype == DK_BFLOAT16 ? launch<Bf16>(kp, head_dim, max_query_len, fp8, s)
                                               : launch<F16>(kp, head_dim, max_query_len, fp8, s));
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
