// Attention of the new tokens of a ragged batch over a paged KV cache (gfx950):
// sequence s brings query tokens [start[s], start[s + 1]), the last ones of its
// seq_lens[s] cached tokens, one of them (decode) or thousands (a prompt).
//
//   x_ij = scale * q_i . k_j,  capped to  cap * tanh(x_ij / cap),
//   less slope_h * |i - j|,  over the keys j that token i sees:
//   j <= i and j > i - window, or j < prefix_s;
//   out_i = sum_j softmax_j(x_ij) v_j,  zeros where it sees no key.
#pragma once

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
  int hkv;
  int split_items;         // tile_work: workgroups that the tiles of a call may be split over; 0: never split
  int shares;              // row_work: workgroups a KV head, of equal shares of all key tiles; 0: one a sequence
  int tile_groups;         // workgroups of tile_work
  int row_from;            // the first workgroup of row_work
  int short_rows;          // rows of a KV head up to which a sequence runs in row_work: 16 or 32
  int slot_rows;           // row_work: rows of a slot, as many as max_query_len allows
  // Partial results, row by row of an item or slot: sums, and their reference
  // maximum (log2 units) and exp-sum.
  float *tile_ws, *tile_ml, *ws, *ws_ml;
  int32_t* ws_first;       // row_work: a sequence's first workgroup, and how many
  uint32_t bs_mul;         // j / block_size = (j * bs_mul) >> bs_shift, for j < 2^31
  int bs_shift;
  int biased;              // slopes are given
  float v_scale;           // of an fp8 cache (1 otherwise)
  // In log2 units: the cap (0: none) and the positive factor of q.k, whose sign
  // goes to q: the score's, or with a cap that of the exponent of e^(2 y) in
  // tanh y = 1 - 2 / (e^(2 y) + 1).
  float cap2, scale2;
  uint32_t q_sign;
};

// The kernel's arguments, to be loaded where they are used: an argument that
// the compiler sees only here does not stay in scalar registers around it.
// KParams is the one parameter, at the start of the argument segment.
typedef const __attribute__((address_space(4))) KParams Args;
__device__ __forceinline__ Args& fresh_args() {
  auto a = (Args*)__builtin_amdgcn_kernarg_segment_ptr();
  __asm__ volatile("" : "+s"(a));
  return *a;
}

// 8 e4m3fn bytes as 8 elements of E, exactly (scale 1; every e4m3fn value is
// one of E).
template <typename E>
__device__ __forceinline__ u32x4 fp8x8_to(u32x2 w) {
  u32x4 out;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (std::is_same<E, Bf16>::value) {
      out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, false));
      out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], 1.0f, true));
    } else {
      out[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, false));
      out[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], 1.0f, true));
    }
  }
  return out;
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
constexpr int kRsrcWord3 = 0x00020000;      // word 3 of a gfx9-family buffer resource for raw loads
constexpr int kSeqsPerThread = 4;
// Sequences of few rows are not cut up to so many keys: the joining launch costs
// more than it gives. Nor up to kWholeKeysMany where kManyPairs (sequence, KV
// head) pairs fill the CUs by themselves: 32 sequences of 100-900 keys, 8 KV
// heads, 31.7 us cut and 25.2 whole (cold); 29 of 1-1800 keys 36.4 and 33.3.
constexpr int kWholeKeys = 512, kWholeKeysMany = 2048, kManyPairs = 192;
// Key tiles that a workgroup takes at least (7 pairs x 2 heads of 71-569 keys,
// head_dim 256: 25.2 us with 16, 21.9 with 8), and by which an equal part of a
// sequence may be longer than an equal share of all, for the sake of one piece a
// workgroup (48 speculating sequences of 200-8000 keys: 66.8 us with 8, 62.5 with
// 32; twice the share is too many: 32 sequences of 500-8000 keys 105 and 134 us).
constexpr int kMinShare = 8, kMorePart = 32;
// Key tiles of a part of a row tile at least, so that its sums' way through
// memory stays small against it. (4, 8 and 16 measured the same within 1% at a
// 512-token chunk on 16000 keys and beside 32 decoding sequences.)
constexpr int kMinPart = 8;
constexpr int kWideRows = 192;  // head_dim up to which 32 rows share a reading: 256 has no registers for them

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

// Rows, (token, query head of the group) pairs, of a wave of tile_work: 32, or
// 16 where a head is wide and the sums of 32 would leave one wave a SIMD (nine
// ragged prompts, head_dim 256: 376 us with 32 rows, 286 with 16).
constexpr int wave_rows(int d) { return d <= 128 ? 32 : 16; }
constexpr int tile_rows(int d) { return kTileWaves * wave_rows(d); }

// All ones where key j lies in [0, pre) or [lo, hi), else 0. (By sign bits:
// comparisons would put a lane mask into scalar registers for every load, and
// short cuts branches that wait for the loads before them.)
__device__ __forceinline__ int in_ranges(int j, int pre, int lo, int hi) {
  return ((j - pre) | ((lo - 1 - j) & (j - hi))) >> 31;
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

template <typename Params>
__device__ __forceinline__ int div_block(const Params& p, int j) {
  return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(j)) * p.bs_mul) >> p.bs_shift);
}

// cap tanh(y) in log2 units, for a product q.k: tanh y = 1 - 2 / (e^(2 y) + 1)
// has the right ends and an absolute error of some 2^-23, a few 1e-5 of a score
// under caps up to kExactCap. Larger ones take tanh's series where |y| < 0.1.
constexpr float kExactCap = 64.0f;
template <bool LARGE, typename Params>
__device__ __forceinline__ float capped(const Params& p, float product) {
  const float z = product * p.scale2;  // 2 y log2 e
  const float t = p.cap2 - 2.0f * p.cap2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(z) + 1.0f);
  if constexpr (!LARGE) return t;
  const float y = z * (0.5f / kLog2e), y2 = y * y;
  const float series = p.cap2 * y * (1.0f + y2 * (-1.0f / 3.0f + y2 * (2.0f / 15.0f - y2 * (17.0f / 315.0f))));
  return fabsf(y) < 0.1f ? series : t;
}

// What a sequence brings to this call.
struct Seq {
  int first, n, len, pre;
};

template <typename Params>
__device__ __forceinline__ Seq make_seq(const Params& p, int start, int end, int len, int pre) {
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

// 4 columns of an output row, rounded; in one store where rows are 8-byte aligned.
template <typename E, typename Params>
__device__ __forceinline__ void store4(const Params& p, uint16_t* dst, f32x4 y) {
  if ((reinterpret_cast<uintptr_t>(p.out) % 8 == 0) && p.o_st % 4 == 0 && p.o_sh % 4 == 0) {
    *reinterpret_cast<u32x2*>(dst) = u32x2{pack2<E>(y[0], y[1]), pack2<E>(y[2], y[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = E::from_float(y[i]);
  }
}

// Row tiles of a sequence: none where its few rows run in row_work.
template <int D>
__device__ __forceinline__ int row_tiles(Args& p, int start, int end) {
  const int first = min(max(start, 0), p.num_tokens);
  const int64_t rows = static_cast<int64_t>(max(min(end, p.num_tokens) - first, 0)) * p.group;
  return rows > p.short_rows ? static_cast<int>((rows + tile_rows(D) - 1) / tile_rows(D)) : 0;
}

// Prefix sums over sequences, 4 a thread: of the thread's units w, from `base`
// on, to `before`; returns the units in all.
__device__ __forceinline__ int scan_units(int base, LocateSmem& sm, const int (&w)[kSeqsPerThread],
                                          int (&before)[kSeqsPerThread]) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kSeqsPerThread; ++i) sum += w[i];
  int scan = sum;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int v = __shfl_up(scan, off, kWave);
    if (lane >= off) scan += v;
  }
  lds_barrier();  // the last scan's totals and find have been read
  if (lane == kWave - 1) sm.wave_total[wave] = scan;
  if (tid == 0) sm.seq = -1;
  lds_barrier();
  int at = base + scan - sum, total = 0;
#pragma unroll
  for (int i = 0; i < kTileWaves; ++i) {
    if (i < wave) at += sm.wave_total[i];
    total += sm.wave_total[i];
  }
#pragma unroll
  for (int i = 0; i < kSeqsPerThread; ++i) {
    before[i] = at;
    at += w[i];
  }
  return __builtin_amdgcn_readfirstlane(total);
}

// weight(s) units a sequence; plan(total) is then told how many there are, and
// says whether units(w) parts of a sequence are counted instead of its w units.
// target() names one of them: the sequence that holds it and which one of the
// sequence's it is (seq = -1: past the last).
template <typename Weight, typename PlanFn, typename Units, typename Target>
__device__ __forceinline__ void locate(int num_seqs, LocateSmem& sm, Weight weight, PlanFn plan, Units units,
                                       Target target, int& seq, int& local) {
  constexpr int kStep = kTileThreads * kSeqsPerThread;
  const int mine = static_cast<int>(threadIdx.x) * kSeqsPerThread;
  const bool one = num_seqs <= kStep;  // one step: the units stay in registers
  int w[kSeqsPerThread], before[kSeqsPerThread];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < kSeqsPerThread; ++i) w[i] = s0 + mine + i < num_seqs ? weight(s0 + mine + i) : 0;
  };
  int total = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += kStep) {
    load(s0);
    total += scan_units(total, sm, w, before);
  }
  const bool parts = plan(total);
  const int want = target();
  int base = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += kStep) {
    if (!one) load(s0);
    if (parts) {
#pragma unroll
      for (int i = 0; i < kSeqsPerThread; ++i) w[i] = units(w[i]);
    }
    if (!one || parts) base += scan_units(base, sm, w, before);  // else `before` still holds
#pragma unroll
    for (int i = 0; i < kSeqsPerThread; ++i) {
      if (want >= before[i] && want < before[i] + w[i]) {
        sm.seq = s0 + mine + i;
        sm.local = want - before[i];
      }
    }
    if (!one && want < base) break;
  }
  lds_barrier();
  seq = __builtin_amdgcn_readfirstlane(sm.seq);
  local = __builtin_amdgcn_readfirstlane(sm.local);
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

// A row tile of a sequence: its rows, the positions of the first and the last,
// the keys that some row sees besides the prefix, and the key tiles that hold them.
template <int D>
struct RowTile {
  int row0, rows, pos0, pos1, lo, hi;
  KeyTiles tiles;
  __device__ __forceinline__ RowTile(Args& p, const Seq& sq, int local) {
    row0 = local * tile_rows(D);
    rows = min(sq.n * p.group - row0, tile_rows(D));
    pos0 = sq.len - sq.n + row0 / p.group;
    pos1 = sq.len - sq.n + (row0 + rows - 1) / p.group;
    lo = max(pos0 - p.window + 1, 0);
    hi = max(pos1 + 1, 0);
    tiles = key_tiles<tile_keys<D>()>(sq.pre, lo, hi);
  }
  // Key tiles of one of `parts` parts.
  __device__ __forceinline__ int per_part(int parts) const {
    return parts > 1 ? max((tiles.count + parts - 1) / parts, kMinPart) : tiles.count;
  }
};

// Workgroups over which the key tiles of a row tile are spread, so that all
// make up to split_items.
__device__ __forceinline__ int parts_of(Args& p, int total) {
  return p.split_items > 0 && total > 0 ? max(p.split_items / (total * p.hkv), 1) : 1;
}

template <int D>
struct TileSmem {
  static constexpr int TK = tile_keys<D>();
  // Rows lie next to one another (loads straight to LDS fill 1 KB in lane order),
  // with the 16-byte chunk c of row r in the place of c ^ k_swap(r), c ^ v_swap(r):
  // reads of one chunk of 16 K rows, and transpose reads of 64 (32) bytes of 4 (8)
  // V rows, take all 64 banks.
  static constexpr int M = D / 8 % 16 == 0 ? 16 : D / 8 % 8 == 0 ? 8 : 4;  // chunks a swap stays within
  static constexpr int G = wave_rows(D) / 8;                               // chunks of a transpose read
  static __device__ __forceinline__ int k_swap(int r) { return r / (16 / M) % M; }
  static __device__ __forceinline__ int v_swap(int r) { return r / (16 / M) % (M / G) * G; }
  struct __attribute__((aligned(16))) Stage {
    uint16_t k[TK * D];
    uint16_t v[TK * D];
  } stage[2];
  // Infinities and NaN taken out of a stage's V rows: whether a wave's rows had
  // any, and then a bit for each column (infinity or NaN; minus infinity or NaN).
  int bad[2][kTileWaves];
  uint32_t up[2][TK][D / 32], down[2][TK][D / 32];
  LocateSmem loc;
};

// Prompts: a workgroup takes 128 rows (64 of wide heads) of one KV head, (token,
// query head of the group) pairs of one sequence, 32 (16) a wave, and all key
// tiles that they see (or an equal part of them). Scores are formed transposed,
// S^T = K Q^T on 32x32x16 (16x16x32) MFMAs, so that a lane holds keys
// 8 g + 4 part + i of one row, g and i its elements, part = lane / 32 (16): the
// maximum and sum of a row need one exchange (two), and the weights are, rounded
// to the dtype, the B operand of O^T = V^T P^T as they stand, with V^T read
// transposed from LDS. O^T has its row in the same lane again, so rescaling is
// a multiplication. Two key tiles are in LDS: one under the products, the next
// on its way.
//
// Bound by a wave's own chain of products, exponentials and LDS reads at two
// waves a SIMD (LDS and registers allow no third): at two prompts of 8192 tokens,
// 32 / 8 heads of 128, the matrix units are busy 49% of the time, the vector units 47%
// and LDS 25%; 1.11 ms, 987 TFLOP/s of the 1360 that a large product reaches.
// Heads of 256: 0.25 ms for nine prompts of 134 GFLOP (vector units 41%, LDS 26%,
// matrix units 25%).
template <typename E, int D>
struct TileMath {
  static constexpr int WR = wave_rows(D);
  typedef float acc_t __attribute__((ext_vector_type(WR == 32 ? 16 : 4)));
  static __device__ __forceinline__ acc_t mma(u32x4 a, u32x4 b, acc_t c) {
    if constexpr (WR == 32) return mfma_32x32x16<E>(a, b, c);
    else return E::mfma_16x16x32(a, b, c);
  }
  // Over the lanes that hold a row.
  static __device__ __forceinline__ float row_max(float v) {
    if constexpr (WR == 16) return rows_max(v);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  }
  static __device__ __forceinline__ float row_sum(float v) {
    if constexpr (WR == 16) return rows_sum(v);
    const auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(x[0]) + __uint_as_float(x[1]);
  }
};

template <typename E, int D, bool FP8, bool BS16>
__device__ __forceinline__ void tile_work(Args& p, TileSmem<D>& sm) {
  using Smem = TileSmem<D>;
  constexpr int TK = Smem::TK, G = Smem::G;
  using Math = TileMath<E, D>;
  using Acc = typename Math::acc_t;
  constexpr int WR = Math::WR;
  constexpr int NE = WR == 32 ? 16 : 4;  // elements of a lane in an accumulator
  constexpr int KB = TK / WR;        // key blocks of a tile
  constexpr int NB = D / WR;         // column blocks of the output
  constexpr int CS = 8 * (kWave / WR);  // columns of a step of Q.K^T, and keys of one of P.V
  constexpr int KS = D / CS;
  constexpr int PS = TK / CS;
  constexpr int RW = TK / kTileWaves;  // key rows that a wave loads
  constexpr int CPR = D / 8;         // 8-element chunks of a row
  constexpr int NI = RW * CPR / kWave;
  constexpr int ELT = FP8 ? 1 : 2;
  using Chunk = typename std::conditional<FP8, u32x2, u32x4>::type;
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int lr = lane % WR, part4 = 4 * (lane / WR);

  // Later tiles (long ones under a causal mask) first; the KV heads of a tile
  // next to one another, so that with 8 of them each XCD's L2 holds one head.
  const int item = p.tile_groups - 1 - static_cast<int>(blockIdx.x);
  const int kv_head = p.hkv - 1 - item % p.hkv;
  // With few tiles each goes over as many workgroups as make split_items in
  // all; how many tiles there are is known only now.
  int seq, local, parts = 1;
  locate(
      p.num_seqs, sm.loc, [&](int s) { return row_tiles<D>(p, p.starts[s], p.starts[s + 1]); },
      [&](int total) {
        parts = parts_of(p, total);
        return false;
      },
      [](int w) { return w; }, [&] { return item / p.hkv / parts; }, seq, local);
  const int part = item / p.hkv % parts;
  if (seq < 0) return;
  const Seq sq = make_seq(p, scalar_load(p.starts, seq), scalar_load(p.starts, seq + 1), scalar_load(p.lens, seq),
                          p.prefix != nullptr ? scalar_load(p.prefix, seq) : 0);
  const RowTile<D> rt(p, sq, local);
  const int row0 = rt.row0, rows = rt.rows, pos0 = rt.pos0, pos1 = rt.pos1, lo = rt.lo, hi = rt.hi;
  const KeyTiles tiles = rt.tiles;
  const int per = rt.per_part(parts);
  const int n0 = min(part * per, tiles.count), n1 = min(n0 + per, tiles.count);
  if (parts > 1 && part > 0 && n0 == n1) return;  // fewer parts than asked for
  // Positions of this wave's first and last row.
  const int wave_row0 = min(WR * wave, rows - 1), wave_row1 = min(WR * wave + WR - 1, rows - 1);
  const bool wave_live = WR * wave < rows;
  const int wpos0 = sq.len - sq.n + (row0 + wave_row0) / p.group;
  const int wpos1 = sq.len - sq.n + (row0 + wave_row1) / p.group;
  // This lane's row; rows past the last one repeat it and are not stored.
  const int row = row0 + min(WR * wave + lr, rows - 1);
  const int tok = row / p.group;
  const int q_head = kv_head * p.group + (row - tok * p.group);
  const int pos = sq.len - sq.n + tok;
  const int64_t token = sq.first + tok;
  u32x4 qf[KS];  // B operand: row lr, columns CS s + 2 part4 ...
  {
    const uint16_t* src = p.q + token * p.q_st + static_cast<int64_t>(q_head) * p.q_sh + 2 * part4;
    const bool wide = (reinterpret_cast<uintptr_t>(p.q) % 16 == 0) && p.q_st % 8 == 0 && p.q_sh % 8 == 0;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if (wide) {
        qf[s] = *reinterpret_cast<const u32x4*>(src + CS * s);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          qf[s][e] = static_cast<uint32_t>(src[CS * s + 2 * e]) | static_cast<uint32_t>(src[CS * s + 2 * e + 1]) << 16;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) qf[s][e] ^= p.q_sign;
    }
  }
  const float slope2 = p.slopes != nullptr ? p.slopes[q_head] * kLog2e : 0.0f;

  // Row and column of this lane's chunks in the wave's RW key rows.
  auto chunk_row = [&](int i) { return kWave % CPR == 0 ? lane / CPR + i * (kWave / CPR) : (lane + kWave * i) / CPR; };
  auto chunk_col = [&](int i) { return 8 * (kWave % CPR == 0 ? lane % CPR : (lane + kWave * i) % CPR); };
  // The columns that belong there.
  auto k_col = [&](int i) { return chunk_col(i) ^ 8 * Smem::k_swap(RW * wave + chunk_row(i)); };
  auto v_col = [&](int i) { return chunk_col(i) ^ 8 * Smem::v_swap(RW * wave + chunk_row(i)); };
  // Tiles go to LDS past the registers where 16 keys lie in one cache block and
  // need no conversion (cold, through registers and past them: two prompts of 8192
  // tokens 1157 and 1091 us, four of 2000 with heads of 256 260 and 223).
  constexpr bool DIRECT = BS16 && !FP8;
  Chunk rk[NI], rv[NI];

  const char* kbase = static_cast<const char*>(p.k) + ELT * (static_cast<int64_t>(kv_head) * p.k_sh);
  const char* vbase = static_cast<const char*>(p.v) + ELT * (static_cast<int64_t>(kv_head) * p.v_sh);
  const int64_t table_row = static_cast<int64_t>(seq) * p.bt_stride;
  // A key that some row of the workgroup sees.
  auto used = [&](int j) { return in_ranges(j, sq.pre, lo, hi); };
  auto page_of = [&](int t) { return min(max(t, 0), p.num_blocks - 1); };

  auto load = [&](int n, [[maybe_unused]] typename Smem::Stage* to) {
    const int t0 = tiles.index(n) * TK;
    const int r0 = t0 + RW * wave;
    const int all = t0 + TK <= sq.pre || (t0 >= lo && t0 + TK <= hi) ? -1 : 0;  // every key of the tile
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
      int hide[NI] = {};  // -1 (past num_records: zeros) for rows that no one sees
      if (all == 0) {
#pragma unroll
        for (int i = 0; i < NI; ++i) hide[i] = ~used(r0 + chunk_row(i));
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int ko = hide[i] | ELT * (chunk_row(i) * p.k_st + k_col(i));
        const int vo = hide[i] | ELT * (chunk_row(i) * p.v_st + v_col(i));
        if constexpr (DIRECT) {
          using lds_ptr = __attribute__((address_space(3))) void*;
          const int at = RW * wave * D + 8 * kWave * i;  // and 16 bytes a lane from there
          __builtin_amdgcn_raw_ptr_buffer_load_lds(brk, (lds_ptr)(to->k + at), 16, ko, 0, 0, 0);
          __builtin_amdgcn_raw_ptr_buffer_load_lds(brv, (lds_ptr)(to->v + at), 16, vo, 0, 0, 0);
        } else {
          rk[i] = __builtin_amdgcn_raw_buffer_load_b64(brk, ko, 0, 0);
          rv[i] = __builtin_amdgcn_raw_buffer_load_b64(brv, vo, 0, 0);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int j = r0 + chunk_row(i);
        rk[i] = rv[i] = Chunk{};
        if (used(j) != 0) {
          const int blk = div_block(p, j);
          const int64_t page = page_of(p.tables[table_row + blk]);
          const int64_t off = j - blk * p.block_size;
          rk[i] = *reinterpret_cast<const Chunk*>(kbase + ELT * (page * p.k_sb + off * p.k_st + k_col(i)));
          rv[i] = *reinterpret_cast<const Chunk*>(vbase + ELT * (page * p.v_sb + off * p.v_st + v_col(i)));
        }
      }
    }
  };
  // Every row of the workgroup sees all keys of the tile.
  auto all_see = [&](int t0) { return t0 + TK <= sq.pre || (t0 + TK - 1 <= pos0 && t0 > pos1 - p.window); };
  auto store = [&](int n, int st) {
    const bool look = !all_see(tiles.index(n) * TK);
    auto place = [&](uint16_t* stage, int i) {
      return reinterpret_cast<u32x4*>(stage + (RW * wave + chunk_row(i)) * D + chunk_col(i));
    };
    u32x4 v[NI];
    if constexpr (DIRECT) {
      __builtin_amdgcn_s_waitcnt((7 << 4) | (15 << 8));  // vmcnt(0): this wave's rows are in LDS
      if (!look) return;
#pragma unroll
      for (int i = 0; i < NI; ++i) v[i] = *place(sm.stage[st].v, i);
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        if constexpr (FP8) v[i] = fp8x8_to<E>(rv[i]);
        else v[i] = rv[i];
      }
    }
    if (look) {
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
          reinterpret_cast<uint8_t*>(sm.up[st][r])[v_col(i) / 8] = static_cast<uint8_t>(up);
          reinterpret_cast<uint8_t*>(sm.down[st][r])[v_col(i) / 8] = static_cast<uint8_t>(down);
          if constexpr (DIRECT) *place(sm.stage[st].v, i) = v[i];
        }
      }
    }
    if constexpr (DIRECT) return;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if constexpr (FP8) *place(sm.stage[st].k, i) = fp8x8_to<E>(rk[i]);
      else *place(sm.stage[st].k, i) = rk[i];
      *place(sm.stage[st].v, i) = v[i];
    }
  };

  Acc acc[NB];  // O^T: row lr, columns WR b + 8 (i / 4) + part4 + i % 4
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = Acc{};
  float m_ref = -__builtin_huge_valf();  // log2 units
  float l_run = 0.0f;                    // this lane's share of the row's sum

  auto compute = [&](int n, int st, const typename Smem::Stage* from) {
    const int t0 = tiles.index(n) * TK;
    // Seen by no row of this wave / by all of them.
    if (!wave_live || (t0 >= sq.pre && (t0 > wpos1 || t0 + TK <= wpos0 - p.window + 1))) return;
    const bool full = t0 + TK <= sq.pre || (t0 + TK - 1 <= wpos0 && t0 > wpos1 - p.window);
    Acc s[KB];
    const uint16_t* kt = from->k + lr * D;
    const int kc = 2 * part4 ^ 8 * Smem::k_swap(lr);
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      s[b] = Acc{};
#pragma unroll
      for (int c = 0; c < KS; ++c) {
        const u32x4 ka = *reinterpret_cast<const u32x4*>(kt + WR * b * D + (CS * c ^ kc));
        s[b] = Math::mma(ka, qf[c], s[b]);
      }
    }
    // 8 K reads ahead of the products (left alone, the compiler keeps 2, and each
    // pair of products waits for LDS: 1212 against 1179 us for two prompts of
    // 8192 tokens).
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
    for (int x = 0; x < KB * KS - 8; ++x) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, 8, 0);
    float factor = p.scale2;
    if (p.cap2 > 0.0f) {
      if (p.cap2 <= kExactCap * kLog2e) {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int i = 0; i < NE; ++i) s[b][i] = capped<false>(p, s[b][i]);
      } else {
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
          for (int i = 0; i < NE; ++i) s[b][i] = capped<true>(p, s[b][i]);
      }
      factor = 1.0f;
    }
    if (p.slopes != nullptr) {
      const int away0 = fresh_vgpr(pos - t0 - part4);
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < NE; ++i)
          s[b][i] = s[b][i] * factor - slope2 * static_cast<float>(abs(away0 - (WR * b + 8 * (i / 4) + i % 4)));
      factor = 1.0f;
    }
    if (!full) {
      // Past a prefix, key j is seen where 0 <= pos - j < window.
      // (fresh_vgpr: formed here, not 32 differences kept in registers across the tiles)
      const int away0 = fresh_vgpr(pos - t0 - part4), to_prefix = fresh_vgpr(sq.pre - t0 - part4);
#pragma unroll
      for (int b = 0; b < KB; ++b)
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          const int at = WR * b + 8 * (i / 4) + i % 4;
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
      for (int i = 0; i < NE; ++i) top = fmaxf(top, s[b][i]);
    top = Math::row_max(top);
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
        for (int i = 0; i < NE; ++i) acc[b][i] *= alpha;
    }
    const float ref = m_ref == -__builtin_huge_valf() ? 0.0f : m_ref;  // nothing seen yet
    u32x4 pk[PS];  // B operand: row lr, CS keys a step
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < NE; i += 2) {
        const float x = __builtin_amdgcn_exp2f(s[b][i] * factor - ref);
        const float y = __builtin_amdgcn_exp2f(s[b][i + 1] * factor - ref);
        l_run += x + y;
        pk[(NE * b + i) / 8][(NE * b + i) % 8 / 2] = pack2<E>(x, y);
      }
    const int vr = part4 + (lane % 16) / 4, vc = 8 * Smem::v_swap(vr);
    const uint16_t* vt = from->v + vr * D + (WR == 32 ? 16 * ((lane / 16) % 2) : 0) + 4 * (lane % 4);
    // A operand of O^T: columns WR b + lr, the keys of step c in the order of pk[c].
    auto v_operand = [&](int c, int b) {
      using lds_v4i16 = __attribute__((address_space(3))) s16x4;
      const u32x2 x = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + CS * c * D + (WR * b ^ vc))));
      const u32x2 y = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + (CS * c + CS / 2) * D + (WR * b ^ vc))));
      return u32x4{x[0], x[1], y[0], y[1]};
    };
#pragma unroll
    for (int c = 0; c < PS; ++c)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = Math::mma(v_operand(c, b), pk[c], acc[b]);
    if (all_see(t0)) return;
    int bad = 0;
#pragma unroll
    for (int w = 0; w < kTileWaves; ++w) bad |= sm.bad[st][w];
    if (__builtin_amdgcn_readfirstlane(bad) == 0) return;
    // Infinities and NaN among values that not every row sees: a row takes
    // those whose key has a weight there (0 x infinity would be NaN).
    uint32_t up[D / 32] = {}, down[D / 32] = {};
#pragma unroll 1
    for (int j = 0; j < TK; ++j) {
      if (__builtin_amdgcn_readfirstlane(sm.bad[st][j / RW]) == 0) continue;
      // Key j is element `at` of the lanes of part (j % WR / 4) % (64 / WR).
      const int at = NE * (j / WR) + 4 * (j % WR / (kWave / WR * 4)) + j % 4;
      uint32_t word = 0;
#pragma unroll
      for (int c = 0; c < PS; ++c) {
        if (c != at / 8) continue;
#pragma unroll
        for (int w = 0; w < 4; ++w) word |= w == at % 8 / 2 ? pk[c][w] : 0u;
      }
      word = at % 2 != 0 ? word >> 16 : word & 0xffffu;
      const uint32_t takes = __shfl(word, lr + WR * (j / 4 % (kWave / WR)), kWave) != 0 ? 0xffffffffu : 0u;
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
        up[b] |= sm.up[st][j][b] & takes;
        down[b] |= sm.down[st][j][b] & takes;
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int u = static_cast<int>(up[WR * b / 32] >> (part4 + WR * b % 32));
      const int d = static_cast<int>(down[WR * b / 32] >> (part4 + WR * b % 32));
#pragma unroll
      for (int i = 0; i < NE; ++i) {
        constexpr int kInf = 0x7f800000;
        const int at = 31 - (8 * (i / 4) + i % 4);
        acc[b][i] += __int_as_float(((u << at) >> 31) & kInf);
        acc[b][i] -= __int_as_float(((d << at) >> 31) & kInf);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  // (restrict: reads of one stage need not wait for loads to the other, which the
  // compiler otherwise makes them: one prompt of 2048 tokens 67.6 us, and 76.2 so.)
  auto step = [&](int n, int st, const typename Smem::Stage* __restrict__ from, typename Smem::Stage* __restrict__ to) {
    if (n + 1 < n1) load(n + 1, to);
    compute(n, st, from);
  };

  if (n0 < n1) {
    load(n0, sm.stage);
    store(n0, 0);
    lds_barrier();
    for (int n = n0; n < n1; ++n) {
      const int st = (n - n0) & 1;
      step(n, st, sm.stage + st, sm.stage + (st ^ 1));
      if (n + 1 < n1) store(n + 1, st ^ 1);
      lds_barrier();
    }
  }

  l_run = Math::row_sum(l_run);
  if (WR * wave + lr >= rows) return;
  if (parts > 1) {
    // Partial results: sums against m_ref, joined by tile_join_kernel.
    const int64_t slot = static_cast<int64_t>(item) * tile_rows(D) + WR * wave + lr;
    float* dst = p.tile_ws + slot * D + part4;
    if (part4 == 0) {
      p.tile_ml[2 * slot] = m_ref;
      p.tile_ml[2 * slot + 1] = l_run;
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int g = 0; g < NE / 4; ++g)
        *reinterpret_cast<f32x4*>(dst + WR * b + 8 * g) =
            f32x4{acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]};
    return;
  }
  const float inv = l_run == 0.0f ? 0.0f : p.v_scale / l_run;
  uint16_t* dst = p.out + token * p.o_st + static_cast<int64_t>(q_head) * p.o_sh + part4;
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int g = 0; g < NE / 4; ++g) {
      const f32x4 y = {acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]};
      store4<E>(p, dst + WR * b + 8 * g, l_run == 0.0f ? f32x4{0.f, 0.f, 0.f, 0.f} : y * inv);
    }
}

// The workgroups of tile_work alone (wide heads; the others share a launch with row_work).
template <typename E, int D, bool FP8, bool BS16>
__global__ __launch_bounds__(kTileThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void tile_kernel(const KParams) {
  __shared__ TileSmem<D> sm;
  tile_work<E, D, FP8, BS16>(fresh_args(), sm);
}

// Joins the parts of row tiles over which tile_work was spread, in their
// order. Workgroup (x, y) takes 16 rows of tile x / hkv, KV head x % hkv.
template <typename E, int D>
__global__ __launch_bounds__(kTileThreads) void tile_join_kernel(const KParams) {
  Args& p = fresh_args();
  constexpr int LD = D / 4;                  // lanes of a row
  constexpr int RS = kTileThreads / LD;      // rows side by side
  __shared__ LocateSmem loc;
  int seq, local, parts = 1;
  const int kv_head = static_cast<int>(blockIdx.x) % p.hkv;
  const int item0 = static_cast<int>(blockIdx.x) / p.hkv;
  locate(
      p.num_seqs, loc, [&](int s) { return row_tiles<D>(p, p.starts[s], p.starts[s + 1]); },
      [&](int total) {
        parts = parts_of(p, total);
        return false;
      },
      [](int w) { return w; }, [&] { return item0; }, seq, local);
  if (seq < 0 || parts == 1) return;
  const Seq sq = make_seq(p, scalar_load(p.starts, seq), scalar_load(p.starts, seq + 1), scalar_load(p.lens, seq),
                          p.prefix != nullptr ? scalar_load(p.prefix, seq) : 0);
  const RowTile<D> rt(p, sq, local);
  const int per = rt.per_part(parts);
  const int used = max((rt.tiles.count + per - 1) / per, 1);
  const int d = 4 * (static_cast<int>(threadIdx.x) % LD);
  for (int r = 16 * static_cast<int>(blockIdx.y) + static_cast<int>(threadIdx.x) / LD;
       r < min(16 * static_cast<int>(blockIdx.y) + 16, rt.rows); r += RS) {
    if (static_cast<int>(threadIdx.x) >= RS * LD) break;
    // Part i's item is (item0 parts + i) hkv + the KV head, counted from the last (tile_kernel).
    const int64_t slot = (static_cast<int64_t>(item0) * parts * p.hkv + (p.hkv - 1 - kv_head)) * tile_rows(D) + r;
    const int64_t step = static_cast<int64_t>(p.hkv) * tile_rows(D);
    float M = -__builtin_huge_valf();
#pragma unroll 4
    for (int i = 0; i < used; ++i) M = fmaxf(M, p.tile_ml[2 * (slot + i * step)]);
    const float ref = M == -__builtin_huge_valf() ? 0.0f : M;
    float L = 0.0f;
    f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < used; ++i) {
      const float f = __builtin_amdgcn_exp2f(p.tile_ml[2 * (slot + i * step)] - ref);
      L += f * p.tile_ml[2 * (slot + i * step) + 1];
      O += f * *reinterpret_cast<const f32x4*>(p.tile_ws + (slot + i * step) * D + d);
    }
    const int row = rt.row0 + r, tok = row / p.group;
    uint16_t* dst = p.out + static_cast<int64_t>(sq.first + tok) * p.o_st +
                    static_cast<int64_t>(kv_head * p.group + row - tok * p.group) * p.o_sh + d;
    store4<E>(p, dst, L == 0.0f ? f32x4{0.f, 0.f, 0.f, 0.f} : O * (p.v_scale / L));
  }
}

// LDS of row_work: each wave's current key tile, then, at the end of a piece,
// the waves' sums in the same place.
template <int D, int R, bool FP8>
struct RowSmem {
  static constexpr int TT = FP8 ? 32 : 16;  // keys of a tile: as many bytes in flight with either cache
  static constexpr int P = D + 16;          // row pitch, elements: 4 rows on distinct banks for the transpose reads
  static constexpr int OP = D + 4;          // row pitch, floats
  struct __attribute__((aligned(16))) Tile {
    uint16_t k[TT * P];
    uint16_t v[TT * P];
    uint32_t up[TT][D / 32], down[TT][D / 32];  // as in TileSmem
  };
  union {
    Tile tile[kTileWaves];
    float o[kTileWaves][16 * R * OP];
  };
  float m[kTileWaves][16 * R], l[kTileWaves][16 * R];
  LocateSmem loc;
};

template <int D, int R>
constexpr int row_occupancy() {  // waves per SIMD
  return D <= 64 ? (R == 1 ? 3 : 2) : D <= 128 ? 2 : 1;
}

// Decode and speculation: up to 16 R rows a KV head (R = 1 or 2). Bound by the reading of the
// cache, so all rows take each key tile once, a wave streams whole rows of its
// own tiles (two in flight in registers) and the work is cut over the cache's
// length: with `shares`, workgroup g of a KV head takes the g-th of equal
// shares of all sequences' key tiles, whatever their lengths. A piece that is
// not a whole sequence leaves its sums in slot g + s (sequence s; no two pieces
// share one) for row_join_kernel. Scores are S^T = K Q^T and the output O^T =
// V^T P^T on 16x16 MFMAs: lane l holds rows l % 16 (and + 16) of both.
// 64 sequences of 605 MB in all: 103 us, 5.8 TB/s with the joining launch; one
// of 128K keys (537 MB) 92 us; 32 with windows (68 MB) 23 us, of which joining
// and the second launch are 5; 48 speculating over 203 MB of fp8: 56 us (two
// waves a SIMD that wait for their own loads and LDS writes: vector units 32%
// busy, LDS 33%, matrix units 13%).
template <typename E, int D, int R, bool FP8, bool BS16, typename Params>
__device__ __forceinline__ void row_work(const Params& p, RowSmem<D, R, FP8>& sm) {
  using Smem = RowSmem<D, R, FP8>;
  constexpr int TT = Smem::TT, P = Smem::P, OP = Smem::OP;
  constexpr int TG = TT / 16;           // 16-key groups of a tile: each lies in one cache block (BS16)
  constexpr int CH = D / 32, NB = D / 16;
  constexpr int ELT = FP8 ? 1 : 2;
  constexpr int RB = D * ELT;           // bytes of a K (or V) row
  constexpr int NI = 16 * RB / 1024;    // 16-byte loads of a lane for a group of K (or V)
  constexpr int DEPTH = 2;              // tiles in flight
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int l16 = lane % 16, lg = lane / 16;
  // Workgroup g of a KV head (formed where they are used, as the arguments).
  auto head_of = [](Args& x) { return (static_cast<int>(blockIdx.x) - x.row_from) % x.hkv; };
  auto group_of = [](Args& x) { return (static_cast<int>(blockIdx.x) - x.row_from) / x.hkv; };

  struct Work {
    Seq sq;
    int rows, pos0, lo;
    KeyTiles tiles;
  };
  auto work_of = [&](const Seq& sq) {
    Work w;
    w.sq = sq;
    const int64_t rows = static_cast<int64_t>(sq.n) * p.group;
    // (slot_rows: no more than the caller's bound on the new tokens allows.)
    w.rows = rows <= 16 * R ? min(static_cast<int>(rows), fresh_args().slot_rows) : 0;
    w.pos0 = sq.len - sq.n;
    w.lo = max(w.pos0 - p.window + 1, 0);
    w.tiles = key_tiles<TT>(sq.pre, w.lo, sq.len);
    return w;
  };
  // A sequence of any rows has a tile, so that rows that see nothing are written too.
  auto weight_of = [&](const Work& w) { return w.rows > 0 ? max(w.tiles.count, 1) : 0; };

  int seq, local, share = 0;
  bool single = false;
  if (Args& a = fresh_args(); a.shares > 0) {
    locate(
        a.num_seqs, sm.loc,
        [&](int s) {
          return weight_of(work_of(make_seq(a, a.starts[s], a.starts[s + 1], a.lens[s], a.prefix != nullptr ? a.prefix[s] : 0)));
        },
        [&](int all) {
          share = max((all + a.shares - 1) / a.shares, kMinShare);
          if (a.num_seqs >= a.shares) return false;
          // One piece a workgroup, equal parts of one sequence, where the parts
          // get only a little longer by it.
          // (share >= all / (shares - seqs + 1): the parts, of up to share - 1 more
          // units each than they hold, are shares at most.)
          const int most = a.shares - a.num_seqs + 1;
          const int longer = max((all + most - 1) / most, kMinShare);
          if (longer - share > kMorePart) return false;
          share = longer;
          single = true;
          return true;
        },
        [&](int units) { return (units + share - 1) / share; },
        [&] { return single ? group_of(a) : static_cast<int>(min(static_cast<int64_t>(group_of(a)) * share, int64_t{0x7fffffff})); },
        seq, local);
    if (seq < 0) return;
  } else {
    seq = group_of(fresh_args());
    local = 0;
  }
  int left = share;

  typename Smem::Tile& tile = sm.tile[wave];

  for (;; ++seq, local = 0) {
    Args& a = fresh_args();
    if (seq >= a.num_seqs) return;
    const int kv_head = head_of(a);
    const char* kbase = static_cast<const char*>(a.k) + ELT * (static_cast<int64_t>(kv_head) * a.k_sh);
    const char* vbase = static_cast<const char*>(a.v) + ELT * (static_cast<int64_t>(kv_head) * a.v_sh);
    const Seq sq = make_seq(a, scalar_load(a.starts, seq), scalar_load(a.starts, seq + 1), scalar_load(a.lens, seq),
                            a.prefix != nullptr ? scalar_load(a.prefix, seq) : 0);
    const Work w = work_of(sq);
    const int weight = weight_of(w);
    if (weight == 0) {
      if (share == 0) return;
      continue;
    }
    if (single) {  // part `local` of this sequence
      const int parts = (weight + share - 1) / share;
      left = (weight + parts - 1) / parts;
      local = min(local * left, weight);
    }
    const int u0 = local, u1 = share > 0 ? min(weight, local + left) : weight;
    const int per = left;
    left -= u1 - u0;
    const bool whole = u0 == 0 && u1 == weight;
    if (share > 0 && u0 == 0 && tid == 0) {  // for row_join_kernel: the first of its pieces' workgroups, and how many
      int32_t* first = a.ws_first + 2 * (static_cast<int64_t>(seq) * a.hkv + kv_head);
      first[0] = group_of(a);
      first[1] = whole ? 0 : single ? (weight + per - 1) / per : 1 + (weight - u1 + share - 1) / share;
    }
    // This lane's rows (the last one from there on).
    int q_head[R], pos[R];
    u32x4 qf[R][CH];  // B operand: row 16 r + l16, columns 32 c + 8 lg ...
    float slope2[R];
    const bool wide = (reinterpret_cast<uintptr_t>(a.q) % 16 == 0) && a.q_st % 8 == 0 && a.q_sh % 8 == 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int row = min(16 * r + l16, w.rows - 1);
      const int tok = row / a.group;
      q_head[r] = kv_head * a.group + (row - tok * a.group);
      pos[r] = w.pos0 + tok;
      const uint16_t* src =
          a.q + static_cast<int64_t>(sq.first + tok) * a.q_st + static_cast<int64_t>(q_head[r]) * a.q_sh + 8 * lg;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (wide) {
          qf[r][c] = *reinterpret_cast<const u32x4*>(src + 32 * c);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            qf[r][c][e] = static_cast<uint32_t>(src[32 * c + 2 * e]) | static_cast<uint32_t>(src[32 * c + 2 * e + 1]) << 16;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) qf[r][c][e] ^= a.q_sign;
      }
      slope2[r] = a.slopes != nullptr ? a.slopes[q_head[r]] * kLog2e : 0.0f;
    }
    auto used = [&](int j) { return in_ranges(j, sq.pre, w.lo, sq.len); };
    auto page_at = [&](auto& c, int j) {
      return min(max(c.tables[static_cast<int64_t>(seq) * c.bt_stride + div_block(c, j)], 0), c.num_blocks - 1);
    };

    f32x4 acc[R][NB];  // O^T: row 16 r + l16, columns 16 b + 4 lg + i
    float m_ref[R], l_run[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[r][b] = f32x4{0.f, 0.f, 0.f, 0.f};
      m_ref[r] = -__builtin_huge_valf();
      l_run[r] = 0.0f;
    }

    struct Regs {
      u32x4 k[TG * NI], v[TG * NI];
    } buf[DEPTH];

    int pages[TG];  // lane e: the cache block of this wave's e-th tile from c0 on (-1: no key of it is seen)
    // The wave's i-th tile is u0 + wave + 4 i.
    auto tile_at = [&](int i) { return w.tiles.index(u0 + wave + kTileWaves * i) * TT; };
    auto load = [&](int i, int e, bool live, Regs& r) {
      const int t0 = tile_at(i);
      const int all = t0 + TT <= sq.pre || (t0 >= w.lo && t0 + TT <= sq.len) ? -1 : 0;  // every key of the tile
#pragma unroll
      for (int h = 0; h < TG; ++h) {
        const int r0 = t0 + 16 * h;
        if constexpr (BS16) {
          const int page = __builtin_amdgcn_readlane(pages[h], e);
          const int nrec = live && page >= 0 ? 0x7fffffff : 0;
          const int off = r0 - div_block(p, r0) * p.block_size;
          const int64_t pg = page < 0 ? 0 : page;
          const char* kt = kbase + ELT * (pg * p.k_sb + static_cast<int64_t>(off) * p.k_st);
          const char* vt = vbase + ELT * (pg * p.v_sb + static_cast<int64_t>(off) * p.v_st);
          const auto brk = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(kt), 0, nrec, kRsrcWord3);
          const auto brv = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(vt), 0, nrec, kRsrcWord3);
          auto fetch = [&](const __amdgpu_buffer_rsrc_t rsrc, int stride, u32x4* to) {
#pragma unroll
            for (int x = 0; x < NI; ++x) {
              // 1 KB of rows end to end: with whole rows, one offset a lane and scalar steps.
              constexpr bool kStep = 1024 % RB == 0 && D < 256;  // (256: no scalar registers left for them)
              const int o = (kStep ? 0 : 1024 * x) + 16 * lane;
              const int step = kStep ? x * (1024 / RB) * stride * ELT : 0;
              int off = o / RB * stride * ELT + o % RB;
              off |= ~(all | used(r0 + (1024 * x + 16 * lane) / RB));  // -1, past num_records: zeros
              to[x] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, step, 2);
            }
          };
          fetch(brk, p.k_st, r.k + NI * h);
          fetch(brv, p.v_st, r.v + NI * h);
        } else {
#pragma unroll
          for (int x = 0; x < NI; ++x) {
            const int o = 1024 * x + 16 * lane;
            const int j = r0 + o / RB;
            r.k[NI * h + x] = r.v[NI * h + x] = u32x4{0u, 0u, 0u, 0u};
            if (live && used(j) != 0) {
              const int blk = div_block(p, j);
              const int64_t page = page_at(p, j);
              const int64_t off = j - blk * p.block_size;
              r.k[NI * h + x] = *reinterpret_cast<const u32x4*>(kbase + ELT * (page * p.k_sb + off * p.k_st) + o % RB);
              r.v[NI * h + x] = *reinterpret_cast<const u32x4*>(vbase + ELT * (page * p.v_sb + off * p.v_st) + o % RB);
            }
          }
        }
      }
    };

    // Every row sees all keys of the tile from t0 on.
    auto all_see = [&](int t0) { return t0 + TT <= sq.pre || (t0 + TT - 1 <= w.pos0 && t0 > sq.len - 1 - p.window); };
    // Tile i to LDS in the dtype. Where some rows see a key and others do not
    // (not where all are of one position), infinities and NaN of V are taken
    // out; whether this lane had any.
    auto stage = [&](int i, const Regs& r) {
      bool bad = false;
      const bool mixed = sq.n > 1 && !all_see(tile_at(i));
#pragma unroll
      for (int x = 0; x < TG * NI; ++x) {
        const int o = 1024 * (x % NI) + 16 * lane;
        const int rr = 16 * (x / NI) + o / RB, col = (o % RB) / ELT;
        u32x4 v0, v1;
        if constexpr (FP8) {
          *reinterpret_cast<u32x4*>(tile.k + rr * P + col) = fp8x8_to<E>(u32x2{r.k[x][0], r.k[x][1]});
          *reinterpret_cast<u32x4*>(tile.k + rr * P + col + 8) = fp8x8_to<E>(u32x2{r.k[x][2], r.k[x][3]});
          v0 = fp8x8_to<E>(u32x2{r.v[x][0], r.v[x][1]});
          v1 = fp8x8_to<E>(u32x2{r.v[x][2], r.v[x][3]});
        } else {
          *reinterpret_cast<u32x4*>(tile.k + rr * P + col) = r.k[x];
          v0 = r.v[x];
        }
        if (mixed) {
          uint32_t up, down;
          v0 = take_out<E>(v0, up, down);
          reinterpret_cast<uint8_t*>(tile.up[rr])[col / 8] = static_cast<uint8_t>(up);
          reinterpret_cast<uint8_t*>(tile.down[rr])[col / 8] = static_cast<uint8_t>(down);
          bad = bad || (up | down) != 0;
          if constexpr (FP8) {
            v1 = take_out<E>(v1, up, down);
            reinterpret_cast<uint8_t*>(tile.up[rr])[col / 8 + 1] = static_cast<uint8_t>(up);
            reinterpret_cast<uint8_t*>(tile.down[rr])[col / 8 + 1] = static_cast<uint8_t>(down);
            bad = bad || (up | down) != 0;
          }
        }
        *reinterpret_cast<u32x4*>(tile.v + rr * P + col) = v0;
        if constexpr (FP8) *reinterpret_cast<u32x4*>(tile.v + rr * P + col + 8) = v1;
      }
      return bad;
    };

    auto consume = [&](int i, bool bad) {
      const int t0 = tile_at(i);
      const bool full = all_see(t0);
      f32x4 s[R][TG];  // keys t0 + 16 h + 4 lg + i of row 16 r + l16
#pragma unroll
      for (int h = 0; h < TG; ++h) {
#pragma unroll
        for (int x = 0; x < R; ++x) s[x][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const u32x4 ka = *reinterpret_cast<const u32x4*>(tile.k + (16 * h + l16) * P + 8 * lg + 32 * c);
#pragma unroll
          for (int x = 0; x < R; ++x) s[x][h] = E::mfma_16x16x32(ka, qf[x][c], s[x][h]);
        }
      }
      // 16-bit caches: weights as a sum of two parts of the dtype, exact to 2^-16,
      // since the products are a small part of a call that waits for memory. An
      // fp8 cache brings twice the keys in that time: its weights are rounded
      // once, as in tile_work.
      u32x2 hi[R][TG], lo[R][TG];
#pragma unroll
      for (int x = 0; x < R; ++x) {
        float factor = p.scale2;
        if (p.cap2 > 0.0f) {
          if (p.cap2 <= kExactCap * kLog2e) {
#pragma unroll
            for (int h = 0; h < TG; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[x][h][e] = capped<false>(p, s[x][h][e]);
          } else {
#pragma unroll
            for (int h = 0; h < TG; ++h)
#pragma unroll
              for (int e = 0; e < 4; ++e) s[x][h][e] = capped<true>(p, s[x][h][e]);
          }
          factor = 1.0f;
        }
        if (p.biased != 0) {
          const int away0 = fresh_vgpr(pos[x] - t0 - 4 * lg);
#pragma unroll
          for (int h = 0; h < TG; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[x][h][e] = s[x][h][e] * factor - slope2[x] * static_cast<float>(abs(away0 - 16 * h - e));
          factor = 1.0f;
        }
        if (!full) {
          const int away0 = fresh_vgpr(pos[x] - t0 - 4 * lg), to_prefix = fresh_vgpr(sq.pre - t0 - 4 * lg);
#pragma unroll
          for (int h = 0; h < TG; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool sees =
                  static_cast<uint32_t>(away0 - 16 * h - e) < static_cast<uint32_t>(p.window) || 16 * h + e < to_prefix;
              s[x][h][e] = sees ? s[x][h][e] * factor : -__builtin_huge_valf();
            }
          factor = 1.0f;
        }
        float top = -__builtin_huge_valf();
#pragma unroll
        for (int h = 0; h < TG; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, s[x][h][e]);
        top = rows_max(top) * factor;
        if (__any(top > m_ref[x] + 8.0f)) {  // the reference follows only where a tile passes it by 2^8
          const float m_new = fmaxf(m_ref[x], top);
          const float alpha = __builtin_amdgcn_exp2f(m_ref[x] - (m_new == -__builtin_huge_valf() ? 0.0f : m_new));
          m_ref[x] = m_new;
          l_run[x] *= alpha;
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[x][b] *= alpha;
        }
        const float ref = m_ref[x] == -__builtin_huge_valf() ? 0.0f : m_ref[x];
#pragma unroll
        for (int h = 0; h < TG; ++h) {
          float w4[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w4[e] = __builtin_amdgcn_exp2f(s[x][h][e] * factor - ref);
            l_run[x] += w4[e];
          }
          hi[x][h] = u32x2{pack2<E>(w4[0], w4[1]), pack2<E>(w4[2], w4[3])};
          if constexpr (!FP8)
            lo[x][h] = u32x2{pack2<E>(w4[0] - E::lo(hi[x][h][0]), w4[1] - E::hi(hi[x][h][0])),
                             pack2<E>(w4[2] - E::lo(hi[x][h][1]), w4[3] - E::hi(hi[x][h][1]))};
        }
      }
      const uint16_t* vt = tile.v + (4 * lg + l16 / 4) * P + 4 * (l16 % 4);
      using lds_v4i16 = __attribute__((address_space(3))) s16x4;
      auto v_read = [&](int h, int b) {  // columns 16 b + l16, keys 16 h + 4 lg ...
        return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(vt + 16 * h * P + 16 * b)));
      };
      if constexpr (FP8) {
        // 32 keys a product, in the order in which a lane has their weights.
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const u32x2 v0 = v_read(0, b), v1 = v_read(1, b);
#pragma unroll
          for (int x = 0; x < R; ++x)
            acc[x][b] = E::mfma_16x16x32(u32x4{v0[0], v0[1], v1[0], v1[1]},
                                         u32x4{hi[x][0][0], hi[x][0][1], hi[x][1][0], hi[x][1][1]}, acc[x][b]);
        }
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const u32x2 va = v_read(0, b);
#pragma unroll
          for (int x = 0; x < R; ++x) {
            acc[x][b] = E::mfma_16x16x16(va, hi[x][0], acc[x][b]);
            acc[x][b] = E::mfma_16x16x16(va, lo[x][0], acc[x][b]);
          }
        }
      }
      if (__any(bad)) {
        // As in tile_kernel: a row takes the infinities whose key has a weight there.
#pragma unroll
        for (int x = 0; x < R; ++x) {
          uint32_t up[CH] = {}, down[CH] = {};
#pragma unroll 1
          for (int j = 0; j < TT; ++j) {
            uint32_t word = 0;
#pragma unroll
            for (int h = 0; h < TG; ++h)
#pragma unroll
              for (int y = 0; y < 2; ++y) word |= h == j / 16 && y == j % 4 / 2 ? hi[x][h][y] : 0u;
            word = j % 2 != 0 ? word >> 16 : word & 0xffffu;
            const uint32_t takes = __shfl(word, l16 + 16 * (j % 16 / 4), kWave) != 0 ? 0xffffffffu : 0u;
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              up[c] |= tile.up[j][c] & takes;
              down[c] |= tile.down[j][c] & takes;
            }
          }
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            const int u = static_cast<int>(up[b / 2] >> (16 * (b % 2) + 4 * lg));
            const int d = static_cast<int>(down[b / 2] >> (16 * (b % 2) + 4 * lg));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              acc[x][b][e] += __int_as_float(((u << (31 - e)) >> 31) & 0x7f800000);
              acc[x][b][e] -= __int_as_float(((d << (31 - e)) >> 31) & 0x7f800000);
            }
          }
        }
      }
    };

    const int count = min(u1, w.tiles.count) - u0;  // 0: no key is seen
    const int mine = count > wave ? (count - wave + kTileWaves - 1) / kTileWaves : 0;
    for (int c0 = 0; c0 < mine; c0 += kWave) {
      const int m = min(mine - c0, kWave);
      if constexpr (BS16) {
        Args& c = fresh_args();
#pragma unroll
        for (int h = 0; h < TG; ++h) {
          pages[h] = -1;
          if (lane < m) {
            const int r0 = tile_at(c0 + lane) + 16 * h;
            if (r0 < sq.pre || (r0 + 16 > w.lo && r0 < sq.len)) pages[h] = page_at(c, r0);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        load(c0 + d, d, d < m, buf[d]);
        __builtin_amdgcn_sched_barrier(0);
      }
      for (int i = 0; i < m; i += DEPTH) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          if (i + d < m) consume(c0 + i + d, stage(c0 + i + d, buf[d]));
          // Past the end too, from no records, so that the waits stay for the oldest tile.
          load(c0 + i + d + DEPTH, min(i + d + DEPTH, kWave - 1), i + d + DEPTH < m, buf[d]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }

    // The waves' sums to one.
    Args& b = fresh_args();
    const int head = head_of(b), g = group_of(b);
    lds_barrier();  // every wave has read its last tile
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float l_all = rows_sum(l_run[r]);
      if (lg == 0) {
        sm.m[wave][16 * r + l16] = m_ref[r];
        sm.l[wave][16 * r + l16] = l_all;
      }
      if (16 * r + l16 < w.rows) {
#pragma unroll
        for (int n = 0; n < NB; ++n) *reinterpret_cast<f32x4*>(&sm.o[wave][(16 * r + l16) * OP + 16 * n + 4 * lg]) = acc[r][n];
      }
    }
    lds_barrier();
    const int64_t slot = (static_cast<int64_t>(g + seq) * b.hkv + head) * b.slot_rows;
    for (int idx = tid; idx < w.rows * (D / 4); idx += kTileThreads) {
      const int r = idx / (D / 4), d = 4 * (idx % (D / 4));
      float M = sm.m[0][r];
#pragma unroll
      for (int x = 1; x < kTileWaves; ++x) M = fmaxf(M, sm.m[x][r]);
      const float ref = M == -__builtin_huge_valf() ? 0.0f : M;
      float L = 0.0f;
      f32x4 O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < kTileWaves; ++x) {
        const float f = __builtin_amdgcn_exp2f(sm.m[x][r] - ref);
        L += f * sm.l[x][r];
        O += f * *reinterpret_cast<const f32x4*>(&sm.o[x][r * OP + d]);
      }
      if (whole) {
        const int rt = r / b.group;
        uint16_t* dst = b.out + static_cast<int64_t>(sq.first + rt) * b.o_st +
                        static_cast<int64_t>(head * b.group + r - rt * b.group) * b.o_sh + d;
        store4<E>(b, dst, L == 0.0f ? f32x4{0.f, 0.f, 0.f, 0.f} : O * (b.v_scale / L));
      } else {
        *reinterpret_cast<f32x4*>(b.ws + (slot + r) * D + d) = O;
        if (d == 0) {
          b.ws_ml[2 * (slot + r)] = M;
          b.ws_ml[2 * (slot + r) + 1] = L;
        }
      }
    }
    if (single || left <= 0) return;
    lds_barrier();  // the sums have been read: the next piece's tiles may take their place
  }
}

template <typename E, int D, int R, bool FP8, bool BS16>
__global__ __launch_bounds__(kTileThreads)
__attribute__((amdgpu_waves_per_eu(row_occupancy<D, R>(), row_occupancy<D, R>())))
void row_kernel(const KParams p) {
  __shared__ RowSmem<D, R, FP8> sm;
  row_work<E, D, R, FP8, BS16>(p, sm);
}

// Both in one launch: the tiles' workgroups, then the rows', which run beside
// the last tiles. (Up to head_dim 128: the others need all registers for the rows.)
template <typename E, int D, bool FP8, bool BS16>
__global__ __launch_bounds__(kTileThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void mixed_kernel(const KParams) {
  constexpr size_t kBytes = std::max(sizeof(TileSmem<D>), sizeof(RowSmem<D, 1, FP8>));
  __shared__ __attribute__((aligned(16))) char raw[kBytes];
  if (static_cast<int>(blockIdx.x) < fresh_args().tile_groups)
    tile_work<E, D, FP8, BS16>(fresh_args(), *reinterpret_cast<TileSmem<D>*>(raw));
  else
    row_work<E, D, 1, FP8, BS16>(fresh_args(), *reinterpret_cast<RowSmem<D, 1, FP8>*>(raw));
}

// Joins the pieces of row_work's cut sequences, in their order: a wave a row.
template <typename E, int D>
__global__ __launch_bounds__(kTileThreads) void row_join_kernel(const KParams p) {
  constexpr int LD = D / 4;                        // lanes of a row
  constexpr int SETS = kWave / LD > 0 ? kWave / LD : 1;  // pieces side by side
  const int lane = threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) / kWave);
  const int kv_head = static_cast<int>(blockIdx.x) % p.hkv;
  const int seq = static_cast<int>(blockIdx.x) / p.hkv;
  const int r = static_cast<int>(blockIdx.y) * kTileWaves + wave;
  const Seq sq = make_seq(p, scalar_load(p.starts, seq), scalar_load(p.starts, seq + 1), 0, 0);
  const int64_t rows = static_cast<int64_t>(sq.n) * p.group;
  if (rows > p.short_rows || r >= min(static_cast<int>(rows), p.slot_rows)) return;  // a tiled sequence, or no such row
  const int64_t entry = 2 * (static_cast<int64_t>(seq) * p.hkv + kv_head);
  const int g = p.ws_first[entry], count = p.ws_first[entry + 1];
  if (count == 0) return;  // written whole
  const int64_t slot = (static_cast<int64_t>(g + seq) * p.hkv + kv_head) * p.slot_rows + r;
  const int64_t step = static_cast<int64_t>(p.hkv) * p.slot_rows;  // the next workgroup's slot
  float M = -__builtin_huge_valf();
  for (int i = lane; i < count; i += kWave) M = fmaxf(M, p.ws_ml[2 * (slot + i * step)]);
  M = wave_max(M);
  const float ref = M == -__builtin_huge_valf() ? 0.0f : M;
  const int set = lane / LD, d = 4 * (lane % LD);
  float L = 0.0f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  if (set < SETS) {
#pragma unroll 4
    for (int i = set; i < count; i += SETS) {
      const float f = __builtin_amdgcn_exp2f(p.ws_ml[2 * (slot + i * step)] - ref);
      L += f * p.ws_ml[2 * (slot + i * step) + 1];
      O += f * *reinterpret_cast<const f32x4*>(p.ws + (slot + i * step) * D + d);
    }
  }
#pragma unroll
  for (int x = 1; x < SETS; ++x) {
    const int from = lane % LD + x * LD;
    const float l2 = __shfl(L, from, kWave);
    const f32x4 o2 = {__shfl(O[0], from, kWave), __shfl(O[1], from, kWave), __shfl(O[2], from, kWave), __shfl(O[3], from, kWave)};
    if (set == 0) {
      L += l2;
      O += o2;
    }
  }
  if (set != 0) return;
  const int rt = r / p.group;
  uint16_t* dst = p.out + static_cast<int64_t>(sq.first + rt) * p.o_st +
                  static_cast<int64_t>(kv_head * p.group + r - rt * p.group) * p.o_sh + d;
  store4<E>(p, dst, L == 0.0f ? f32x4{0.f, 0.f, 0.f, 0.f} : O * (p.v_scale / L));
}

// How a call is cut, from what the host knows: the sizes and the bounds.
struct Plan {
  int64_t tile_groups = 0;  // workgroups of tile_kernel; 0: every sequence has few rows
  int split_items = 0;      // as in KParams
  int64_t joins = 0;        // workgroups (x) of tile_join_kernel
  int64_t tile_ws = 0;      // rows of its partial results
  int64_t row_groups = 0;   // and of row_kernel
  int short_rows = 16, shares = 0, slot_rows = 32;
  int64_t slots = 0;        // row_kernel's
  int64_t ws_bytes = 0;
  int64_t tile_ml_at = 0, row_at = 0, ml_at = 0, first_at = 0;  // floats from the workspace's start
};

template <typename E, int D, bool FP8>
hipError_t launch_all(KParams kp, const Plan& plan, hipStream_t s) {
  const dim3 block(kTileThreads);
  // Rows of a 16-key group within the 2^31 bytes of a buffer resource.
  const bool bs16 = kp.block_size % 16 == 0 && int64_t{16} * 2 * std::max(kp.k_st, kp.v_st) < (int64_t{1} << 31);
  const unsigned tiles = static_cast<unsigned>(plan.tile_groups), rows = static_cast<unsigned>(plan.row_groups);
  if (D <= 128 && tiles > 0) {
    if constexpr (D <= 128) {
      kp.row_from = kp.tile_groups;
      if (bs16) hipLaunchKernelGGL((mixed_kernel<E, D, FP8, true>), dim3(tiles + rows), block, 0, s, kp);
      else hipLaunchKernelGGL((mixed_kernel<E, D, FP8, false>), dim3(tiles + rows), block, 0, s, kp);
    }
  } else {
    if constexpr (D > 128) {
      if (tiles > 0) {
        if (bs16) hipLaunchKernelGGL((tile_kernel<E, D, FP8, true>), dim3(tiles), block, 0, s, kp);
        else hipLaunchKernelGGL((tile_kernel<E, D, FP8, false>), dim3(tiles), block, 0, s, kp);
      }
    }
    if (kp.short_rows == 16) {
      if (bs16) hipLaunchKernelGGL((row_kernel<E, D, 1, FP8, true>), dim3(rows), block, 0, s, kp);
      else hipLaunchKernelGGL((row_kernel<E, D, 1, FP8, false>), dim3(rows), block, 0, s, kp);
    } else {
      if constexpr (D <= kWideRows) {
        if (bs16) hipLaunchKernelGGL((row_kernel<E, D, 2, FP8, true>), dim3(rows), block, 0, s, kp);
        else hipLaunchKernelGGL((row_kernel<E, D, 2, FP8, false>), dim3(rows), block, 0, s, kp);
      }
    }
  }
  if (kp.split_items > 0) {
    const dim3 join(static_cast<unsigned>(plan.joins), tile_rows(D) / 16);
    hipLaunchKernelGGL((tile_join_kernel<E, D>), join, block, 0, s, kp);
  }
  if (kp.shares > 0) {
    const dim3 join(static_cast<unsigned>(kp.num_seqs * kp.hkv), static_cast<unsigned>((kp.slot_rows + 3) / 4));
    hipLaunchKernelGGL((row_join_kernel<E, D>), join, block, 0, s, kp);
  }
  return hipGetLastError();
}

template <typename E>
hipError_t launch(const KParams& kp, const Plan& plan, int d, bool fp8, hipStream_t s) {
  if (fp8) {
    switch (d) {
      case 64: return launch_all<E, 64, true>(kp, plan, s);
      case 128: return launch_all<E, 128, true>(kp, plan, s);
      case 192: return launch_all<E, 192, true>(kp, plan, s);
      default: return launch_all<E, 256, true>(kp, plan, s);
    }
  }
  switch (d) {
    case 64: return launch_all<E, 64, false>(kp, plan, s);
    case 96: return launch_all<E, 96, false>(kp, plan, s);
    case 128: return launch_all<E, 128, false>(kp, plan, s);
    case 192: return launch_all<E, 192, false>(kp, plan, s);
    default: return launch_all<E, 256, false>(kp, plan, s);
  }
}

extern template hipError_t launch<Bf16>(const KParams&, const Plan&, int, bool, hipStream_t);
extern template hipError_t launch<F16>(const KParams&, const Plan&, int, bool, hipStream_t);

}  // namespace varlen
}  // namespace dk
