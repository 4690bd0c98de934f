// Attention weights accumulated beside the paged cache: for every cached token and
// KV head the weight that a step's queries give it,
//
//   w[slot(t), h] = decay w[slot(t), h] + sum_ij exp(scale q_ij . k_t - lse_ij)
//
// over the sequence's rows i that see the token (row i of n sits at position
// context - n + i and sees t up to there) and the heads j of the group.
//
// Decode (one row a sequence): K is read once.  A workgroup takes one KV head's keys,
// the scores go to LDS, and once their maximum and sum are known the weights follow;
// long contexts are split, their scores kept in memory for a second kernel.  HBM bound
// (98k and 131k keys: K and the kept scores 97 us, 4.9 TB/s, the weights 16), latency
// bound for short contexts (700 keys 10 us, 60 of 300-800 in fp8 14).
//
// Chunks: the normaliser of a row takes all of its keys and the weight of a key all
// of its rows, so scores are computed twice rather than kept: weights_lse_kernel holds
// 64 rows of q a wave in registers and streams K through LDS (S^T = K Q^T, a row's
// maximum and sum in its column's lanes), weights_columns_kernel holds 64 keys a wave
// and streams q (S = Q K^T, a key's sum in its column's lanes).  Neither product's
// result leaves the registers.  A key's sum is one wave's; a row's maximum and sum are
// joined between the waves that share its keys (short sequences) and, by
// weights_join_kernel, between the pieces that do, in an order that the lengths set, so
// that the result is one only.  Kept scores would be 4 bytes a pair, written and read
// (the windows below 131 us, reading K again 48).  4 windows of 32 rows over 8-32k keys take 48 and 48 us, 3.5 TB/s of K with
// vector instructions issuing in 44% of the first (a fourth tile's room: 51); 8 chunks of
// 512 rows over 1.5-4.6k keys 86 and 82 us, where the matrix and the vector units run
// one after another more than beside each other: 26% and 53% of the first.
//
// Products are exact (1-byte codes as 16-bit operands of q's type, fp32 on the fp32
// MFMA), their sums, the softmax and the weights fp32.
#include <type_traits>

#include "mkv_device.hpp"

namespace mkv {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

// (lambdas whose arrays have to stay in registers)
#define MKV_INLINE __attribute__((always_inline))

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kNegBig = -1e30f;
constexpr float kNegInf = -__builtin_huge_valf();
// a row's running maximum moves only when a tile exceeds it by more than 2^8
constexpr float kRescaleSlack = 8.0f;

struct WeightArgs {
  const char* q;
  const char* k;
  const float* k_scale;
  float* weights;
  PagedIndex idx;
  const void* ctx;
  int ctx_i64;
  const int32_t* cu;  // NULL: one row a sequence
  int num_seqs;
  int64_t total_q;
  int num_heads, num_kv_heads, group;
  uint32_t inv_group;  // 2^32 / group, rounded up
  float mul;           // scale log2(e)
  int scale_mode;      // 0 none, 1 per tensor, 2 per token and KV head
  float decay;
  // decode
  int unit;            // keys of a workgroup's turn
  int grid_units;      // workgroups of a (sequence, KV head)
  int max_units;
  int pair0;           // the launch's first (sequence, KV head)
  float* ws_t;         // scores of split contexts, of the launch's pairs
  f32x2* ws_ml;        // (pair, unit, query): maximum and sum
  // chunks
  int shares;          // pieces of the normalisers' work, at most
  f32x2* part_ml;      // (piece + block, KV head, row of the block): maximum and sum
  int64_t row_units;   // blocks at most
  float* lse;          // (row) log2 of the normaliser, +inf for a row that sees nothing;
                       // rows by KV head, sequence, token and head of the group
};

template <int CT>
using Op16 = typename std::conditional<CT == MKV_DTYPE_BF16, bf16x8, f16x8>::type;

template <int CT>
MKV_DEV f32x16 mfma32(u32x4 A, u32x4 B, f32x16 C) {
  if constexpr (CT == MKV_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, A), __builtin_bit_cast(bf16x8, B), C, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, A), __builtin_bit_cast(f16x8, B), C, 0, 0, 0);
}
template <int CT>
MKV_DEV f32x4 mfma16(u32x4 A, u32x4 B, f32x4 C) {
  if constexpr (CT == MKV_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, A), __builtin_bit_cast(bf16x8, B), C, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, A), __builtin_bit_cast(f16x8, B), C, 0, 0, 0);
}

// Eight one-byte codes as 16-bit operands, exact.
template <int KV, int CT>
MKV_DEV u32x4 codes_to_16(uint32_t lo, uint32_t hi) {
  if constexpr (KV == MKV_DTYPE_I8) {
    if constexpr (CT == MKV_DTYPE_BF16)
      return u32x4{__builtin_bit_cast(uint32_t, i8x2_to_bf16x2<false>(lo)), __builtin_bit_cast(uint32_t, i8x2_to_bf16x2<true>(lo)),
                   __builtin_bit_cast(uint32_t, i8x2_to_bf16x2<false>(hi)), __builtin_bit_cast(uint32_t, i8x2_to_bf16x2<true>(hi))};
    else
      return u32x4{__builtin_bit_cast(uint32_t, i8x2_to_f16x2<false>(lo)), __builtin_bit_cast(uint32_t, i8x2_to_f16x2<true>(lo)),
                   __builtin_bit_cast(uint32_t, i8x2_to_f16x2<false>(hi)), __builtin_bit_cast(uint32_t, i8x2_to_f16x2<true>(hi))};
  } else if constexpr (CT == MKV_DTYPE_BF16) {
    return u32x4{__builtin_bit_cast(uint32_t, fp8x2_to_bf16x2<false>(lo)), __builtin_bit_cast(uint32_t, fp8x2_to_bf16x2<true>(lo)),
                 __builtin_bit_cast(uint32_t, fp8x2_to_bf16x2<false>(hi)), __builtin_bit_cast(uint32_t, fp8x2_to_bf16x2<true>(hi))};
  } else {
    return u32x4{__builtin_bit_cast(uint32_t, fp8x2_to_f16x2<false>(lo)), __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<true>(lo)),
                 __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<false>(hi)), __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<true>(hi))};
  }
}

MKV_DEV float other_half(float x) {  // the value of lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
// over the 16 lanes of a DPP row, in each of them
template <class F>
MKV_DEV float row_all(float x, F f) {
  asm volatile("" : "+v"(x));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xf, 0xf, false)));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xf, 0xf, false)));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xf, 0xf, false)));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xf, 0xf, false)));
  return x;
}
MKV_DEV float sum_of_rows(float x) {  // the sum over the wave's four DPP rows, lane by lane
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// 1 / the sum of a softmax; nothing seen: 0, NaN stays
MKV_DEV float inverse(float l) { return l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l; }

struct Seq {
  int64_t q0, n;      // rows of q
  int64_t first;      // position of row 0, or keys where it is past them
  int keys;           // of the context, within the block table
};
MKV_DEV Seq seq_of(const WeightArgs& a, int s) {
  Seq r;
  r.q0 = s;
  r.n = 1;
  if (a.cu) {
    r.q0 = min(max((int64_t)a.cu[s], (int64_t)0), a.total_q);
    r.n = min(max((int64_t)a.cu[s + 1], r.q0), a.total_q) - r.q0;
  }
  const int64_t c = max(load_index(a.ctx, s, a.ctx_i64), (int64_t)0);
  r.keys = (int)min(c, (int64_t)a.idx.max_blocks << a.idx.bs_log2);
  // (a row past the keys sees all of them; the pieces' work stays within doubles' whole
  // numbers whatever the length given)
  r.first = min(c - r.n, (int64_t)r.keys);
  return r;
}
// slot of token t, or -1 (a lane's own)
MKV_DEV int slot_of(const WeightArgs& a, int seq, int t) {
  const int32_t p = a.idx.block_tables[(int64_t)seq * a.idx.bt_stride + (t >> a.idx.bs_log2)];
  return p >= 0 && p < a.idx.num_blocks ? (p << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : -1;
}

// ---------------------------------------------------------------------------
// Decode.  The scores are 16 queries by 16 keys (16x16 MFMA, A = q, B = K): lane
// (c, kg) holds key c and queries 4 i + kg, i < NI, so that a group of up to four
// costs one exponential a key and lane.  A lane loads its key's chunks 4 j + kg of 16
// bytes; the contraction's order is free, and q's operands follow it.
// ---------------------------------------------------------------------------
template <int KV, int CT, int D>
struct DecodeTile {
  static constexpr int kEb = DTypeInfo<KV>::kBytes;
  static constexpr int kLoads = D * kEb / 64;  // 16-byte loads a lane
  u32x4 w[kLoads];
  float scale;
};

template <int KV, int CT, int D>
struct DecodeQ {
  static constexpr int kOps = KV == MKV_DTYPE_F32 ? D / 16 : D / 32;
  u32x4 w[kOps];
  // kg: the lane's share of the contraction
  MKV_DEV void load(const char* row, int kg) {
#pragma unroll
    for (int s = 0; s < kOps; ++s) {
      const int d = KV == MKV_DTYPE_F32 ? 16 * s + 4 * kg
                    : DTypeInfo<KV>::kBytes == 2 ? 32 * s + 8 * kg : 64 * (s >> 1) + 16 * kg + 8 * (s & 1);
      w[s] = ld16(row + d * (KV == MKV_DTYPE_F32 ? 4 : 2));
    }
  }
  MKV_DEV void keep(bool ok) {
#pragma unroll
    for (int s = 0; s < kOps; ++s)
#pragma unroll
      for (int e = 0; e < 4; ++e) w[s][e] = ok ? w[s][e] : 0u;
  }
};

template <int KV, int CT, int D>
MKV_DEV f32x4 decode_scores(const DecodeQ<KV, CT, D>& q, const DecodeTile<KV, CT, D>& k) {
  using T = DecodeTile<KV, CT, D>;
  f32x4 s = f32x4{};
  if constexpr (KV == MKV_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(q.w[i][e]), __uint_as_float(k.w[i][e]), s, 0, 0, 0);
  } else if constexpr (T::kEb == 2) {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) s = mfma16<CT>(q.w[i], k.w[i], s);
  } else {
#pragma unroll
    for (int i = 0; i < T::kLoads; ++i) {
      s = mfma16<CT>(q.w[2 * i], codes_to_16<KV, CT>(k.w[i][0], k.w[i][1]), s);
      s = mfma16<CT>(q.w[2 * i + 1], codes_to_16<KV, CT>(k.w[i][2], k.w[i][3]), s);
    }
  }
  return s;
}

// The tiles of a wave: tile n holds keys k0 + 16 (n kWaves + wave) on.  Their block
// entries come by one load, a lane a tile (64 of them at most).
struct WaveTiles {
  const WeightArgs& a;
  int k0, k1, num, wave, entry;
  MKV_DEV WaveTiles(const WeightArgs& args, int seq, int k0_, int k1_, int wave_)
      : a(args), k0(k0_), k1(k1_), num(((k1_ - k0_ + 15) / 16 - wave_ + kWaves - 1) / kWaves), wave(wave_) {
    const int t = min(key(threadIdx.x & 63), k1 - 1);
    entry = a.idx.block_tables[(int64_t)seq * a.idx.bt_stride + (t >> a.idx.bs_log2)];
  }
  MKV_DEV int key(int n) const { return k0 + 16 * (n * kWaves + wave); }
  MKV_DEV bool is_there(int e) const { return e >= 0 && e < a.idx.num_blocks; }
  MKV_DEV int slot(int e, int t) const { return (e << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)); }
};

// Their weights, four tiles a round, all of the wave's lanes writing (lane row kg the
// kg-th tile's keys).  The old weights of the first kHeld rounds come ahead, under the
// scores' loads.
template <int NI>
struct TileWeights {
  static constexpr int kHeld = 4;
  const WeightArgs& a;
  const WaveTiles& w;
  int64_t fresh;  // tokens from here on came with these rows and start from 0
  int h, lane;
  int slot[kHeld];
  float old[kHeld];

  MKV_DEV int key(int round) const { return w.key(4 * round + (lane >> 4)) + (lane & 15); }
  MKV_DEV int slot_at(int round) const {
    const int e = __shfl(w.entry, 4 * round + (lane >> 4)), t = key(round);
    return t < w.k1 && w.is_there(e) ? w.slot(e, t) : -1;
  }
  MKV_DEV float load(int s) const { return a.weights[(int64_t)max(s, 0) * a.num_kv_heads + h]; }
  MKV_DEV TileWeights(const WeightArgs& args, const WaveTiles& tiles, int64_t first, int h_, bool used = true)
      : a(args), w(tiles), fresh(first), h(h_), lane(threadIdx.x & 63) {
    if (!used) return;
#pragma unroll
    for (int r = 0; r < kHeld; ++r) slot[r] = slot_at(r);
    if (a.decay != 0.0f) {
#pragma unroll
      for (int r = 0; r < kHeld; ++r) old[r] = load(slot[r]);
    }
  }
  template <class E>
  MKV_DEV void round(int r, int s, float was, E e) const {
    float mine = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = 0.0f;
      if (4 * r + j < w.num) {
#pragma unroll
        for (int i = 0; i < NI; ++i) x += e(4 * r + j, i);
      }
      x = sum_of_rows(x);
      mine = lane >> 4 == j ? x : mine;
    }
    if (a.decay != 0.0f && key(r) < fresh) mine = __builtin_fmaf(a.decay, was, mine);
    if (s >= 0) a.weights[(int64_t)s * a.num_kv_heads + h] = mine;
  }
  // e(n, i): the weight of this lane's key and i-th query in tile n
  template <bool MORE, class E>
  MKV_DEV void write(E e) const {
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
      if (4 * r < w.num) round(r, slot[r], old[r], e);
    if constexpr (MORE) {
      for (int r = kHeld; 4 * r < w.num; ++r) {
        const int s = slot_at(r);
        round(r, s, a.decay != 0.0f ? load(s) : 0.0f, e);
      }
    }
  }
};

constexpr int kSplitKeys = 1024;  // of a unit: 16 tiles a wave

// The workgroup's pair and first unit.  Workgroups go to the XCDs by turns.  A unit's
// heads share the weights' cache lines and stay together where the units are a multiple of
// 8, and then the sequences' first units, the only ones with keys under a wide table, are
// on unlike XCDs (60 sequences of 300-800 tokens under tables of 32,768: 38 us; all first
// units on one XCD: 171).
MKV_DEV void place_of(const WeightArgs& a, int& pair, int& x) {
  pair = blockIdx.x / a.grid_units;
  x = (int)(blockIdx.x % a.grid_units + (a.pair0 + pair) / a.num_kv_heads) % a.grid_units;
}

// One workgroup a (sequence, KV head) where its scores fit the LDS; else (SPLIT) a
// workgroup a unit of the keys, whose scores go to memory with their running maximum
// and sum, and weights_finish_kernel.
template <int KV, int CT, int D, int NI, bool SPLIT>
__global__ __launch_bounds__(kThreads) void weights_decode_kernel(WeightArgs a) {
  using Tile = DecodeTile<KV, CT, D>;
  // Tiles of a wave in a batch, two batches in flight: twice as many leave half the
  // workgroups on a CU (contexts of 98k and 131k keys 109 us against 100).
  constexpr int kAhead = KV == MKV_DTYPE_F32 ? 1 : 2;
  extern __shared__ float scores[];                    // (tile, i, lane)
  __shared__ float part_m[kWaves][4 * NI], part_l[kWaves][4 * NI];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, kg = lane >> 4;
  int pair, x;
  place_of(a, pair, x);
  const int seq = (a.pair0 + pair) / a.num_kv_heads, h = (a.pair0 + pair) % a.num_kv_heads;
  const Seq sq = seq_of(a, seq);
  const int units = (int)(((int64_t)sq.keys + a.unit - 1) / a.unit);
  if (x >= units) return;
  // row r = 4 kg + i of the product is query 4 i + kg of the group
  const int query = 4 * (c & 3) + (c >> 2);
  constexpr int kQBytes = D * (KV == MKV_DTYPE_F32 ? 4 : 2);
  DecodeQ<KV, CT, D> q;
  q.load(a.q + (sq.q0 * a.num_heads + h * a.group + min(query, a.group - 1)) * kQBytes, kg);
  const int64_t row_bytes = (int64_t)a.num_kv_heads * D * Tile::kEb;
  const char* const kbase = a.k + (int64_t)h * D * Tile::kEb + 16 * kg;
  float mul = a.mul;
  if (a.scale_mode == 1) mul *= load_uniform_f32(a.k_scale);
  bool begun = false;
  for (int u = x; u < units; u += a.grid_units) {
    const int k0 = u * a.unit, k1 = min(sq.keys, k0 + a.unit);
    const WaveTiles w(a, seq, k0, k1, wave);
    float m[NI], l[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      m[i] = kNegBig;
      l[i] = 0.0f;
    }
    auto load = [&](Tile (&t)[kAhead], uint32_t& here, int n0) MKV_INLINE {
      here = 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (n0 + j < w.num) {
          const int key = w.key(n0 + j), e = __builtin_amdgcn_readlane(w.entry, n0 + j);
          here |= w.is_there(e) ? 1u << j : 0u;
          // (keys past the last: the tile's first, which is there)
          const int64_t slot = w.slot(w.is_there(e) ? e : 0, key) + (key + c < k1 ? c : 0);
          const char* p = kbase + slot * row_bytes;
#pragma unroll
          for (int i = 0; i < Tile::kLoads; ++i) t[j].w[i] = ld16(p + 64 * i);
          t[j].scale = a.scale_mode == 2 ? a.k_scale[slot * a.num_kv_heads + h] : 1.0f;
        }
      }
    };
    auto take = [&](const Tile (&t)[kAhead], uint32_t here, int n0) MKV_INLINE {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (n0 + j < w.num) {
          const f32x4 s = decode_scores<KV, CT, D>(q, t[j]);
          const bool sees = (here >> j & 1) && w.key(n0 + j) + c < k1;
          const float f = mul * t[j].scale;
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const float v = sees ? s[i] * f : kNegInf;
            scores[(((n0 + j) * kWaves + wave) * NI + i) * 64 + lane] = v;
            if constexpr (SPLIT) {
              const float top = fmaxf(m[i], v);
              l[i] = __builtin_fmaf(l[i], __builtin_amdgcn_exp2f(m[i] - top), __builtin_amdgcn_exp2f(v - top));
              m[i] = top;
            } else {
              m[i] = fmaxf(m[i], v);
            }
          }
        }
      }
    };
    Tile t0[kAhead], t1[kAhead];
    uint32_t h0, h1;
    load(t0, h0, 0);
    load(t1, h1, kAhead);
    if (!begun) q.keep(query < a.group);
    begun = true;
    const TileWeights<NI> out(a, w, sq.first, h, !SPLIT);
    for (int n0 = 0; n0 < w.num; n0 += 2 * kAhead) {
      take(t0, h0, n0);
      load(t0, h0, n0 + 2 * kAhead);
      take(t1, h1, n0 + kAhead);
      load(t1, h1, n0 + 3 * kAhead);
    }
    if constexpr (SPLIT) {
      // (here: stores among the loads would have to end before the loads behind them)
      float* const kept = a.ws_t + ((int64_t)pair * a.max_units + u) * (a.unit / 16) * NI * 64 + lane;
      for (int n = 0; n < w.num; ++n)
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int at = ((n * kWaves + wave) * NI + i) * 64;
          kept[at] = scores[at + lane];
        }
    }
    // ---- the queries' maxima and sums, of the wave and of all ----
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const float top = row_all(m[i], [](float v, float w) { return fmaxf(v, w); });
      if constexpr (SPLIT) {
        l[i] *= __builtin_amdgcn_exp2f(m[i] - top);
      } else {
        for (int n = 0; n < w.num; ++n) {
          float* const at = scores + ((n * kWaves + wave) * NI + i) * 64 + lane;
          const float e = __builtin_amdgcn_exp2f(*at - top);
          l[i] += e;
          *at = e;
        }
      }
      m[i] = top;
      l[i] = row_all(l[i], [](float v, float w) { return v + w; });
      if (c == 0) {
        part_m[wave][4 * i + kg] = m[i];
        part_l[wave][4 * i + kg] = l[i];
      }
    }
    __syncthreads();
    float f[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      float top = part_m[0][4 * i + kg], sum = 0.0f;
#pragma unroll
      for (int v = 1; v < kWaves; ++v) top = fmaxf(top, part_m[v][4 * i + kg]);
#pragma unroll
      for (int v = 0; v < kWaves; ++v) sum += part_l[v][4 * i + kg] * __builtin_amdgcn_exp2f(part_m[v][4 * i + kg] - top);
      if (SPLIT && wave == 0 && c == 0) a.ws_ml[((int64_t)pair * a.max_units + u) * 4 * NI + 4 * i + kg] = f32x2{top, sum};
      f[i] = 4 * i + kg < a.group ? inverse(sum) * __builtin_amdgcn_exp2f(m[i] - top) : 0.0f;
    }
    if constexpr (SPLIT) {
      __syncthreads();  // (the parts are read)
    } else {
      // (a lane row without a query: its factor would meet no finite score)
      out.template write<true>([&](int n, int i) {
        return 4 * i + kg < a.group ? scores[((n * kWaves + wave) * NI + i) * 64 + lane] * f[i] : 0.0f;
      });
    }
  }
}

// Split contexts: the weights from the kept scores and the units' maxima and sums.
template <int NI>
__global__ __launch_bounds__(kThreads) void weights_finish_kernel(WeightArgs a) {
  constexpr int Q = 4 * NI;  // queries
  constexpr int kHeld = 4 * TileWeights<NI>::kHeld;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), kg = lane >> 4;
  int pair, x;
  place_of(a, pair, x);
  const int seq = (a.pair0 + pair) / a.num_kv_heads, h = (a.pair0 + pair) % a.num_kv_heads;
  const Seq sq = seq_of(a, seq);
  const int units = (int)(((int64_t)sq.keys + a.unit - 1) / a.unit);
  if (x >= units) return;
  const f32x2* ml = a.ws_ml + (int64_t)pair * a.max_units * Q + lane % Q;
  float mi[NI], li[NI];
  for (int u = x; u < units; u += a.grid_units) {
    const int k0 = u * a.unit, k1 = min(sq.keys, k0 + a.unit);
    const WaveTiles w(a, seq, k0, k1, wave);
    // the wave's scores (a unit is 1024 keys: all of them)
    const float* kept = a.ws_t + ((int64_t)pair * a.max_units + u) * (a.unit / 16) * NI * 64 + lane;
    float t[kHeld][NI];
#pragma unroll
    for (int n = 0; n < kHeld; ++n)
#pragma unroll
      for (int i = 0; i < NI; ++i) t[n][i] = kept[((min(n, max(w.num - 1, 0)) * kWaves + wave) * NI + i) * 64];
    const TileWeights<NI> out(a, w, sq.first, h);
    if (u == x) {
      // a lane's query is lane % Q, its units every 64 / Q-th
      float m = kNegBig, l = 0.0f;
      for (int v = lane / Q; v < units; v += 64 / Q) {
        const f32x2 part = ml[(int64_t)v * Q];
        const float top = fmaxf(m, part[0]);
        l = l * __builtin_amdgcn_exp2f(m - top) + part[1] * __builtin_amdgcn_exp2f(part[0] - top);
        m = top;
      }
#pragma unroll
      for (int o = Q; o < 64; o <<= 1) {
        const float m2 = __shfl_xor(m, o), l2 = __shfl_xor(l, o), top = fmaxf(m, m2);
        l = l * __builtin_amdgcn_exp2f(m - top) + l2 * __builtin_amdgcn_exp2f(m2 - top);
        m = top;
      }
      l = inverse(l);
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        mi[i] = __shfl(m, 4 * i + kg);
        li[i] = __shfl(l, 4 * i + kg);
      }
    }
    out.template write<false>([&](int n, int i) {
      return 4 * i + kg < a.group ? __builtin_amdgcn_exp2f(t[n][i] - mi[i]) * li[i] : 0.0f;
    });
  }
}

// ---------------------------------------------------------------------------
// Chunks.  LDS tiles: rows as they are in memory, 16-byte chunk i of row r at i ^
// swz(r), so that 16 rows' reads of one chunk meet no bank twice.  Lane (c, h) reads
// its row's chunks 2 s + h.
// ---------------------------------------------------------------------------
template <int RB>
struct Rows {
  static constexpr int kChunks = RB / 16;
  static constexpr int kPerDma = 1024 / RB;  // rows of a wave's load
  MKV_DEV static int swz(int r) {
    return RB >= 256 ? r & 15 : RB == 128 ? r >> 1 & 7 : r >> 2 & 3;
  }
  MKV_DEV static int offset(int r, int chunk) { return r * RB + ((chunk ^ swz(r)) << 4); }
};

MKV_DEV void dma16(__amdgpu_buffer_rsrc_t r, char* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
}
template <int N>
MKV_DEV void wait_vm() {  // all but the wave's last N vector memory operations are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 0xf70 | (N >> 4 << 14));
  asm volatile("" ::: "memory");
}
// The workgroup's waves meet, their LDS operations done; loads stay in flight.
MKV_DEV void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
MKV_DEV int div_group(const WeightArgs& a, int r) { return a.group == 1 ? r : (int)__umulhi((uint32_t)r, a.inv_group); }

// Sums over the wave's lanes up to each, by DPP moves.
MKV_DEV int wave_scan(int x) {
  auto add = [&](auto ctrl, auto rows) {
    x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
  };
  using All = std::integral_constant<int, 0xf>;
  add(std::integral_constant<int, 0x111>{}, All{});  // row_shr 1, 2, 4, 8
  add(std::integral_constant<int, 0x112>{}, All{});
  add(std::integral_constant<int, 0x114>{}, All{});
  add(std::integral_constant<int, 0x118>{}, All{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});  // row_bcast 15, 31
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return x;
}
MKV_DEV double wave_scan(double x) {  // (whole numbers: exact)
  auto add = [&](auto ctrl, auto rows) {
    const int64_t b = __builtin_bit_cast(int64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)b, decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(b >> 32), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    x += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  };
  using All = std::integral_constant<int, 0xf>;
  add(std::integral_constant<int, 0x111>{}, All{});
  add(std::integral_constant<int, 0x112>{}, All{});
  add(std::integral_constant<int, 0x114>{}, All{});
  add(std::integral_constant<int, 0x118>{}, All{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return x;
}
MKV_DEV int64_t lane64(int64_t x, int l) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
                   (uint32_t)__builtin_amdgcn_readlane((int)x, l));
}
MKV_DEV double lane64(double x, int l) { return __builtin_bit_cast(double, lane64(__builtin_bit_cast(int64_t, x), l)); }
// Which of the sequences' parts (sequence q has parts(q)) number i is: the sequence
// and its place in it; false past the last.  Every wave works it out alike, a lane a
// sequence, so that workgroups' numbers have no gaps.
struct Place {
  int seq, at, parts;
  int first;  // number of the sequence's first part
  Seq q;
};
template <class F>
MKV_DEV bool find_part(const WeightArgs& a, int i, Place& p, F parts) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    const Seq q = seq_of(a, min(s0 + lane, a.num_seqs - 1));
    const int n = s0 + lane < a.num_seqs ? parts(q) : 0, upto = base + wave_scan(n);
    const uint64_t mine = __builtin_amdgcn_ballot_w64(i >= upto - n && i < upto);
    if (mine) {
      const int l = __builtin_ctzll(mine);
      p.seq = s0 + l;
      p.parts = __builtin_amdgcn_readlane(n, l);
      p.first = __builtin_amdgcn_readlane(upto, l) - p.parts;
      p.at = i - p.first;
      p.q = Seq{lane64(q.q0, l), lane64(q.n, l), lane64(q.first, l), __builtin_amdgcn_readlane(q.keys, l)};
      return true;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

template <class F>
MKV_DEV int count_parts(const WeightArgs& a, F parts) {
  const int lane = threadIdx.x & 63;
  int total = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    const Seq q = seq_of(a, min(s0 + lane, a.num_seqs - 1));
    total += __builtin_amdgcn_readlane(wave_scan(s0 + lane < a.num_seqs ? parts(q) : 0), 63);
  }
  return total;
}

template <int KV, int CT, int D>
struct Formats {
  static constexpr bool kF32 = KV == MKV_DTYPE_F32, kCodes = DTypeInfo<KV>::kBytes == 1;
  static constexpr int kEb = DTypeInfo<KV>::kBytes;
  static constexpr int kQb = kF32 ? 4 : 2;
  static constexpr int kOps = kF32 ? D / 8 : D / 16;  // 16-byte operands of a lane's row of 32
  static constexpr int kBlocks = kF32 ? 1 : 2;        // blocks of 32 that a wave holds
};

// N MFMAs with V vector operations after each: what the scheduler is asked for where
// products stand beside another block's exponentials.
template <int N, int V>
MKV_DEV void mix() {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x402, V, 0);
  }
}

// S[b] = A B[b]^T of blocks of 32 rows, from their operands.
template <bool F32, int CT, int NB, int N>
MKV_DEV void products(const u32x4 (&A)[N], const u32x4 (&B)[NB][N], f32x16 (&S)[NB]) {
#pragma unroll
  for (int b = 0; b < NB; ++b) S[b] = f32x16{};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          S[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(A[i][e]), __uint_as_float(B[b][i][e]), S[b], 0, 0, 0);
    } else {
#pragma unroll
      for (int b = 0; b < NB; ++b) S[b] = mfma32<CT>(A[i], B[b][i], S[b]);
    }
  }
}

// A tile of K, a block of 32 at least for every group of waves that shares it out;
// three tiles' room, so that loads have two tiles' time.
template <int R>
constexpr int kStreamKeys = R == 1 ? 128 : 64;
constexpr int kMinPiece = 256;  // keys

// The normalisers' work is (block of ROWS rows, its keys) after (block, its keys), in
// the sequences' order, dealt out in even pieces: a piece may end one block and begin
// the next.  Pieces are two workgroups a CU, which run at once (where three tiles take 96 KB
// of LDS, in two rounds: fp32 heads of 128, and 64 rows a block of 16-bit ones); twice,
// three and four times that many took longer.  Block b of a sequence costs what its last
// row sees, in keys x group,
//   E(b) = first group + (b + 1) ROWS,   C(b) = E(0) + .. + E(b - 1),
// and the loads ahead of them as much as kMinPiece keys (64 sequences of 6-11 tokens, 3 or
// 4 rows each: 19 us; without it their blocks share 8 pieces, 46),
// whole numbers that doubles hold exactly.
template <int ROWS, int TILE>
struct Pieces {
  const WeightArgs& a;
  double total = 0.0;
  int num;       // pieces
  Seq own;       // of the lane's sequence (of the first 64)

  MKV_DEV Seq lane_seq(int s0) const {
    return s0 == 0 ? own : seq_of(a, min(s0 + (int)(threadIdx.x & 63), a.num_seqs - 1));
  }
  MKV_DEV int blocks(const Seq& q) const { return (int)((q.n * a.group + ROWS - 1) / ROWS); }
  MKV_DEV double cost(const Seq& q, int b) const {  // C(b)
    return (double)b * ((double)max(q.first, (int64_t)0) * a.group + 0.5 * ROWS * (b + 1) + ahead());
  }
  MKV_DEV double start(int i) const { return i >= num ? total : floor(total * i / num); }
  MKV_DEV double ahead() const { return (double)a.group * kMinPiece; }  // of a block, whatever its keys
  MKV_DEV explicit Pieces(const WeightArgs& args) : a(args) {
    const int lane = threadIdx.x & 63;
    own = seq_of(a, min(lane, a.num_seqs - 1));
    for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
      const Seq q = lane_seq(s0);
      total += lane64(wave_scan(s0 + lane < a.num_seqs ? cost(q, blocks(q)) : 0.0), 63);
    }
    const double most = total / ahead();
    num = uniform(most < a.shares ? (int)most + 1 : a.shares);
  }
  // The sequence in which x lies (x < total): costs and blocks ahead of it.
  MKV_DEV void find(double x, Seq& q, int& seq, double& base, int& base_blocks) const {
    const int lane = threadIdx.x & 63;
    base = 0.0;
    base_blocks = 0;
    for (int s0 = 0;; s0 += 64) {
      const Seq s = lane_seq(s0);
      const bool mine = s0 + lane < a.num_seqs;
      const int n = mine ? blocks(s) : 0;
      const double c = mine ? cost(s, n) : 0.0;
      const double upto = base + wave_scan(c);
      const int upto_n = wave_scan(n);
      const uint64_t here = __builtin_amdgcn_ballot_w64(mine && x < upto);
      if (here || s0 + 64 >= a.num_seqs) {
        // (none: cu_seqlens_q falls, and the sequences' work overlaps past 2^53)
        const int l = here ? __builtin_ctzll(here) : 63;
        seq = min(s0 + l, a.num_seqs - 1);
        q = Seq{here ? lane64(s.q0, l) : 0, lane64(s.n, l), lane64(s.first, l), __builtin_amdgcn_readlane(s.keys, l)};
        base = lane64(upto - c, l);
        base_blocks += __builtin_amdgcn_readlane(upto_n - n, l);
        return;
      }
      base = lane64(upto, 63);
      base_blocks += __builtin_amdgcn_readlane(upto_n, 63);
    }
  }
  // The last block of the sequence that begins at y or ahead of it.
  MKV_DEV int block_of(const Seq& q, double y) const {
    int lo = 0, hi = blocks(q) - 1;
    while (lo < hi) {
      const int mid = lo + (hi - lo + 1) / 2;
      if (cost(q, mid) <= y) lo = mid;
      else hi = mid - 1;
    }
    return uniform(lo);
  }
  // The key at which a piece that begins (ends) y into a block does.
  MKV_DEV int key_of(double y) const { return uniform((int)(max(y - ahead(), 0.0) / a.group) / TILE * TILE); }
};

// The rows' normalisers.  R groups of waves hold different rows, 4 / R take different
// keys of the same.
template <int KV, int CT, int D, int R>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(R == 1 ? 1 : 2))) void weights_lse_kernel(WeightArgs a) {
  using F = Formats<KV, CT, D>;
  using K = Rows<D * F::kEb>;
  constexpr int RB = D * F::kEb, KG = kWaves / R, NQ = F::kBlocks, kRows = 32 * NQ * R;
  constexpr int kStream = kStreamKeys<R>, kOwn = kStream / kWaves, kSubs = kOwn / 16, kDma = 16 * RB / 1024;
  // (arrays by name: reads of one do not wait for the loads into another)
  __shared__ __align__(16) char tile0[kStream * RB], tile1[kStream * RB], tile2[kStream * RB];
  __shared__ __align__(16) float scales[3][F::kCodes ? kStream : 4];
  __shared__ f32x2 joined[KG > 1 ? kWaves : 1][32 * NQ];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 31, hf = lane >> 5, rg = wave % R, kg = wave / R;
  const int h = blockIdx.x % a.num_kv_heads, piece = blockIdx.x / a.num_kv_heads;
  const Pieces<kRows, kStream> work(a);
  if (piece >= work.num) return;
  float mul = a.mul;
  if (a.scale_mode == 1) mul *= load_uniform_f32(a.k_scale);
  // the maximum is of raw scores and wants mul > 0: its sign goes into q (0: q is 0)
  uint32_t sign = 0u, keep = 0xffffffffu;
  if (!(mul > 0.0f) && mul == mul) {
    sign = mul < 0.0f ? (F::kF32 ? 0x80000000u : 0x80008000u) : 0u;
    keep = mul < 0.0f ? keep : 0u;
    mul = mul < 0.0f ? -mul : 1.0f;
  }
  // ---- loads of tiles: a wave its share, sub-tiles of 16 keys never across a block ----
  const int64_t row_bytes = (int64_t)a.num_kv_heads * RB;
  uint32_t voff[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int r = i * K::kPerDma + lane / K::kChunks;
    voff[i] = (uint32_t)(r * row_bytes) + 16 * ((lane % K::kChunks) ^ K::swz(r));
  }
  const double end = work.start(piece + 1);
  for (double x = work.start(piece); x < end;) {
    Seq sq;
    int seq, base_blocks;
    double base;
    work.find(x, sq, seq, base, base_blocks);
    const int block = work.block_of(sq, x - base);
    const double c0 = base + work.cost(sq, block), c1 = base + work.cost(sq, block + 1);
    const bool whole = x <= c0 && end >= c1;
    const int rows = (int)sq.n * a.group;
    const int row0 = block * kRows + rg * 32 * NQ;  // this wave's first
    // keys below limit(r) are seen by row r
    auto limit = [&](int r) { return (int)min(max(sq.first + div_group(a, r) + 1, (int64_t)0), (int64_t)sq.keys); };
    const int k_end = limit(min(block * kRows + kRows, rows) - 1);
    const int kb0 = min(work.key_of(x - c0), k_end), k1 = end >= c1 ? k_end : min(work.key_of(end - c0), k_end);
    x = c1 > x ? c1 : end;  // (no end of a block ahead: as below)
    const bool active = row0 < rows;
    const int low = active ? limit(row0) : 0, high = active ? limit(min(row0 + 32 * NQ, rows) - 1) : 0;
    u32x4 q[NQ][F::kOps];
    int lim[NQ];
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      const int r = row0 + 32 * b + c;
      const bool ok = r < rows;
      const int tok = div_group(a, ok ? r : 0), j = (ok ? r : 0) - tok * a.group;
      const char* p = a.q + ((sq.q0 + tok) * a.num_heads + h * a.group + j) * (int64_t)(D * F::kQb);
      lim[b] = ok ? limit(r) : 0;
#pragma unroll
      for (int s = 0; s < F::kOps; ++s) {
        const int d = F::kF32 ? 8 * s + 4 * hf : !F::kCodes ? 16 * s + 8 * hf : 16 * (2 * (s >> 1) + hf) + 8 * (s & 1);
        q[b][s] = ld16(p + d * F::kQb);  // (within q for any row)
      }
    }
    // The tile's block entries, a lane a sub-tile, come a tile ahead of its loads.
    auto entries = [&](int kb) -> int {
      const int t = kb + 16 * (lane & (kStream / 16 - 1));
      const int blk = min(t >> a.idx.bs_log2, a.idx.max_blocks - 1);
      return a.idx.block_tables[(int64_t)seq * a.idx.bt_stride + blk];
    };
    // which sub-tiles are there, a bit each
    auto presence = [&](int kb, int e) -> uint32_t {
      const bool ok = kb + 16 * (lane & (kStream / 16 - 1)) < k1 && e >= 0 && e < a.idx.num_blocks;
      return (uint32_t)__builtin_amdgcn_ballot_w64(ok) & ((1u << kStream / 16) - 1);
    };
    float scale_next[3] = {1.0f, 1.0f, 1.0f};
    uint32_t there[3];
    auto issue = [&](int kb, int e, auto nth) MKV_INLINE {
      constexpr int to_tile = decltype(nth)::value;
      char* const to = to_tile == 0 ? tile0 : to_tile == 1 ? tile1 : tile2;
      there[to_tile] = presence(kb, e);
#pragma unroll
      for (int u = 0; u < kSubs; ++u) {
        const int sub = wave * kSubs + u, t = kb + 16 * sub;
        const bool ok = there[to_tile] >> sub & 1;
        const int64_t slot = ok ? ((int64_t)__builtin_amdgcn_readlane(e, sub) << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : 0;
        // (rows past the last read zeros)
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            (void*)(a.k + slot * row_bytes + (int64_t)h * RB), (short)0,
            ok ? (int)((min(k1 - t, 16) - 1) * row_bytes + RB) : 0, 0x00020000);
#pragma unroll
        for (int i = 0; i < kDma; ++i) dma16(r, to + 16 * sub * RB + i * 1024, voff[i]);
      }
      if (F::kCodes && a.scale_mode == 2 && tid < kStream) {
        const int t = kb + tid, slot = t < k1 ? slot_of(a, seq, t) : -1;
        scale_next[to_tile] = slot >= 0 ? a.k_scale[(int64_t)slot * a.num_kv_heads + h] : 0.0f;
      }
    };
    float m[NQ], l[NQ];
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      m[b] = kNegBig;
      l[b] = 0.0f;
    }
    // The scores of 32 keys wait while the next block's products run, so that one
    // wave's matrix and vector operations overlap.
    f32x16 pend[NQ];
#pragma unroll
    for (int b = 0; b < NQ; ++b) pend[b] = kNegInf;  // (adds nothing)
    int pend_key = -0x40000000;  // its first key
    bool pend_lo = true, pend_up = true;
    float pend_scale[F::kCodes ? 16 : 1];
#pragma unroll
    for (int e = 0; e < (F::kCodes ? 16 : 1); ++e) pend_scale[e] = 1.0f;
    auto k_operand = [&](const char* at, u32x4 (&k)[F::kOps]) MKV_INLINE {
      if constexpr (!F::kCodes) {
#pragma unroll
        for (int s = 0; s < F::kOps; ++s) k[s] = *reinterpret_cast<const u32x4*>(at + K::offset(c, 2 * s + hf));
      } else {
#pragma unroll
        for (int s = 0; s < F::kOps; s += 2) {
          const u32x4 w = *reinterpret_cast<const u32x4*>(at + K::offset(c, s + hf));
          k[s] = codes_to_16<KV, CT>(w[0], w[1]);
          k[s + 1] = codes_to_16<KV, CT>(w[2], w[3]);
        }
      }
    };
    auto softmax = [&](auto masked) MKV_INLINE {  // of what waits
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        f32x16& s = pend[b];
        if (F::kCodes && a.scale_mode == 2) {
#pragma unroll
          for (int e = 0; e < 16; ++e) s[e] *= pend_scale[F::kCodes ? e : 0];
        }
        if constexpr (decltype(masked)::value) {
          const int lm = min(lim[b], k1) - pend_key - 4 * hf;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int kl = 8 * (e >> 2) + (e & 3);
            s[e] = kl < lm && (e < 8 ? pend_lo : pend_up) ? s[e] : kNegInf;
          }
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, other_half(mx));
        mx = fmaxf(mx * mul, kNegBig);
        const float m_new = mx > m[b] + kRescaleSlack ? mx : m[b];
        l[b] *= __builtin_amdgcn_exp2f(m[b] - m_new);
        m[b] = m_new;
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          sum0 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], mul, -m[b]));
          sum1 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], mul, -m[b]));
        }
        l[b] += sum0 + sum1;
      }
    };
    auto needs_mask = [&] { return pend_key + 32 > min(low, k1) || !pend_lo || !pend_up; };
    auto attend = [&](const char* at, const float* sc, int key0, bool lo_there, bool up_there) MKV_INLINE {
      u32x4 k[F::kOps];
      k_operand(at, k);
      f32x16 s[NQ];
      if (needs_mask()) {
        products<F::kF32, CT, NQ>(k, q, s);
        softmax(std::true_type{});
      } else {  // (one basic block: the products among the exponentials)
        products<F::kF32, CT, NQ>(k, q, s);
        softmax(std::false_type{});
        mix<F::kF32 ? 64 : NQ * F::kOps, F::kF32 ? 2 : 8>();
      }
#pragma unroll
      for (int b = 0; b < NQ; ++b) pend[b] = s[b];
      pend_key = key0;
      pend_lo = lo_there;
      pend_up = up_there;
      if (F::kCodes && a.scale_mode == 2) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 y = *reinterpret_cast<const f32x4*>(sc + 8 * g + 4 * hf);
#pragma unroll
          for (int e = 0; e < 4; ++e) pend_scale[F::kCodes ? 4 * g + e : 0] = y[e];
        }
      }
    };
    int e_next = 0;
    auto step = [&](int kb, auto nth) MKV_INLINE {
      constexpr int n = decltype(nth)::value;
      if (kb >= k1) return;
      const char* const tile = n == 0 ? tile0 : n == 1 ? tile1 : tile2;
      if (kb + kStream < k1)
        wait_vm<kSubs * kDma>();  // (the next tile's loads may be on their way)
      else
        wait_vm<0>();
      if (F::kCodes && a.scale_mode == 2 && tid < kStream) scales[n][tid] = scale_next[n];
      meet();  // the tile is here, and everyone is done with the one before
      if (kb + 2 * kStream < k1) {
        const int e = e_next;
        e_next = entries(kb + 3 * kStream);
        issue(kb + 2 * kStream, e, std::integral_constant<int, (n + 2) % 3>{});
      }
#pragma unroll
      for (int kbl0 = 0; kbl0 < kStream / 32; kbl0 += KG) {
        const int kbl = kbl0 + kg, key0 = kb + 32 * kbl;
        if (kbl >= kStream / 32 || key0 >= min(high, k1)) break;
        attend(tile + 32 * kbl * RB, &scales[n][F::kCodes ? 32 * kbl : 0], key0, there[n] >> 2 * kbl & 1, there[n] >> (2 * kbl + 1) & 1);
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    meet();  // (everyone is done with the block before)
    if (kb0 < k1) {
      const int e0 = entries(kb0), e1 = entries(kb0 + kStream);
      e_next = entries(kb0 + 2 * kStream);
      issue(kb0, e0, I0{});
      if (kb0 + kStream < k1) issue(kb0 + kStream, e1, I1{});
    }
#pragma unroll
    for (int b = 0; b < NQ; ++b)
#pragma unroll
      for (int s = 0; s < F::kOps; ++s) {
        const uint32_t k = row0 + 32 * b + c < rows ? keep : 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) q[b][s][e] = (q[b][s][e] ^ sign) & k;
      }
    for (int kb = kb0; kb < k1; kb += 3 * kStream) {
      step(kb, I0{});
      step(kb + kStream, I1{});
      step(kb + 2 * kStream, I2{});
    }
    softmax(std::true_type{});
#pragma unroll
    for (int b = 0; b < NQ; ++b) l[b] += other_half(l[b]);
    if constexpr (KG > 1) {
      if (hf == 0) {
#pragma unroll
        for (int b = 0; b < NQ; ++b) joined[wave][32 * b + c] = f32x2{m[b], l[b]};
      }
      meet();
      if (kg > 0) continue;
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        float top = m[b], sum = 0.0f;
#pragma unroll
        for (int g = 1; g < KG; ++g) top = fmaxf(top, joined[g * R + rg][32 * b + c][0]);
#pragma unroll
        for (int g = 0; g < KG; ++g) {
          const f32x2 v = joined[g * R + rg][32 * b + c];
          sum += v[1] * __builtin_amdgcn_exp2f(v[0] - top);
        }
        m[b] = top;
        l[b] = sum;
      }
    }
    if (hf) continue;
#pragma unroll
    for (int b = 0; b < NQ; ++b) {
      const int r = row0 + 32 * b + c;
      if (r >= rows) continue;
      if (whole)
        a.lse[(h * a.total_q + sq.q0) * a.group + r] = l[b] == 0.0f ? -kNegInf : m[b] + __builtin_amdgcn_logf(l[b]);
      else if ((uint32_t)(base_blocks + block) < a.row_units)  // (more of them: cu_seqlens_q falls)
        // (pieces and blocks rise together: their sum is a place of its own)
        a.part_ml[((int64_t)(piece + base_blocks + block) * a.num_kv_heads + h) * kRows + r - block * kRows] = f32x2{m[b], l[b]};
    }
  }
}

// Rows whose keys were in several pieces, a workgroup a block of them.
template <int ROWS, int TILE>
__global__ __launch_bounds__(kThreads) void weights_join_kernel(WeightArgs a) {
  const int h = blockIdx.x % a.num_kv_heads, number = blockIdx.x / a.num_kv_heads;
  const Pieces<ROWS, TILE> work(a);
  Place p;
  if (!find_part(a, number, p, [&](const Seq& q) { return work.blocks(q); })) return;
  double base = 0.0;
  for (int s0 = 0; s0 <= p.seq; s0 += 64) {
    const Seq q = work.lane_seq(s0);
    base += lane64(wave_scan(s0 + (int)(threadIdx.x & 63) < p.seq ? work.cost(q, work.blocks(q)) : 0.0), 63);
  }
  const double c0 = base + work.cost(p.q, p.at), c1 = base + work.cost(p.q, p.at + 1);
  // the pieces from `lo` to `hi` have a part of it
  int lo = (int)(c0 / work.total * work.num), hi = (int)(c1 / work.total * work.num);
  while (lo > 0 && work.start(lo) > c0) --lo;
  while (lo + 1 < work.num && work.start(lo + 1) <= c0) ++lo;
  hi = min(hi, work.num - 1);
  while (hi + 1 < work.num && work.start(hi + 1) < c1) ++hi;
  while (hi > lo && work.start(hi) >= c1) --hi;
  const int n = hi - lo + 1;
  if (n == 1) return;
  const int rows = (int)p.q.n * a.group - p.at * ROWS;
  const f32x2* part = a.part_ml + ((int64_t)(lo + number) * a.num_kv_heads + h) * ROWS;
  const int64_t step = (int64_t)a.num_kv_heads * ROWS;
  for (int r = threadIdx.x; r < min(rows, ROWS); r += kThreads) {
    constexpr int kAhead = 8;
    float m = kNegBig, l = 0.0f;
    for (int z0 = 0; z0 < n; z0 += kAhead) {
      f32x2 v[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) v[j] = part[min(z0 + j, n - 1) * step + r];
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (z0 + j < n) {
          const float top = fmaxf(m, v[j][0]);
          l = l * __builtin_amdgcn_exp2f(m - top) + v[j][1] * __builtin_amdgcn_exp2f(v[j][0] - top);
          m = top;
        }
    }
    a.lse[(h * a.total_q + p.q.q0) * a.group + p.at * ROWS + r] = l == 0.0f ? -kNegInf : m + __builtin_amdgcn_logf(l);
  }
}

// The keys' weights.  A workgroup takes an even run of the units of 256 keys (fp32: 128)
// of all sequences, one after another: 4 windows of 32 rows over 8-32k keys 48 us, 3.5
// TB/s, by a workgroup a unit 59 (it finds its sequence, and its pages, first); 8 chunks
// of 512 rows, bound by products and exponentials, 82 and 84.  Runs that end within a
// unit need a kernel more to join them: 86.
template <int KV, int CT, int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void weights_columns_kernel(WeightArgs a) {
  using F = Formats<KV, CT, D>;
  constexpr int RB = D * F::kQb;
  using Q = Rows<RB>;
  constexpr int NK = F::kBlocks, kUnit = 32 * NK * kWaves, kTile = 16384 / RB;  // rows of q a tile: 32, 64 or 128
  constexpr int kDma = kTile / kWaves / Q::kPerDma;
  constexpr int kNorms = kTile > 64 ? kTile / 64 : 1;  // loads of their normalisers
  __shared__ __align__(16) char tile0[kTile * RB], tile1[kTile * RB], tile2[kTile * RB];
  __shared__ __align__(16) float norm0[64 * kNorms], norm1[64 * kNorms], norm2[64 * kNorms];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 31, hf = lane >> 5;
  float mul0 = a.mul;
  if (a.scale_mode == 1) mul0 *= load_uniform_f32(a.k_scale);
  auto units_of = [&](const Seq& q) { return (q.keys + kUnit - 1) / kUnit; };
  const int h = blockIdx.x % a.num_kv_heads, i = blockIdx.x / a.num_kv_heads, shares = gridDim.x / a.num_kv_heads;
  const int64_t total = count_parts(a, units_of);
  const int begin = (int)(total * i / shares), end = (int)(total * (i + 1) / shares);
  Place place;
  if (begin == end || !find_part(a, begin, place, units_of)) return;
  int seq = place.seq, unit = place.at, units = place.parts;
  Seq sq = place.q;
  for (int left = end - begin; left; --left, ++unit) {
    if (unit >= units) {  // on to the next sequence with any
      do {
        sq = seq_of(a, ++seq);
        units = units_of(sq);
      } while (units == 0 && seq + 1 < a.num_seqs);
      unit = 0;
    }
    const int rows = (int)sq.n * a.group;
    const int unit0 = unit * kUnit, key0 = unit0 + wave * 32 * NK;  // this wave's first key
    // ---- this lane's keys ----
    u32x4 k[NK][F::kOps];
    float mul[NK], sum[NK], old[NK];
    int slot[NK];
#pragma unroll
    for (int b = 0; b < NK; ++b)
      slot[b] = a.idx.block_tables[(int64_t)seq * a.idx.bt_stride + (min(key0 + 32 * b + c, sq.keys - 1) >> a.idx.bs_log2)];
#pragma unroll
    for (int b = 0; b < NK; ++b) {
      const int t = key0 + 32 * b + c;
      slot[b] = t < sq.keys && slot[b] >= 0 && slot[b] < a.idx.num_blocks
                    ? (slot[b] << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : -1;
      const int64_t row = (int64_t)max(slot[b], 0) * a.num_kv_heads + h;
      const char* p = a.k + row * (int64_t)(D * F::kEb);
#pragma unroll
      for (int s = 0; s < F::kOps; ++s) {
        if constexpr (F::kEb >= 2) {
          k[b][s] = ld16(p + 16 * (2 * s + hf));
        } else {
          const u32x2 w = ld8(p + 8 * (2 * s + hf));
          k[b][s] = codes_to_16<KV, CT>(w[0], w[1]);
        }
      }
      mul[b] = a.scale_mode == 2 ? mul0 * a.k_scale[row] : mul0;
      old[b] = a.decay != 0.0f ? a.weights[row] : 0.0f;
      sum[b] = 0.0f;
    }
    // ---- key t is seen by the rows from (t - first) group on: those that see any of
    // the unit's keys, and each lane's keys' first ----
    auto first_row = [&](int t) {
      return (int)min(max((int64_t)t - sq.first, (int64_t)0) * a.group, (int64_t)0x7fffffff);
    };
    const int r_begin = min(first_row(unit0), rows) / kTile * kTile;
    const int none = first_row(key0), all = first_row(key0 + 32 * NK - 1);
    int from[NK];
#pragma unroll
    for (int b = 0; b < NK; ++b) from[b] = first_row(key0 + 32 * b + c);
    const int64_t norms = (h * a.total_q + sq.q0) * a.group;
    auto issue = [&](int r0, auto nth) {
      constexpr int n = decltype(nth)::value;
      char* const to = n == 0 ? tile0 : n == 1 ? tile1 : tile2;
      float* const to_norm = n == 0 ? norm0 : n == 1 ? norm1 : norm2;
      const int tok0 = div_group(a, r0), tok1 = div_group(a, min(r0 + kTile, rows) - 1);
      const int64_t head = (sq.q0 + tok0) * a.num_heads + h * a.group;  // tok0's first row
      const __amdgpu_buffer_rsrc_t r =
          __builtin_amdgcn_make_buffer_rsrc((void*)(a.q + head * RB), (short)0,
                                            ((tok1 - tok0) * a.num_heads + a.group) * RB, 0x00020000);
#pragma unroll
      for (int i = 0; i < kDma; ++i) {
        const int in = wave * (kTile / kWaves) + i * Q::kPerDma + lane / Q::kChunks;
        const int row = r0 + in, tok = div_group(a, row);
        const uint32_t off = (uint32_t)(((tok - tok0) * a.num_heads + row - tok * a.group) * RB) +
                             16 * ((lane % Q::kChunks) ^ Q::swz(in));
        // (rows past the last read zeros)
        dma16(r, to + (wave * (kTile / kWaves) + i * Q::kPerDma) * RB, row < rows ? off : 0x7ffffff0u);
      }
      // (every wave loads the same normalisers to the same place, and counts as many)
      const __amdgpu_buffer_rsrc_t ln = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(a.lse + norms + r0), (short)0, min(rows - r0, kTile) * 4, 0x00020000);
#pragma unroll
      for (int i = 0; i < kNorms; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(ln, (__attribute__((address_space(3))) void*)(to_norm + 64 * i), 4,
                                                 4 * lane + 256 * i, 0, 0, 0);
    };
    // 32 rows of q from row0 on against this wave's keys
    auto attend = [&](const char* at, const float* norm_at, int row0, auto masked) {
      u32x4 q[F::kOps];
#pragma unroll
      for (int s = 0; s < F::kOps; ++s) q[s] = *reinterpret_cast<const u32x4*>(at + Q::offset(c, 2 * s + hf));
      f32x4 norm[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) norm[g] = *reinterpret_cast<const f32x4*>(norm_at + 8 * g + 4 * hf);
      f32x16 s[NK];
      products<F::kF32, CT, NK>(q, k, s);
#pragma unroll
      for (int b = 0; b < NK; ++b) {
        float p[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][e], mul[b], -norm[e >> 2][e & 3]));
        if constexpr (decltype(masked)::value) {
          const int lo = from[b] - row0 - 4 * hf, hi = rows - row0 - 4 * hf;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int r = 8 * (e >> 2) + (e & 3);
            p[e] = r >= lo && r < hi ? p[e] : 0.0f;
          }
        }
        float s0 = p[0], s1 = p[1];
#pragma unroll
        for (int e = 2; e < 16; e += 2) {
          s0 += p[e];
          s1 += p[e + 1];
        }
        sum[b] += s0 + s1;
      }
    };
    auto step = [&](int r0, auto nth) {
      constexpr int n = decltype(nth)::value;
      if (r0 >= rows) return;
      if (r0 + kTile < rows)
        wait_vm<kDma + kNorms>();  // (the next tile's loads may be on their way)
      else
        wait_vm<0>();
      meet();  // the tile is here, and everyone is done with the one before
      if (r0 + 2 * kTile < rows) issue(r0 + 2 * kTile, std::integral_constant<int, (n + 2) % 3>{});
#pragma unroll
      for (int rb = 0; rb < kTile / 32; ++rb) {
        const int row0 = r0 + 32 * rb;
        if (row0 >= rows || row0 + 31 < none) continue;
        const char* const at = (n == 0 ? tile0 : n == 1 ? tile1 : tile2) + 32 * rb * RB;
        const float* const norm_at = (n == 0 ? norm0 : n == 1 ? norm1 : norm2) + 32 * rb;
        if (row0 < all || row0 + 32 > rows)
          attend(at, norm_at, row0, std::true_type{});
        else
          attend(at, norm_at, row0, std::false_type{});
      }
    };
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    meet();  // (everyone is done with the unit before)
    if (r_begin < rows) issue(r_begin, I0{});
    if (r_begin + kTile < rows) issue(r_begin + kTile, I1{});
    for (int r0 = r_begin; r0 < rows; r0 += 3 * kTile) {
      step(r0, I0{});
      step(r0 + kTile, I1{});
      step(r0 + 2 * kTile, I2{});
    }
#pragma unroll
    for (int b = 0; b < NK; ++b) {
      const float w = sum[b] + other_half(sum[b]);
      // (tokens that came with these rows start here, whatever lay there)
      if (hf == 0 && slot[b] >= 0)
        a.weights[(int64_t)slot[b] * a.num_kv_heads + h] =
            a.decay != 0.0f && key0 + 32 * b + c < sq.first ? __builtin_fmaf(a.decay, old[b], w) : w;
    }
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
int log2_exact(int64_t v) {
  if (v <= 0 || (v & (v - 1))) return -1;
  int l = 0;
  while (((int64_t)1 << l) < v) ++l;
  return l;
}

struct Plan {
  bool decode;
  // decode
  int ni, unit, max_units, grid_units;
  int pairs;                     // (sequence, KV head) pairs of a launch
  // chunks
  int row_groups, rows, shares;  // rows: of a block
  int64_t row_units;             // blocks at most
  int column_grid;
  size_t bytes;
};

// Bytes of kept scores at a time.  Their room follows the table's width, which may be far
// past the contexts, so that pairs whose scores do not fit go in up to four turns (60
// sequences of 300-800 tokens, 16/8 heads, fp8, under tables of 131,072: 75 us, and 42 in
// one turn with 0.94 GiB; of 30k tokens, 32/8, bf16, 929 and 906).  Past those, one-row sequences go
// the chunks' way, which keeps no scores.
constexpr size_t kMaxScores = (size_t)256 << 20;
constexpr int kMaxTurns = 4;

Plan make_plan(int num_seqs, int64_t total_q, int heads, int kv_heads, int64_t capacity, bool one_row, bool f32) {
  Plan p{};
  const int group = heads / kv_heads;
  const int64_t pairs = (int64_t)num_seqs * kv_heads;
  if (one_row) {
    p.ni = group <= 4 ? 1 : 4;
    const int most = 4096 / p.ni;  // 64 KB of scores: two workgroups a CU
    p.unit = capacity <= most ? (int)((capacity + 15) / 16 * 16) : kSplitKeys;
    p.max_units = (int)((capacity + p.unit - 1) / p.unit);
    const int64_t room = 16384 / pairs;
    p.grid_units = (int)(p.max_units < room ? p.max_units : room < 1 ? 1 : room);
    const size_t each = p.max_units > 1 ? (size_t)p.max_units * 4 * p.ni * (8 + (size_t)p.unit * 4) : 0;
    if (each <= kMaxScores && (size_t)pairs * each <= kMaxTurns * kMaxScores) {
      const int64_t fit = each ? (int64_t)(kMaxScores / each) : pairs, turns = (pairs + fit - 1) / fit;
      p.pairs = (int)((pairs + turns - 1) / turns);
      p.bytes = (size_t)p.pairs * each;
      p.decode = true;
      return p;
    }
  }
  const int held = f32 ? 32 : 64;  // rows of a wave
  const int64_t rows = total_q * group, mean = rows / num_seqs;
  p.row_groups = mean <= held && !f32 ? 1 : mean <= 2 * held ? 2 : 4;
  p.rows = held * p.row_groups;
  p.row_units = num_seqs + rows / p.rows;
  // pieces for two workgroups a CU
  p.shares = (int)(512 / kv_heads > 0 ? 512 / kv_heads : 1);
  const int unit = f32 ? 128 : 256;
  const int64_t units = (int64_t)num_seqs * ((capacity + unit - 1) / unit);
  p.column_grid = (int)(units < p.shares ? units : p.shares) * kv_heads;
  p.bytes = (size_t)total_q * heads * 4 + (size_t)(p.row_units + p.shares) * kv_heads * p.rows * 8;
  p.bytes = (p.bytes + 15) / 16 * 16;
  return p;
}

template <int KV, int CT, int D>
int launch_weights(WeightArgs& a, const Plan& p, hipStream_t s) {
  if (p.decode) {
    const size_t lds = (size_t)p.unit / 16 * p.ni * 64 * 4;
    const int64_t pairs = (int64_t)a.num_seqs * a.num_kv_heads;
    for (int64_t pair0 = 0; pair0 < pairs; pair0 += p.pairs) {
      const dim3 grid((unsigned)((pairs - pair0 < p.pairs ? pairs - pair0 : p.pairs) * p.grid_units));
      a.pair0 = (int)pair0;
      if (p.max_units == 1) {
        if (p.ni == 1)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_decode_kernel<KV, CT, D, 1, false>), grid, dim3(kThreads), lds, s, a);
        else
          hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_decode_kernel<KV, CT, D, 4, false>), grid, dim3(kThreads), lds, s, a);
      } else {
        if (p.ni == 1)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_decode_kernel<KV, CT, D, 1, true>), grid, dim3(kThreads), lds, s, a);
        else
          hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_decode_kernel<KV, CT, D, 4, true>), grid, dim3(kThreads), lds, s, a);
        if (hipError_t e = hipGetLastError()) return (int)e;
        if (p.ni == 1)
          hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_finish_kernel<1>), grid, dim3(kThreads), 0, s, a);
        else
          hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_finish_kernel<4>), grid, dim3(kThreads), 0, s, a);
      }
      if (hipError_t e = hipGetLastError()) return (int)e;
    }
    return MKV_OK;
  }
  auto normalisers = [&](auto groups) {
    constexpr int R = decltype(groups)::value, kRows = 32 * Formats<KV, CT, D>::kBlocks * R;
    const dim3 grid((unsigned)(p.shares * a.num_kv_heads));
    hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_lse_kernel<KV, CT, D, R>), grid, dim3(kThreads), 0, s, a);
    if (hipError_t e = hipGetLastError()) return (int)e;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_join_kernel<kRows, kStreamKeys<R>>),
                       dim3((unsigned)(p.row_units * a.num_kv_heads)), dim3(kThreads), 0, s, a);
    return (int)hipGetLastError();
  };
  int st = 0;
  if (p.row_groups == 4) {
    st = normalisers(std::integral_constant<int, 4>{});
  } else if (p.row_groups == 2) {
    st = normalisers(std::integral_constant<int, 2>{});
  } else {
    if constexpr (KV != MKV_DTYPE_F32)  // (three of its tiles would not fit the LDS)
      st = normalisers(std::integral_constant<int, 1>{});
  }
  if (st) return st;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_columns_kernel<KV, CT, D>), dim3((unsigned)p.column_grid), dim3(kThreads), 0, s, a);
  return (int)hipGetLastError();
}

template <int KV, int CT>
int launch_dim(WeightArgs& a, const Plan& p, int head_dim, hipStream_t s) {
  return head_dim == 64 ? launch_weights<KV, CT, 64>(a, p, s) : launch_weights<KV, CT, 128>(a, p, s);
}

constexpr int64_t kMaxGrid = 0xffffff;  // workgroups of 256 threads: below 2^32 threads

int check_weights(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
                  int max_blocks, int one_row) {
  if (num_seqs < 0 || total_q < 0 || num_heads <= 0 || num_kv_heads <= 0 || num_kv_heads > (1 << 16) || max_blocks < 0)
    return MKV_ERR_BAD_SHAPE;
  if (head_dim != 64 && head_dim != 128) return MKV_ERR_UNSUPPORTED_HEAD_DIM;
  const int g = num_heads / num_kv_heads;
  if (num_heads % num_kv_heads || g < 1 || g > 16) return MKV_ERR_UNSUPPORTED_GROUP;
  if (log2_exact(block_size) < 4) return MKV_ERR_BAD_BLOCK_SIZE;
  // (a tile's rows of q lie within 2^31 bytes; rows of a KV head and keys are counted
  // in 32 bits, row / group by a product)
  if (num_heads > 8192 || total_q * g >= (1 << 28) || (int64_t)max_blocks * block_size > 0x7fff0000 ||
      (int64_t)num_seqs * (((int64_t)max_blocks * block_size + 127) / 128) > 0x7fffffff)
    return MKV_ERR_BAD_SHAPE;
  if ((int64_t)num_seqs * num_kv_heads > kMaxGrid || total_q * num_heads > kMaxGrid * kThreads) return MKV_ERR_BAD_SHAPE;
  if (one_row && total_q != num_seqs) return MKV_ERR_BAD_SHAPE;
  return MKV_OK;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_paged_weights_workspace_size(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads,
                                                   int head_dim, int block_size, int max_blocks, int kv_dtype,
                                                   int one_row) {
  if (check_weights(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, one_row)) return 0;
  if (num_seqs == 0 || max_blocks == 0) return 0;
  return make_plan(num_seqs, total_q, num_heads, num_kv_heads, (int64_t)max_blocks * block_size, one_row != 0,
                   kv_dtype == MKV_DTYPE_F32)
      .bytes;
}

extern "C" int mkv_paged_weights(float* weights, float decay, const void* q, int q_dtype, const void* k_cache,
                                 int kv_dtype, int64_t num_blocks, const float* k_scale, int kv_scale_mode,
                                 const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                                 const void* context_lens, int context_lens_dtype, const int32_t* cu_seqlens_q,
                                 int num_seqs, int64_t total_q, int num_heads, int num_kv_heads, int head_dim,
                                 int block_size, float sm_scale, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const int one_row = cu_seqlens_q == nullptr;
  if (int st = check_weights(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, one_row)) return st;
  if (num_blocks < 0 || num_blocks * block_size > 0x7fffffff) return MKV_ERR_BAD_SHAPE;
  const bool code = kv_dtype == MKV_DTYPE_FP8E4M3 || kv_dtype == MKV_DTYPE_I8;
  const bool token = code && kv_scale_mode == MKV_SCALE_PER_TOKEN_HEAD;
  if (kv_scale_mode != MKV_SCALE_PER_TENSOR && kv_scale_mode != MKV_SCALE_PER_TOKEN_HEAD) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (!code && kv_dtype != MKV_DTYPE_F32 && kv_dtype != MKV_DTYPE_BF16 && kv_dtype != MKV_DTYPE_F16) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (code ? q_dtype != MKV_DTYPE_BF16 && q_dtype != MKV_DTYPE_F16 : q_dtype != kv_dtype) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (kv_dtype == MKV_DTYPE_I8 && !token) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (context_lens_dtype != MKV_INDEX_I32 && context_lens_dtype != MKV_INDEX_I64) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (num_seqs == 0 || max_blocks == 0 || num_blocks == 0) return MKV_OK;
  if (!weights || (total_q && !q) || !k_cache || !block_tables || !context_lens || (code && !k_scale)) return MKV_ERR_NULL_POINTER;
  if (bt_stride < max_blocks) return MKV_ERR_BAD_STRIDE;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(workspace)) & 15u ||
      reinterpret_cast<uintptr_t>(weights) & 3u)
    return MKV_ERR_MISALIGNED;
  const Plan p = make_plan(num_seqs, total_q, num_heads, num_kv_heads, (int64_t)max_blocks * block_size, one_row != 0,
                           kv_dtype == MKV_DTYPE_F32);
  if (p.bytes > workspace_bytes || (p.bytes && !workspace)) return MKV_ERR_WORKSPACE_TOO_SMALL;
  if (p.decode ? (int64_t)p.pairs * p.grid_units > kMaxGrid : p.row_units * num_kv_heads > kMaxGrid) return MKV_ERR_BAD_SHAPE;
  // (the pieces' work, in doubles, is exact)
  const int64_t group = num_heads / num_kv_heads;
  if (!p.decode && (double)p.row_units * (double)(((int64_t)max_blocks * block_size + kMinPiece + total_q) * group + p.rows) >= 0x1p52)
    return MKV_ERR_BAD_SHAPE;
  WeightArgs a;
  a.q = reinterpret_cast<const char*>(q);
  a.k = reinterpret_cast<const char*>(k_cache);
  a.k_scale = k_scale;
  a.weights = weights;
  a.idx = PagedIndex{block_tables, bt_stride, max_blocks, num_blocks, log2_exact(block_size),
                     (int64_t)num_kv_heads * head_dim};
  a.ctx = context_lens;
  a.ctx_i64 = context_lens_dtype == MKV_INDEX_I64;
  a.cu = cu_seqlens_q;
  a.num_seqs = num_seqs;
  a.total_q = total_q;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads;
  a.inv_group = (uint32_t)((((uint64_t)1 << 32) + a.group - 1) / a.group);
  a.mul = sm_scale * kLog2e;
  a.scale_mode = token ? 2 : code ? 1 : 0;
  a.decay = decay;
  a.unit = p.unit;
  a.grid_units = p.grid_units;
  a.max_units = p.max_units;
  a.pair0 = 0;
  a.ws_ml = reinterpret_cast<f32x2*>(workspace);
  a.ws_t = reinterpret_cast<float*>(a.ws_ml + (p.decode ? (size_t)p.pairs * p.max_units * 4 * p.ni : 0));
  a.shares = p.shares;
  a.row_units = p.row_units;
  a.part_ml = reinterpret_cast<f32x2*>(workspace);
  a.lse = reinterpret_cast<float*>(a.part_ml + (p.decode ? 0 : (size_t)(p.row_units + p.shares) * num_kv_heads * p.rows));
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const bool half = q_dtype == MKV_DTYPE_F16;
  switch (kv_dtype) {
    case MKV_DTYPE_F32: return launch_dim<MKV_DTYPE_F32, MKV_DTYPE_F16>(a, p, head_dim, s);
    case MKV_DTYPE_BF16: return launch_dim<MKV_DTYPE_BF16, MKV_DTYPE_BF16>(a, p, head_dim, s);
    case MKV_DTYPE_F16: return launch_dim<MKV_DTYPE_F16, MKV_DTYPE_F16>(a, p, head_dim, s);
    case MKV_DTYPE_FP8E4M3:
      return half ? launch_dim<MKV_DTYPE_FP8E4M3, MKV_DTYPE_F16>(a, p, head_dim, s)
                  : launch_dim<MKV_DTYPE_FP8E4M3, MKV_DTYPE_BF16>(a, p, head_dim, s);
    default:
      return half ? launch_dim<MKV_DTYPE_I8, MKV_DTYPE_F16>(a, p, head_dim, s)
                  : launch_dim<MKV_DTYPE_I8, MKV_DTYPE_BF16>(a, p, head_dim, s);
  }
}
