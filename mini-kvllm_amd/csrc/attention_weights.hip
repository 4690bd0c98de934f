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
// long contexts are split, their scores kept in memory for a second kernel.
//
// Chunks: the normaliser of a row takes all of its keys and the weight of a key all
// of its rows, so scores are computed twice rather than kept: weights_lse_kernel holds
// 64 rows of q a wave in registers and streams K through LDS (S^T = K Q^T, a row's
// maximum and sum in its column's lanes), weights_columns_kernel holds 64 keys a wave
// and streams q (S = Q K^T, a key's sum in its column's lanes).  Neither product's
// result leaves the registers and no sum is shared, so the result is one only.
//
// Products are exact (1-byte codes as 16-bit operands of q's type, fp32 on the fp32
// MFMA), their sums, the softmax and the weights fp32.
#include <type_traits>

#include "mkv_device.hpp"

namespace mkv {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

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
  float* ws_t;         // scores of split contexts
  f32x2* ws_ml;        // (sequence, KV head, unit, query): maximum and sum
  // chunks
  int splits;          // of a row block's keys
  f32x2* part_ml;      // (split, row): maximum and sum
  float* lse;          // (row) log2 of the normaliser, +inf for a row that sees nothing
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
  int64_t first;      // position of row 0
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
  r.first = c - r.n;
  r.keys = (int)min(c, (int64_t)a.idx.max_blocks << a.idx.bs_log2);
  return r;
}
// slot of token t, or -1 (a lane's own)
MKV_DEV int slot_of(const WeightArgs& a, int seq, int t) {
  const int32_t p = a.idx.block_tables[(int64_t)seq * a.idx.bt_stride + (t >> a.idx.bs_log2)];
  return p >= 0 && p < a.idx.num_blocks ? (p << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : -1;
}
MKV_DEV void add_weight(const WeightArgs& a, const Seq& s, int slot, int h, int t, float w) {
  float* const at = a.weights + (int64_t)slot * a.num_kv_heads + h;
  // (tokens that came with these rows start here, whatever lay there)
  if (a.decay != 0.0f && t < s.first) w = __builtin_fmaf(a.decay, *at, w);
  *at = w;
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
  // row `j` of q (j < 0: zeros); kg: the lane's share of the contraction
  MKV_DEV void load(const char* row, bool ok, int kg) {
#pragma unroll
    for (int s = 0; s < kOps; ++s) {
      const int d = KV == MKV_DTYPE_F32 ? 16 * s + 4 * kg
                    : DTypeInfo<KV>::kBytes == 2 ? 32 * s + 8 * kg : 64 * (s >> 1) + 16 * kg + 8 * (s & 1);
      w[s] = u32x4{0, 0, 0, 0};
      if (ok) w[s] = ld16(row + d * (KV == MKV_DTYPE_F32 ? 4 : 2));
    }
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

// The tiles of a wave, four at a time: their weights from e(tile, i), all of the
// wave's lanes writing (lane row kg the kg-th tile's keys).
template <int NI, class E>
MKV_DEV void write_tiles(const WeightArgs& a, const Seq& sq, int seq, int h, int k0, int k1, int tiles, int wave, E e) {
  const int lane = threadIdx.x & 63, c = lane & 15, kg = lane >> 4;
  for (int i0 = 0; i0 * kWaves + wave < tiles; i0 += 4) {
    const int t = k0 + 16 * ((i0 + kg) * kWaves + wave) + c;
    const int slot = t < k1 ? slot_of(a, seq, t) : -1;
    float mine = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float w = 0.0f;
      if ((i0 + j) * kWaves + wave < tiles) {
#pragma unroll
        for (int i = 0; i < NI; ++i) w += e((i0 + j) * kWaves + wave, i);
      }
      w = sum_of_rows(w);
      mine = kg == j ? w : mine;
    }
    if (slot >= 0) add_weight(a, sq, slot, h, t, mine);
  }
}

template <int KV, int CT, int D, int NI>
__global__ __launch_bounds__(kThreads) void weights_decode_kernel(WeightArgs a) {
  using Tile = DecodeTile<KV, CT, D>;
  constexpr int kAhead = KV == MKV_DTYPE_F32 ? 2 : 4;  // tiles of a wave in a batch; two batches in flight
  extern __shared__ float scores[];                    // (tile, i, lane)
  __shared__ float part[2][kWaves][4 * NI];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 15, kg = lane >> 4;
  const int pair = blockIdx.x / a.grid_units, x = blockIdx.x % a.grid_units;
  const int seq = pair / a.num_kv_heads, h = pair % a.num_kv_heads;
  const Seq sq = seq_of(a, seq);
  const int units = (int)(((int64_t)sq.keys + a.unit - 1) / a.unit);
  if (x >= units) return;
  // row r = 4 kg + i of the product is query 4 i + kg of the group
  const int query = 4 * (c & 3) + (c >> 2);
  constexpr int kQBytes = D * (KV == MKV_DTYPE_F32 ? 4 : 2);
  DecodeQ<KV, CT, D> q;
  q.load(a.q + (sq.q0 * a.num_heads + h * a.group + min(query, a.group - 1)) * kQBytes, query < a.group, kg);
  const int64_t row_bytes = (int64_t)a.num_kv_heads * D * Tile::kEb;
  const char* const kbase = a.k + (int64_t)h * D * Tile::kEb + 16 * kg;
  float mul = a.mul;
  if (a.scale_mode == 1) mul *= load_uniform_f32(a.k_scale);
  const bool split = units > 1;
  for (int u = x; u < units; u += a.grid_units) {
    const int k0 = u * a.unit, k1 = min(sq.keys, k0 + a.unit);
    const int tiles = (k1 - k0 + 15) / 16;
    float m[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) m[i] = kNegBig;
    auto load = [&](Tile (&t)[kAhead], uint32_t& here, int i0) {
      here = 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int tile = (i0 + j) * kWaves + wave, key = k0 + 16 * tile;
        if (tile < tiles) {
          const int64_t phys = a.idx.physical_block(seq, key >> a.idx.bs_log2);
          here |= phys >= 0 ? 1u << j : 0u;
          // (keys past the last: the tile's first, which is there)
          const int64_t slot = (max(phys, (int64_t)0) << a.idx.bs_log2) + (key & ((1 << a.idx.bs_log2) - 1)) + (key + c < k1 ? c : 0);
          const char* p = kbase + slot * row_bytes;
#pragma unroll
          for (int i = 0; i < Tile::kLoads; ++i) t[j].w[i] = ld16(p + 64 * i);
          t[j].scale = a.scale_mode == 2 ? a.k_scale[slot * a.num_kv_heads + h] : 1.0f;
        }
      }
    };
    auto take = [&](const Tile (&t)[kAhead], uint32_t here, int i0) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int tile = (i0 + j) * kWaves + wave;
        if (tile < tiles) {
          const f32x4 s = decode_scores<KV, CT, D>(q, t[j]);
          const bool sees = (here >> j & 1) && k0 + 16 * tile + c < k1;
          const float f = mul * t[j].scale;
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            const float v = sees ? s[i] * f : kNegInf;
            m[i] = fmaxf(m[i], v);
            scores[(tile * NI + i) * 64 + lane] = v;
          }
        }
      }
    };
    {
      Tile t0[kAhead], t1[kAhead];
      uint32_t h0, h1;
      load(t0, h0, 0);
      for (int i0 = 0; i0 * kWaves + wave < tiles; i0 += 2 * kAhead) {
        load(t1, h1, i0 + kAhead);
        take(t0, h0, i0);
        load(t0, h0, i0 + 2 * kAhead);
        take(t1, h1, i0 + kAhead);
      }
    }
    // ---- the queries' maxima and sums ----
#pragma unroll
    for (int i = 0; i < NI; ++i) m[i] = row_all(m[i], [](float u, float v) { return fmaxf(u, v); });
    if (c == 0) {
#pragma unroll
      for (int i = 0; i < NI; ++i) part[0][wave][4 * i + kg] = m[i];
    }
    __syncthreads();
    float l[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      for (int v = 0; v < kWaves; ++v) m[i] = fmaxf(m[i], part[0][v][4 * i + kg]);
      l[i] = 0.0f;
    }
    for (int tile = wave; tile < tiles; tile += kWaves)
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        float* const at = scores + (tile * NI + i) * 64 + lane;
        const float e = __builtin_amdgcn_exp2f(*at - m[i]);
        l[i] += e;
        if (split)
          a.ws_t[(((int64_t)pair * a.max_units + u) * (a.unit / 16) * NI + tile * NI + i) * 64 + lane] = *at;
        else
          *at = e;
      }
#pragma unroll
    for (int i = 0; i < NI; ++i) l[i] = row_all(l[i], [](float u, float v) { return u + v; });
    if (c == 0) {
#pragma unroll
      for (int i = 0; i < NI; ++i) part[1][wave][4 * i + kg] = l[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      l[i] = 0.0f;
      for (int v = 0; v < kWaves; ++v) l[i] += part[1][v][4 * i + kg];
    }
    if (split) {
      if (wave == 0 && c == 0) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
          a.ws_ml[((int64_t)pair * a.max_units + u) * 4 * NI + 4 * i + kg] = f32x2{m[i], l[i]};
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) l[i] = 4 * i + kg < a.group ? inverse(l[i]) : 0.0f;
      write_tiles<NI>(a, sq, seq, h, k0, k1, tiles, wave, [&](int tile, int i) {
        // (a query that is none: its factor is 0, its score finite or NaN alone)
        return 4 * i + kg < a.group ? scores[(tile * NI + i) * 64 + lane] * l[i] : 0.0f;
      });
    }
  }
}

// Split contexts: the weights from the kept scores and the units' maxima and sums.
template <int NI>
__global__ __launch_bounds__(kThreads) void weights_finish_kernel(WeightArgs a) {
  constexpr int Q = 4 * NI;  // queries
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), kg = lane >> 4;
  const int pair = blockIdx.x / a.grid_units, x = blockIdx.x % a.grid_units;
  const int seq = pair / a.num_kv_heads, h = pair % a.num_kv_heads;
  const Seq sq = seq_of(a, seq);
  const int units = (int)(((int64_t)sq.keys + a.unit - 1) / a.unit);
  if (x >= units || units <= 1) return;
  // a lane's query is lane % Q, its units every 64 / Q-th
  const f32x2* ml = a.ws_ml + (int64_t)pair * a.max_units * Q + lane % Q;
  float m = kNegBig, l = 0.0f;
  for (int u = lane / Q; u < units; u += 64 / Q) m = fmaxf(m, ml[(int64_t)u * Q][0]);
#pragma unroll
  for (int o = Q; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  for (int u = lane / Q; u < units; u += 64 / Q) {
    const f32x2 v = ml[(int64_t)u * Q];
    l += v[1] * __builtin_amdgcn_exp2f(v[0] - m);
  }
#pragma unroll
  for (int o = Q; o < 64; o <<= 1) l += __shfl_xor(l, o);
  l = inverse(l);
  float mi[NI], li[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    mi[i] = __shfl(m, 4 * i + kg);
    li[i] = __shfl(l, 4 * i + kg);
  }
  for (int u = x; u < units; u += a.grid_units) {
    const int k0 = u * a.unit, k1 = min(sq.keys, k0 + a.unit), tiles = (k1 - k0 + 15) / 16;
    const float* t = a.ws_t + ((int64_t)pair * a.max_units + u) * (a.unit / 16) * NI * 64 + lane;
    write_tiles<NI>(a, sq, seq, h, k0, k1, tiles, wave, [&](int tile, int i) {
      return 4 * i + kg < a.group ? __builtin_amdgcn_exp2f(t[(tile * NI + i) * 64] - mi[i]) * li[i] : 0.0f;
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
MKV_DEV void wait_all() {  // the wave's memory operations are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0);
  asm volatile("" ::: "memory");
}
MKV_DEV int div_group(const WeightArgs& a, int r) { return a.group == 1 ? r : (int)__umulhi((uint32_t)r, a.inv_group); }

// Which of the sequences' parts (s has parts(s)) number `i` is, and its place in it;
// false past the last.  Every wave works it out alike, a lane a sequence.
template <class F>
MKV_DEV bool find_part(int num_seqs, int i, int& seq, int& place, F parts) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += 64) {
    const int n = s0 + lane < num_seqs ? parts(s0 + lane) : 0;
    int upto = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(upto, o);
      if (lane >= o) upto += y;
    }
    upto += base;
    const uint64_t mine = __builtin_amdgcn_ballot_w64(i >= upto - n && i < upto);
    if (mine) {
      const int l = __builtin_ctzll(mine);
      seq = s0 + l;
      place = i - __builtin_amdgcn_readlane(upto - n, l);
      return true;
    }
    base = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

template <int KV, int CT, int D>
struct Formats {
  static constexpr bool kF32 = KV == MKV_DTYPE_F32;
  static constexpr int kEb = DTypeInfo<KV>::kBytes;
  static constexpr int kQb = kF32 ? 4 : 2;
  static constexpr int kOps = kF32 ? D / 8 : D / 16;  // 16-byte operands of a lane's row of 32
  static constexpr int kBlocks = kF32 ? 1 : 2;        // blocks of 32 that a wave holds
};

// S = A B^T of two blocks of 32 rows, from their operands.
template <bool F32, int CT, int N>
MKV_DEV f32x16 product(const u32x4 (&A)[N], const u32x4 (&B)[N]) {
  f32x16 s = f32x16{};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(A[i][e]), __uint_as_float(B[i][e]), s, 0, 0, 0);
    } else {
      s = mfma32<CT>(A[i], B[i], s);
    }
  }
  return s;
}

constexpr int kStreamKeys = 128;  // a tile of K

// The rows' normalisers.  R groups of waves hold different rows, 4 / R take different
// keys of the same; blockIdx.y splits the keys further.
template <int KV, int CT, int D, int R>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void weights_lse_kernel(WeightArgs a) {
  using F = Formats<KV, CT, D>;
  using K = Rows<D * F::kEb>;
  constexpr int RB = D * F::kEb, KG = kWaves / R, NQ = F::kBlocks, kRows = 32 * NQ * R;
  constexpr int kOwn = kStreamKeys / kWaves, kSubs = kOwn / 16, kDma = 16 * RB / 1024;
  __shared__ __align__(16) char tile[2][kStreamKeys * RB];
  __shared__ int there[2][kStreamKeys / 16];
  __shared__ float scales[2][kStreamKeys];
  __shared__ f32x2 joined[KG > 1 ? kWaves : 1][32 * NQ];
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int c = lane & 31, hf = lane >> 5, rg = wave % R, kg = wave / R;
  const int h = blockIdx.x % a.num_kv_heads;
  int seq, block;
  if (!find_part(a.num_seqs, blockIdx.x / a.num_kv_heads, seq, block, [&](int s) {
        const Seq q = seq_of(a, s);
        return (int)((q.n * a.group + kRows - 1) / kRows);
      }))
    return;
  seq = uniform(seq);
  const Seq sq = seq_of(a, seq);
  const int rows = (int)sq.n * a.group;
  const int row0 = block * kRows + rg * 32 * NQ;  // this wave's first
  // keys below limit(r) are seen by row r
  auto limit = [&](int r) { return (int)min(max(sq.first + div_group(a, r) + 1, (int64_t)0), (int64_t)sq.keys); };
  const int k_end = limit(min(block * kRows + kRows, rows) - 1);
  // this split's share of them, whole tiles
  const int share = ((k_end + a.splits - 1) / a.splits + kStreamKeys - 1) / kStreamKeys * kStreamKeys;
  const int kb0 = (int)min((int64_t)blockIdx.y * share, (int64_t)k_end), k1 = (int)min((int64_t)kb0 + share, (int64_t)k_end);
  const bool active = row0 < rows;
  const int low = active ? limit(row0) : 0, high = active ? limit(min(row0 + 32 * NQ, rows) - 1) : 0;
  float mul = a.mul;
  if (a.scale_mode == 1) mul *= load_uniform_f32(a.k_scale);
  // the maximum is of raw scores and wants mul > 0: its sign goes into q (0: q is 0)
  uint32_t sign = 0u, keep = 0xffffffffu;
  if (!(mul > 0.0f) && mul == mul) {
    sign = mul < 0.0f ? (F::kF32 ? 0x80000000u : 0x80008000u) : 0u;
    keep = mul < 0.0f ? keep : 0u;
    mul = mul < 0.0f ? -mul : 1.0f;
  }
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
      const int d = F::kF32 ? 8 * s + 4 * hf : F::kEb == 2 ? 16 * s + 8 * hf : 16 * (2 * (s >> 1) + hf) + 8 * (s & 1);
      q[b][s] = ok ? ld16(p + d * F::kQb) : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < 4; ++e) q[b][s][e] = (q[b][s][e] ^ sign) & keep;
    }
  }
  // ---- loads of tiles: a wave 32 keys, sub-tiles of 16 never across a block ----
  const int64_t row_bytes = (int64_t)a.num_kv_heads * RB;
  uint32_t voff[kDma];
#pragma unroll
  for (int i = 0; i < kDma; ++i) {
    const int r = i * K::kPerDma + lane / K::kChunks;
    voff[i] = (uint32_t)(r * row_bytes) + 16 * ((lane % K::kChunks) ^ K::swz(r));
  }
  float scale_next = 1.0f;
  auto issue = [&](int kb, int to) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      const int at = wave * kOwn + 16 * u, t = kb + at;
      const int64_t phys = t < k1 ? a.idx.physical_block(seq, t >> a.idx.bs_log2) : -1;
      const int64_t slot = (max(phys, (int64_t)0) << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1));
      const int left = phys >= 0 ? min(k1 - t, 16) : 0;
      // (rows past the last read zeros)
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(a.k + (phys >= 0 ? slot : 0) * row_bytes + (int64_t)h * RB), (short)0,
          left > 0 ? (int)((left - 1) * row_bytes + RB) : 0, 0x00020000);
#pragma unroll
      for (int i = 0; i < kDma; ++i) dma16(r, &tile[to][at * RB + i * 1024], voff[i]);
      if (lane == 0) there[to][at / 16] = left > 0;
    }
    if (a.scale_mode == 2 && tid < kStreamKeys) {
      const int t = kb + tid, slot = t < k1 ? slot_of(a, seq, t) : -1;
      scale_next = slot >= 0 ? a.k_scale[(int64_t)slot * a.num_kv_heads + h] : 0.0f;
    }
  };
  float m[NQ], l[NQ];
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    m[b] = kNegBig;
    l[b] = 0.0f;
  }
  if (kb0 < k1) issue(kb0, 0);
  for (int kb = kb0, par = 0; kb < k1; kb += kStreamKeys, par ^= 1) {
    if (a.scale_mode == 2 && tid < kStreamKeys) scales[par][tid] = scale_next;
    wait_all();
    __syncthreads();  // the tile is here, and everyone is done with the other one
    if (kb + kStreamKeys < k1) issue(kb + kStreamKeys, par ^ 1);
    for (int kbl = kg; kbl < kStreamKeys / 32; kbl += KG) {
      const int key0 = kb + 32 * kbl;
      if (key0 >= min(high, k1)) break;
      u32x4 k[F::kOps];
      const char* const at = tile[par] + 32 * kbl * RB;
      if constexpr (F::kEb >= 2) {
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
      const bool lo_there = uniform(there[par][2 * kbl]) != 0, up_there = uniform(there[par][2 * kbl + 1]) != 0;
      const bool masked = key0 + 32 > min(low, k1) || !lo_there || !up_there;
#pragma unroll
      for (int b = 0; b < NQ; ++b) {
        f32x16 s = product<F::kF32, CT>(k, q[b]);
        if (a.scale_mode == 2) {
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(&scales[par][32 * kbl + 8 * g + 4 * hf]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * g + e] *= x[e];
          }
        }
        if (masked) {
          const int lm = min(lim[b], k1) - key0 - 4 * hf;
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int kl = 8 * (e >> 2) + (e & 3);
            s[e] = kl < lm && (e < 8 ? lo_there : up_there) ? s[e] : kNegInf;
          }
        }
        float mx = s[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s[e]);
        mx = fmaxf(mx, other_half(mx));
        mx = fmaxf(mx * mul, kNegBig);
        const float m_new = mx > m[b] + kRescaleSlack ? mx : m[b];
        if (__builtin_amdgcn_ballot_w64(m_new != m[b])) {
          l[b] *= __builtin_amdgcn_exp2f(m[b] - m_new);
          m[b] = m_new;
        }
        float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          sum0 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], mul, -m[b]));
          sum1 += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e + 1], mul, -m[b]));
        }
        l[b] += sum0 + sum1;
      }
    }
  }
#pragma unroll
  for (int b = 0; b < NQ; ++b) l[b] += other_half(l[b]);
  if constexpr (KG > 1) {
    if (hf == 0) {
#pragma unroll
      for (int b = 0; b < NQ; ++b) joined[wave][32 * b + c] = f32x2{m[b], l[b]};
    }
    __syncthreads();
    if (kg > 0) return;
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
  if (hf) return;
#pragma unroll
  for (int b = 0; b < NQ; ++b) {
    const int r = row0 + 32 * b + c;
    if (r >= rows) continue;
    const int tok = div_group(a, r);
    const int64_t at = (sq.q0 + tok) * a.num_heads + h * a.group + r - tok * a.group;
    if (a.splits > 1)
      a.part_ml[blockIdx.y * a.total_q * a.num_heads + at] = f32x2{m[b], l[b]};
    else
      a.lse[at] = l[b] == 0.0f ? -kNegInf : m[b] + __builtin_amdgcn_logf(l[b]);
  }
}

__global__ __launch_bounds__(kThreads) void weights_join_kernel(WeightArgs a) {
  const int64_t n = a.total_q * a.num_heads, i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  float m = kNegBig, l = 0.0f;
  for (int z = 0; z < a.splits; ++z) m = fmaxf(m, a.part_ml[z * n + i][0]);
  for (int z = 0; z < a.splits; ++z) {
    const f32x2 v = a.part_ml[z * n + i];
    l += v[1] * __builtin_amdgcn_exp2f(v[0] - m);
  }
  a.lse[i] = l == 0.0f ? -kNegInf : m + __builtin_amdgcn_logf(l);
}

// The keys' weights.
template <int KV, int CT, int D>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2))) void weights_columns_kernel(WeightArgs a) {
  using F = Formats<KV, CT, D>;
  constexpr int RB = D * F::kQb;
  using Q = Rows<RB>;
  constexpr int NK = F::kBlocks, kUnit = 32 * NK * kWaves, kTile = 16384 / RB;  // rows of q a tile: 32, 64 or 128
  constexpr int kDma = kTile / kWaves / Q::kPerDma;
  __shared__ __align__(16) char tile[2][kTile * RB];
  __shared__ __align__(16) float lse[2][kTile];
  __shared__ __align__(16) int last[2][kTile];  // the position of a row: the last that it sees
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6), c = lane & 31, hf = lane >> 5;
  float mul0 = a.mul;
  if (a.scale_mode == 1) mul0 *= load_uniform_f32(a.k_scale);
  for (int64_t at = blockIdx.x;; at += gridDim.x) {
    const int h = (int)(at % a.num_kv_heads);
    int seq, place;
    if (at / a.num_kv_heads > 0x7fffffff ||
        !find_part(a.num_seqs, (int)(at / a.num_kv_heads), seq, place, [&](int s) {
          const Seq q = seq_of(a, s);
          return (q.keys + kUnit - 1) / kUnit;
        }))
      return;
    seq = uniform(seq);
    const Seq sq = seq_of(a, seq);
    const int rows = (int)sq.n * a.group;
    const int unit0 = place * kUnit, key0 = unit0 + wave * 32 * NK;  // this wave's first key
    // ---- this lane's keys ----
    u32x4 k[NK][F::kOps];
    float mul[NK], sum[NK];
    int slot[NK];
#pragma unroll
    for (int b = 0; b < NK; ++b) {
      const int t = key0 + 32 * b + c;
      slot[b] = t < sq.keys ? slot_of(a, seq, t) : -1;
      const char* p = a.k + ((int64_t)max(slot[b], 0) * a.num_kv_heads + h) * (int64_t)(D * F::kEb);
#pragma unroll
      for (int s = 0; s < F::kOps; ++s) {
        if constexpr (F::kEb >= 2) {
          k[b][s] = ld16(p + 16 * (2 * s + hf));
        } else {
          const u32x2 w = ld8(p + 8 * (2 * s + hf));
          k[b][s] = codes_to_16<KV, CT>(w[0], w[1]);
        }
      }
      mul[b] = mul0;
      if (a.scale_mode == 2) mul[b] *= a.k_scale[(int64_t)max(slot[b], 0) * a.num_kv_heads + h];
      sum[b] = 0.0f;
    }
    // ---- rows that see any of the unit's keys ----
    const int64_t skip = max((int64_t)unit0 - sq.first, (int64_t)0) * a.group;
    const int r_begin = (int)min(skip, (int64_t)rows) / kTile * kTile;
    float lse_next = 0.0f;
    int last_next = 0;
    auto issue = [&](int r0, int to) {
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
        dma16(r, &tile[to][(wave * (kTile / kWaves) + i * Q::kPerDma) * RB], row < rows ? off : 0x7ffffff0u);
      }
      if (tid < kTile) {
        const int row = r0 + tid, tok = div_group(a, row);
        lse_next = row < rows ? a.lse[(sq.q0 + tok) * a.num_heads + h * a.group + row - tok * a.group] : -kNegInf;
        last_next = row < rows ? (int)min(max(sq.first + tok, (int64_t)-1), (int64_t)0x7fffffff) : -1;
      }
    };
    __syncthreads();  // (everyone is done with the unit before)
    if (r_begin < rows) issue(r_begin, 0);
    for (int r0 = r_begin, par = 0; r0 < rows; r0 += kTile, par ^= 1) {
      wait_all();
      if (tid < kTile) {
        lse[par][tid] = lse_next;
        last[par][tid] = last_next;
      }
      __syncthreads();
      if (r0 + kTile < rows) issue(r0 + kTile, par ^ 1);
      for (int rb = 0; rb < kTile / 32; ++rb) {
        if (r0 + 32 * rb >= rows) break;
        // (rows' positions rise: the block's first and last)
        const int least = uniform(last[par][32 * rb]);
        const int most = uniform(last[par][min(32 * rb + 31, rows - 1 - r0)]);
        if (most < key0) continue;
        u32x4 q[F::kOps];
#pragma unroll
        for (int s = 0; s < F::kOps; ++s)
          q[s] = *reinterpret_cast<const u32x4*>(tile[par] + 32 * rb * RB + Q::offset(c, 2 * s + hf));
        f32x4 norm[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) norm[g] = *reinterpret_cast<const f32x4*>(&lse[par][32 * rb + 8 * g + 4 * hf]);
#pragma unroll
        for (int b = 0; b < NK; ++b) {
          const f32x16 s = product<F::kF32, CT>(q, k[b]);
          float p[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], mul[b], -norm[e >> 2][e & 3]));
          // rows that end ahead of the block's last key, and those past the last row,
          // whose normaliser makes their weight 0 unless the key is not finite
          if (least < key0 + 32 * b + 31 || r0 + 32 * rb + 32 > rows) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              typedef int i32x4 __attribute__((ext_vector_type(4)));
              const i32x4 end = *reinterpret_cast<const i32x4*>(&last[par][32 * rb + 8 * g + 4 * hf]);
#pragma unroll
              for (int e = 0; e < 4; ++e) p[4 * g + e] = end[e] >= key0 + 32 * b + c ? p[4 * g + e] : 0.0f;
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
      }
    }
#pragma unroll
    for (int b = 0; b < NK; ++b) {
      const float w = sum[b] + other_half(sum[b]);
      if (hf == 0 && slot[b] >= 0) add_weight(a, sq, slot[b], h, key0 + 32 * b + c, w);
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
  // chunks
  int row_groups, splits;
  int64_t row_units;
  int column_grid;
  size_t bytes;
};

constexpr size_t kMaxScores = (size_t)1 << 30;  // bytes of kept scores

Plan make_plan(int num_seqs, int64_t total_q, int heads, int kv_heads, int64_t capacity, bool one_row, bool f32) {
  Plan p{};
  const int group = heads / kv_heads;
  const int64_t pairs = (int64_t)num_seqs * kv_heads;
  if (one_row) {
    p.ni = group <= 4 ? 1 : 4;
    const int most = 4096 / p.ni;  // 64 KB of scores: two workgroups a CU
    p.unit = capacity <= most ? (int)((capacity + 15) / 16 * 16) : 1024;
    p.max_units = (int)((capacity + p.unit - 1) / p.unit);
    const int64_t room = 16384 / pairs;
    p.grid_units = (int)(p.max_units < room ? p.max_units : room < 1 ? 1 : room);
    if (p.max_units > 1)
      p.bytes = (size_t)pairs * p.max_units * 4 * p.ni * (8 + (size_t)p.unit * 4);
    if (p.bytes <= kMaxScores) {
      p.decode = true;
      return p;
    }
  }
  const int held = f32 ? 32 : 64;  // rows of a wave
  const int64_t rows = total_q * group, mean = rows / num_seqs;
  p.row_groups = mean <= held ? 1 : mean <= 2 * held ? 2 : 4;
  p.row_units = num_seqs + rows / (held * p.row_groups);
  const int64_t blocks = p.row_units * kv_heads, tiles = (capacity + kStreamKeys - 1) / kStreamKeys;
  int64_t splits = 1024 / blocks;
  splits = splits > tiles ? tiles : splits;
  p.splits = (int)(splits < 1 ? 1 : splits);
  const int unit = f32 ? 128 : 256;
  const int64_t units = (int64_t)num_seqs * ((capacity + unit - 1) / unit) * kv_heads;
  p.column_grid = (int)(units < 8192 ? units : 8192);
  p.bytes = (size_t)total_q * heads * (4 + (p.splits > 1 ? 8 * (size_t)p.splits : 0));
  p.bytes = (p.bytes + 15) / 16 * 16;
  return p;
}

template <int KV, int CT, int D>
int launch_weights(WeightArgs& a, const Plan& p, hipStream_t s) {
  if (p.decode) {
    const dim3 grid((unsigned)((int64_t)a.num_seqs * a.num_kv_heads * p.grid_units));
    const size_t lds = (size_t)p.unit / 16 * p.ni * 64 * 4;
    if (p.ni == 1)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_decode_kernel<KV, CT, D, 1>), grid, dim3(kThreads), lds, s, a);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_decode_kernel<KV, CT, D, 4>), grid, dim3(kThreads), lds, s, a);
    if (hipError_t e = hipGetLastError()) return (int)e;
    if (p.max_units > 1) {
      if (p.ni == 1)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_finish_kernel<1>), grid, dim3(kThreads), 0, s, a);
      else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_finish_kernel<4>), grid, dim3(kThreads), 0, s, a);
    }
    return (int)hipGetLastError();
  }
  const dim3 grid((unsigned)(p.row_units * a.num_kv_heads), (unsigned)p.splits);
  switch (p.row_groups) {
    case 1: hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_lse_kernel<KV, CT, D, 1>), grid, dim3(kThreads), 0, s, a); break;
    case 2: hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_lse_kernel<KV, CT, D, 2>), grid, dim3(kThreads), 0, s, a); break;
    default: hipLaunchKernelGGL(HIP_KERNEL_NAME(weights_lse_kernel<KV, CT, D, 4>), grid, dim3(kThreads), 0, s, a); break;
  }
  if (hipError_t e = hipGetLastError()) return (int)e;
  if (p.splits > 1) {
    hipLaunchKernelGGL(weights_join_kernel, dim3((unsigned)((a.total_q * a.num_heads + kThreads - 1) / kThreads)),
                       dim3(kThreads), 0, s, a);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
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
  if (p.decode ? (int64_t)num_seqs * num_kv_heads * p.grid_units > kMaxGrid : p.row_units * num_kv_heads > kMaxGrid)
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
  a.ws_ml = reinterpret_cast<f32x2*>(workspace);
  a.ws_t = reinterpret_cast<float*>(a.ws_ml + (p.decode ? (size_t)num_seqs * num_kv_heads * p.max_units * 4 * p.ni : 0));
  a.splits = p.splits;
  a.part_ml = reinterpret_cast<f32x2*>(workspace);
  a.lse = reinterpret_cast<float*>(a.part_ml + (!p.decode && p.splits > 1 ? (size_t)p.splits * total_q * num_heads : 0));
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
