// Attention of trees of drafted tokens over the paged KV cache: the
// verification step of speculative decoding.
//
// Sequence s has n_s drafted tokens in rows cu[s] .. cu[s+1] of q, whose K and V
// are in the cache already, at positions P_s .. P_s + n_s - 1 behind its prefix of
// P_s = context_lens[s] - n_s tokens.  Row i sees the whole prefix and drafted
// token j where mask[cu[s] + i][j] is true (its ancestors and itself):
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = exp(scale q_i . k_j - m_i)
//
// over what it sees; a row that sees nothing gives zeros.
//
// A KV head's rows are its (drafted token, query head of the group) pairs,
// token-major, M = n_s G of them: 4 M flops for every byte pair of a 16-bit cache,
// so small trees are bound by the cache's bytes and trees of M >= 256 by the
// matrix units.  Every wave holds 32 rows and takes keys 32 at a time:
//
//   S^T = K Q^T        (32x32x16 MFMA; A = K from LDS, B = Q^T in registers)
//   O^T += V^T P^T     (A = V^T by transposing LDS reads, B = P^T as it stands in
//                      the S^T accumulators: the order of the contraction over
//                      keys is free, so each lane's own keys are its k-slots)
//
// with a row's softmax state in the lanes of its column.  A workgroup's waves
// are R groups of 32 rows that share each staged K/V tile times KG groups that
// take different keys of the same rows (one row group: four key groups), joined in
// LDS at the end.  Long contexts are split over workgroups by the total length
// of the batch; partial results of a row are joined by a second kernel.
#include <type_traits>

#include "mkv_device.hpp"

namespace mkv {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kHeadDim = 128;
constexpr float kNegBig = -1e30f;
constexpr float kNegInf = -__builtin_huge_valf();
// the running maximum moves only when a tile exceeds it by more than 2^8, so that
// most tiles rescale nothing; any offset of the maximum cancels in the normalisation
constexpr float kRescaleSlack = 8.0f;
// fp16 P: the maximum is offered less 7, so that a row's largest P is 2^7 to 2^15.  P
// 2^21 below the largest is exact to fp16's half step, the rest to 2^-32 of the
// largest (with the largest at 1, a context of 130,000 keys of 2^-26 beside one key
// lost all of them, 2^-8 of the weight in all).
constexpr float kHalfLift = 7.0f;

// Per-token-head V scales are folded into P ahead of its rounding to fp16, so it
// is P times the scale that has to fit: the running maximum is that of score +
// log2 |V scale| (less kHalfLift).  Scales below 2^kLeastScale count as that here
// (a key may have none, and the normaliser's terms, P alone, stay below 2^79), ones
// above 2^kMostScale as that (P stays within fp32's normal range).
constexpr float kLeastScale = -64.0f, kMostScale = 100.0f;
MKV_DEV float scale_log2(float s) {  // (0, infinite and NaN scales: within the bounds)
  return fminf(fmaxf(__builtin_amdgcn_logf(fabsf(s)), kLeastScale), kMostScale);
}
// x 2^d, by halves: scales far apart bring factors below fp32's range to terms
// above 1
MKV_DEV float mul_exp2(float x, float d) {
  const float f = __builtin_amdgcn_exp2f(0.5f * d);
  return x * f * f;
}

struct TreeArgs {
  void* out;
  const void* q;
  const char* k;
  const char* v;
  const float* k_scale;
  const float* v_scale;
  PagedIndex idx;
  const void* ctx;
  int ctx_i64;
  const int32_t* cu;
  const uint8_t* mask;
  int64_t mask_stride;
  int mask_cols;
  int num_seqs;
  int64_t total_q;
  int num_heads;     // query heads
  int num_kv_heads;  // the kernel's (half the caller's with head pairing)
  int scale_heads;   // the caller's KV heads: the stride of a slot's scales
  int group;         // the kernel's query heads to a KV head
  int q_dtype;
  float sm_scale;
  int splits;        // whether sequences may be split (else no partial results)
  int shares;        // the batch's keys over this many make a split
  int min_split;     // keys
  float* ws_o;       // partials: (unit, kv head, row cap, 128)
  float* ws_ml;      // (unit, kv head, row cap, 2)
  int row_cap;
  int row_blocks;
};

// Element i of an int32 or int64 array, without a branch (so that loads of several
// go out together).
MKV_DEV int64_t load_len(const void* p, int i, int i64) {
  const int32_t* x = reinterpret_cast<const int32_t*>(p);
  const int32_t lo = x[(int64_t)i << i64], hi = x[((int64_t)i << i64) + i64];
  return i64 ? (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo) : (int64_t)lo;
}

// Sums over the wave's lanes up to each (the last lane's is the whole), by DPP.
template <typename X>
MKV_DEV X wave_scan(X x) {
  static_assert(sizeof(X) == 4, "");
  auto add = [&](auto ctrl, auto rows) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    x += __builtin_bit_cast(X, y);
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
MKV_DEV float wave_sum(float x) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wave_scan(x)), 63));
}

// A workgroup's place: row block, unit, KV head and sequence with the split's
// number and length, and the sequence's rows and context length as given.
struct Place {
  int rb, unit, kvh, seq, z, len;
  int cu0, cu1;
  int64_t ctx;
};

// A unit is one split of one sequence; units go sequence by sequence.  Splits are
// of `len` keys, the same for every sequence: the batch's keys over the plan's
// shares, in whole tiles.  Every workgroup works this out for itself from the
// context lengths (a lane a sequence), so that the units are numbered without
// gaps: workgroups without work among the others would unbalance the CUs, which
// the hardware fills in a fixed order.
template <int TILE>
struct Units {
  const TreeArgs& a;
  int len, total;
  int before, n;  // this lane's sequence (of the 64 last looked at): its units, and those ahead of them

  int cu0, cu1;       // ... its rows in q, and the length of its context
  int64_t ctx;

  MKV_DEV int keys(int s0) {
    const int s = s0 + (threadIdx.x & 63), i = min(s, a.num_seqs - 1);
    ctx = load_len(a.ctx, i, a.ctx_i64);
    cu0 = a.cu[i];
    cu1 = a.cu[i + 1];
    return s < a.num_seqs ? (int)min(max(ctx, (int64_t)0), (int64_t)a.idx.max_blocks << a.idx.bs_log2) : 0;
  }
  // the units of sequences s0 .. s0 + 63, `base` ahead of them; their number
  MKV_DEV int number(int s0, int k, int base) {
    n = s0 + (int)(threadIdx.x & 63) < a.num_seqs ? max((int)(((uint32_t)k + (uint32_t)len - 1) / (uint32_t)len), 1) : 0;
    const int upto = wave_scan(n);
    before = base + upto - n;
    return __builtin_amdgcn_readlane(upto, 63);
  }
  MKV_DEV explicit Units(const TreeArgs& args) : a(args) {
    const int k0 = keys(0);
    double sum = wave_sum((float)k0);  // (a rule of thumb's accuracy, the same in every wave)
    for (int s0 = 64; s0 < a.num_seqs; s0 += 64) sum += wave_sum((float)keys(s0));
    // (a little more than the even share: at most `shares` units beside the last
    // one of each sequence, whatever the sum's rounding)
    // (at most a block table's largest capacity, 0x7fff0000 keys: one unit then)
    len = (int)fminf((float)sum * 1.0001f / (float)a.shares, 2147418112.0f) + 1;
    len = uniform((max(len, a.min_split) + TILE - 1) / TILE * TILE);
    total = number(0, a.num_seqs > 64 ? keys(0) : k0, 0);
    for (int s0 = 64; s0 < a.num_seqs; s0 += 64) total += number(s0, keys(s0), total);
  }
  // a unit's sequence, its number within it, and what find_work() reads of it
  MKV_DEV bool of_unit(int unit, Place& p) {
    int base = 0;
    for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
      if (a.num_seqs > 64) base += number(s0, keys(s0), base);
      const uint64_t mine = __builtin_amdgcn_ballot_w64(unit >= before && unit < before + n);
      if (mine) {
        const int l = __builtin_ctzll(mine);
        p.seq = s0 + l;
        p.z = unit - __builtin_amdgcn_readlane(before, l);
        take(l, p);
        return true;
      }
    }
    return false;
  }
  // a sequence's first unit, their number, and what find_work() reads of it
  MKV_DEV int of_sequence(int seq, Place& p) {
    if (a.num_seqs > 64) {
      int base = 0;
      for (int s0 = 0; s0 <= seq; s0 += 64) base += number(s0, keys(s0), base);
    }
    p.seq = seq;
    p.unit = __builtin_amdgcn_readlane(before, seq & 63);
    take(seq & 63, p);
    return __builtin_amdgcn_readlane(n, seq & 63);
  }
  MKV_DEV void take(int l, Place& p) const {
    p.cu0 = __builtin_amdgcn_readlane(cu0, l);
    p.cu1 = __builtin_amdgcn_readlane(cu1, l);
    p.ctx = (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(ctx >> 32), l) << 32 |
                      (uint32_t)__builtin_amdgcn_readlane((int)ctx, l));
  }
};

template <int CT>
using Op16 = typename std::conditional<CT == MKV_DTYPE_BF16, bf16x8, f16x8>::type;

template <int CT>
MKV_DEV f32x16 mfma32(Op16<CT> A, Op16<CT> B, f32x16 C) {
  if constexpr (CT == MKV_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(A, B, C, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(A, B, C, 0, 0, 0);
}

MKV_DEV float other_half(float x) {  // the value of lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// The largest of three, NaN where one is (v_maximum3_f32).
MKV_DEV float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}

// LDS tiles: a key's 128 cached elements as they are in the pool (256- or 128-byte
// rows), its 16-byte chunk i at position i ^ swz(key).
// 16-bit: swz is one-to-one on 16 keys (K operand reads: 16 keys, one chunk) and
// moves four neighbouring keys to the four 64-byte quarters of a row (transposed
// V reads: four keys, 32 dims).
// 1-byte: two rows fill the 64 banks; swz is one-to-one on the 8 even (odd) keys
// of 16, and the keys 4h .. 4h+3 and 8+4h .. 8+4h+3 of a transposed V read keep
// their pairs of chunks apart.
// Both read without bank conflicts.
template <int EB>
struct Tile {
  static constexpr int kRow = kHeadDim * EB;
  static constexpr int kChunks = kRow / 16;
  static constexpr int kKeysPerDma = 1024 / kRow;  // a wave's 64 x 16 bytes
  MKV_DEV static int swz(int key) {
    if constexpr (EB == 2) return ((key & 3) << 2) | ((key >> 2) & 3);
    return (key >> 1 & 4) | (key & 2) | (key >> 2 & 1);
  }
  MKV_DEV static int offset(int key, int chunk) { return key * kRow + ((chunk ^ swz(key)) << 4); }
};

template <int N>
MKV_DEV void wait_vm() {  // all but the wave's last N vector memory operations are done
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt((N & 15) | 0xf70 | (N >> 4 << 14));
  asm volatile("" ::: "memory");
}
// The wave's LDS reads and writes are done.
MKV_DEV void wait_lds() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// The workgroup's waves meet, their LDS reads done; LDS DMA stays in flight.
MKV_DEV void meet() {
  wait_lds();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Values that are not finite.  A drafted token that a row does not see weighs
// P = 0 there, and 0 * inf or 0 * NaN would still reach the row's output: where a
// tile of drafted tokens holds such values, the products take zeros in their
// place, and a product of marks with what each row sees says which outputs they
// belong to.  Marks of up to 64 keys add up without mixing.
constexpr float kMarkPos = 1.0f, kMarkNeg = 256.0f, kMarkNan = 32768.0f;
MKV_DEV float mark_of(float x) {
  float m = x == __builtin_huge_valf() ? kMarkPos : 0.0f;
  m = x == -__builtin_huge_valf() ? kMarkNeg : m;
  return x != x ? kMarkNan : m;
}
MKV_DEV float marked_value(float n) {  // 0 without marks
  const float nans = floorf(n * (1.0f / kMarkNan));
  n -= kMarkNan * nans;
  const float negs = floorf(n * (1.0f / kMarkNeg));
  n -= kMarkNeg * negs;
  float v = n > 0.0f ? __builtin_huge_valf() : 0.0f;
  v = negs > 0.0f ? v - __builtin_huge_valf() : v;  // (inf - inf: NaN)
  return nans > 0.0f ? __builtin_nanf("") : v;
}
MKV_DEV bool not_finite(float x) { return !(fabsf(x) < __builtin_huge_valf()); }
// two 16-bit elements: exponent bits all ones
template <int CT>
MKV_DEV bool not_finite2(uint32_t w) {
  constexpr uint32_t e = CT == MKV_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
  return (w & e) == e || ((w >> 16) & e) == e;
}

template <int KV_DT>
constexpr int kOperand = KV_DT == MKV_DTYPE_BF16 ? MKV_DTYPE_BF16 : MKV_DTYPE_F16;

// Workgroup coordinates and the rows and keys that follow from them.
struct Work {
  int seq, kvh;
  int64_t q0;       // first row of the sequence in q
  int rows;         // rows of the KV head: drafted tokens x group
  int64_t prefix;
  int ctx;          // keys, within the block table
};

MKV_DEV Work find_work(const TreeArgs& a, const Place& p) {
  Work w;
  w.kvh = p.kvh;
  w.seq = p.seq;
  const int64_t q0 = min(max((int64_t)p.cu0, (int64_t)0), a.total_q);
  const int64_t q1 = min(max((int64_t)p.cu1, q0), a.total_q);
  const int64_t c = max(p.ctx, (int64_t)0);
  w.q0 = q0;
  w.rows = (int)min(q1 - q0, (int64_t)a.mask_cols) * a.group;
  w.prefix = max(c - (q1 - q0), (int64_t)0);
  w.ctx = (int)min(c, (int64_t)a.idx.max_blocks << a.idx.bs_log2);
  return w;
}

// (false: a workgroup without work)
template <int TILE>
MKV_DEV bool find_place(const TreeArgs& a, Place& p) {
  auto split = [&](int units) {
    const int pairs = units * a.num_kv_heads;
    p.rb = (int)blockIdx.x / pairs;
    const int q = (int)blockIdx.x - p.rb * pairs;
    p.unit = q / a.num_kv_heads;
    p.kvh = q - p.unit * a.num_kv_heads;
    return p.rb < a.row_blocks;
  };
  if (!a.splits) {
    p.len = 0x7fffffff / TILE * TILE;
    p.z = 0;
    const bool ok = split(a.num_seqs);
    p.seq = min(p.unit, a.num_seqs - 1);
    p.cu0 = a.cu[p.seq];
    p.cu1 = a.cu[p.seq + 1];
    p.ctx = load_len(a.ctx, p.seq, a.ctx_i64);
    return ok;
  }
  Units<TILE> u(a);
  p.len = u.len;
  if (!split(u.total)) return false;
  return u.of_unit(p.unit, p);
}

// Element offset of row r (token r / group, head r % group) of the KV head in q
// and out, and with head pairing which half of the 128-wide row it uses.
template <bool PAIR>
MKV_DEV int64_t row_offset(const TreeArgs& a, const Work& w, int r, bool& hi) {
  const int tok = r / a.group, j = r - tok * a.group;
  hi = PAIR && j >= (a.group >> 1);
  return ((w.q0 + tok) * a.num_heads + w.kvh * a.group + j) * kQDim<PAIR>;
}

MKV_DEV void store4(void* out, int dt, int64_t off, const float* x) {
  if (dt == MKV_DTYPE_F32) {
    st16(reinterpret_cast<float*>(out) + off,
         u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])});
  } else {
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = dt == MKV_DTYPE_BF16 ? f32_to_bf16_bits(x[j]) : f32_to_f16_bits(x[j]);
    *reinterpret_cast<u32x2*>(reinterpret_cast<uint16_t*>(out) + off) = u32x2{h[0] | h[1] << 16, h[2] | h[3] << 16};
  }
}

// Rows of a sequence past the mask's width, which name no visible token: zeros.
MKV_DEV void zero_rows_past(const TreeArgs& a, const Work& w) {
  const int64_t q1 = min(max((int64_t)a.cu[w.seq + 1], w.q0), a.total_q);
  const int64_t first = w.q0 + a.mask_cols;
  if (first >= q1) return;
  const int size = a.q_dtype == MKV_DTYPE_F32 ? 4 : 2;
  const int64_t dims = (int64_t)a.num_heads * (kHeadDim * a.num_kv_heads / a.scale_heads);
  uint16_t* o = reinterpret_cast<uint16_t*>(a.out) + first * dims * size / 2;
  for (int64_t i = threadIdx.x; i < (q1 - first) * dims * size / 2; i += blockDim.x) o[i] = 0;
}

// 16 one-byte codes of the pool as exact fp16.
template <int KV_DT>
MKV_DEV f16x8 codes_to_f16(uint32_t lo, uint32_t hi) {
  uint32_t w[4];
  if constexpr (KV_DT == kKvI8PerToken) {
    // 0x64xx is 1024 + xx in fp16: code + 128 in xx, then 1152 off
    const uint32_t c[2] = {lo ^ 0x80808080u, hi ^ 0x80808080u};
    const f16x2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t x = perm(0x64646464u, c[i >> 1], i & 1 ? 0x04030402u : 0x04010400u);
      w[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, x) - off);
    }
  } else {
    w[0] = __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<false>(lo));
    w[1] = __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<true>(lo));
    w[2] = __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<false>(hi));
    w[3] = __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<true>(hi));
  }
  return __builtin_bit_cast(f16x8, u32x4{w[0], w[1], w[2], w[3]});
}

// Keys a wave takes of a tile: two blocks of 32, whose products and softmax run
// side by side; one with four key groups (16-bit tiles of 256 keys would not fit
// twice in a CU's LDS, and short contexts end in the middle of so long a tile).
template <int KV_DT, int R, int KG>
constexpr int kTileKeys = KG == 4 ? 32 : 64;

// The tile's pipeline.  K and V have one LDS buffer each.  A wave reads all of a
// tile's K operands into registers, and the DMA of the next tile's K goes out
// where they were, to land under the softmax and P V; likewise V's once its last
// operands are read.  The second key block's K Q^T is issued among the first's
// exponentials and the first's P V among the second's, so that MFMA and VALU work
// of one wave overlap (two waves a SIMD alone reached little more than the sum of
// the two: 2900 cycles for a tile's 1536 of MFMA and 1200 of VALU).  With one row
// group a wave reads only what it loaded itself and meets no barrier.  One buffer
// (64 KB at most) and at most 256 registers leave room for two workgroups a CU.
template <int KV_DT, int R, int KG, bool PAIR>
MKV_DEV void tree_attention_body(const TreeArgs& a) {
  constexpr int CT = kOperand<KV_DT>;
  constexpr bool kTok = kPerTokenScale<KV_DT>;
  constexpr float kLift = CT == MKV_DTYPE_F16 ? kHalfLift : 0.0f;
  constexpr int kWaves = R * KG, kThreads = 64 * kWaves;
  constexpr int TK = kTileKeys<KV_DT, R, KG>;  // keys a wave takes of a tile
  constexpr int NK = TK * KG;             // keys of a tile
  constexpr int NB = TK / 32;
  constexpr int kEb = DTypeInfo<KV_DT>::kBytes;
  using T = Tile<kEb>;
  constexpr int kOwn = NK / kWaves;                     // keys a wave loads
  constexpr int kDma = kOwn / T::kKeysPerDma;           // loads of K, and of V, a wave
  constexpr int kSubs = kOwn > 16 ? kOwn / 16 : 1;      // 16-key sub-tiles (never across a block) they lie in
  constexpr bool kShared = R > 1;
  static_assert(kOwn % T::kKeysPerDma == 0 && kDma >= 1, "whole loads");
  constexpr int kSums = R * 4 * (KG - 1) * 4096;  // (what the key groups hand each other, over both)
  constexpr int kBuf = NK * T::kRow > kSums / 2 ? NK * T::kRow : kSums / 2;
  __shared__ __align__(16) char lds_k[kBuf], lds_v[kBuf];
  __shared__ f32x2 join_ml[KG > 1 ? kWaves * 32 : 1];
  __shared__ int slots[kShared ? 2 * (NK / 16) : 1];  // of each sub-tile, -1 absent, by the tile's parity
  constexpr int kHeads = PAIR ? 2 : 1;
  constexpr int kScLoads = kTok ? 2 * kHeads * TK / 64 : 1;
  __shared__ __align__(16) float sc_all[kTok ? kWaves * 3 * kHeads * TK : 4];  // a wave's own: [head][K, V, log2 |V|][TK]

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int rg = wave % R, kg = wave / R;
  const int c = lane & 31, h = lane >> 5;
  Place place;
  if (!find_place<NK>(a, place)) return;
  const int len = place.len;
  const Work w = find_work(a, place);
  const bool zeroes = place.rb == 0 && place.z == 0 && w.kvh == 0;
  if (place.rb * 32 * R >= w.rows) {
    if (zeroes) zero_rows_past(a, w);
    return;
  }
  const int kb0 = place.z * len, k1 = (int)min((int64_t)kb0 + len, (int64_t)w.ctx);
  const int prefix = (int)min(w.prefix, (int64_t)0x7fffffff);
  const bool split = w.ctx > len;

  // ---- loads of tiles ----
  const int64_t row_bytes = (int64_t)a.num_kv_heads * T::kRow;
  const int64_t head_bytes = (int64_t)w.kvh * T::kRow;
  const int own0 = wave * kOwn;  // first key of the tile that this wave loads
  const int sub0 = own0 & ~15;
  // lane's key and chunk of a load; loads of one sub-tile differ in the key's
  // upper bits, which reach the swizzle's low bits
  const int ld_key = lane / T::kChunks;
  constexpr int kPerSub = kDma / kSubs;
  uint32_t voff[kPerSub];
#pragma unroll
  for (int i = 0; i < kPerSub; ++i) {
    const int key = (own0 & 15) + i * T::kKeysPerDma + ld_key;
    voff[i] = (uint32_t)(key * row_bytes) + 16 * ((lane % T::kChunks) ^ T::swz(key));
  }
  // The tile whose K is loaded next: its sub-tiles' first token slots, and the
  // rows of each that lie within the context in a present block.  The block
  // entries come a tile ahead by a vector load (a scalar one would share its
  // counter with the LDS reads), a run of lanes a sub-tile.
  int32_t slot[kSubs], left[kSubs];
  const int32_t* bt_row = a.idx.block_tables + (int64_t)w.seq * a.idx.bt_stride;
  auto entry_load = [&](int kb) -> int32_t {
    const int blk = (kb + sub0 + 16 * (lane / (64 / kSubs))) >> a.idx.bs_log2;
    return bt_row[min(blk, a.idx.max_blocks - 1)];
  };
  auto entry_use = [&](int kb, int32_t e) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      const int t = kb + sub0 + 16 * u;
      const int phys = __builtin_amdgcn_readlane(e, 64 / kSubs * u);
      const bool ok = t < k1 && phys >= 0 && phys < (int)a.idx.num_blocks;
      slot[u] = ok ? (phys << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : 0;
      left[u] = ok ? min(k1 - t, 16) : 0;
    }
  };
  auto dma = [&](const char* pool, char* buf) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      // (rows past the last read zeros)
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(pool + slot[u] * row_bytes + head_bytes), (short)0,
          left[u] > 0 ? (int)((left[u] - 1) * row_bytes + T::kRow) : 0, 0x00020000);
#pragma unroll
      for (int i = 0; i < kPerSub; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(buf + (own0 + u * 16) * T::kRow + i * 1024), 16, voff[i], 0, 0, 0);
    }
  };
  float sc_raw[kScLoads];
  float* const sc = sc_all + (kTok ? wave * 3 * kHeads * TK : 0);
  auto load_scales = [&](int kb, int turn) {
    if constexpr (kTok) {
#pragma unroll
      for (int i = 0; i < kScLoads; ++i) {
        const int at = lane + 64 * i, key = at % TK, which = at / TK;  // K head 0, V head 0, K head 1, V head 1
        int sl;
        if constexpr (kShared)
          sl = slots[turn * (NK / 16) + (kg * TK + key) / 16];
        else
        {
          sl = -1;
#pragma unroll
          for (int u = 0; u < kSubs; ++u) sl = key >> 4 == u && left[u] > 0 ? slot[u] : sl;
        }
        sc_raw[i] = 0.0f;
        if (sl >= 0 && kb + kg * TK + key < k1)
          sc_raw[i] = ((which & 1) ? a.v_scale : a.k_scale)[(int64_t)(sl + (key & 15)) * a.scale_heads + w.kvh * kHeads + (which >> 1)];
      }
    }
  };
  // ---- q: this lane's row; step s of the contraction takes dims 16 s + 8 h .. + 7
  // (16-bit: chunk 2 s + h), or the lower or upper half of chunk 2 (s / 2) + h ----
  const int row = place.rb * 32 * R + rg * 32 + c;
  const bool row_ok = row < w.rows;
  bool hi = false;
  const int64_t q_off = row_offset<PAIR>(a, w, row_ok ? row : 0, hi);
  float score_mul = a.sm_scale * kLog2e;
  u32x4 raw[8];  // (its loads go out ahead of the tiles')
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    const int st = PAIR ? s & 3 : s;
    const int d = kEb == 2 ? 16 * st + 8 * h : 16 * (2 * (st >> 1) + h) + 8 * (st & 1);
    raw[s] = ld16(reinterpret_cast<const uint16_t*>(a.q) + q_off + d);  // (within q for any row)
  }
  const bool any = kb0 < k1;
  int32_t e_ahead = 0;
  if (any) {
    e_ahead = entry_load(kb0);
    const int32_t e_next = entry_load(kb0 + NK);
    entry_use(kb0, e_ahead);
    e_ahead = e_next;
    if constexpr (kShared) {
      if (lane == 0) {
#pragma unroll
        for (int u = 0; u < kSubs; ++u) slots[sub0 / 16 + u] = left[u] > 0 ? slot[u] : -1;
      }
      if constexpr (kTok) __syncthreads();
    }
    load_scales(kb0, 0);
    dma(a.k, lds_k);
    dma(a.v, lds_v);
  }

  Op16<CT> qop[8];
  {
    // the loop keeps raw scores and wants score_mul > 0: a negative scale (the
    // softmax's times a per-tensor K scale) moves its sign into q, a zero one makes
    // q zero
    if constexpr (KV_DT == MKV_DTYPE_FP8E4M3) score_mul *= load_uniform_f32(a.k_scale);
    uint32_t sign = 0u, keep = 0xffffffffu;
    if (!(score_mul > 0.0f) && score_mul == score_mul) {
      sign = score_mul < 0.0f ? 0x80008000u : 0u;
      keep = score_mul < 0.0f ? keep : 0u;
      score_mul = score_mul < 0.0f ? -score_mul : 1.0f;
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const bool mine = row_ok && (!PAIR || (s >> 2) == (int)hi);  // (a row past the last: zeros)
      const uint32_t k = mine ? keep : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) raw[s][j] = (raw[s][j] ^ sign) & k;
    }
    if (kEb == 2 || a.q_dtype == MKV_DTYPE_F16) {  // q's type is the operands'
#pragma unroll
      for (int s = 0; s < 8; ++s) qop[s] = __builtin_bit_cast(Op16<CT>, raw[s]);
    } else {
      // a bf16 q's row times a power of two: exact in fp16 but for elements
      // below 2^-24 of the row's largest
      float top = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          top = max3(top, __uint_as_float(raw[s][j] << 16 & 0x7fffffffu), __uint_as_float(raw[s][j] & 0x7fff0000u));
      top = fmaxf(top, other_half(top));
      float f = 1.0f;
      if (top > 0.0f && top < __builtin_huge_valf()) {
        // (rows below 2^-60 take that one's power, so that f and its inverse are in
        // fp32's range; elements below 2^-82 lose bits)
        const int e = max(ilogbf(top), -60);
        f = ldexpf(1.0f, 8 - e);
        score_mul *= ldexpf(1.0f, e - 8);
      }
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const f16x2 x = {(_Float16)(__uint_as_float(raw[s][j] << 16) * f),
                           (_Float16)(__uint_as_float(raw[s][j] & 0xffff0000u) * f)};
          raw[s][j] = __builtin_bit_cast(uint32_t, x);
        }
#pragma unroll
      for (int s = 0; s < 8; ++s) qop[s] = __builtin_bit_cast(Op16<CT>, raw[s]);
    }
  }

  const uint8_t* mask_row = a.mask + (w.q0 + (row_ok ? row / a.group : 0)) * a.mask_stride;
  f32x16 acc[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) acc[b] = f32x16{};
  float m_run = kNegBig, l_run = 0.0f;

  // transposed V reads: within a 16-lane group, lane d of the result holds dim d
  // of keys 4h + 0..3 and 8 + 4h + 0..3 of 16.  16-bit: two reads, lane 4i + q
  // reading key i (+ 4h, + 8) at dims 4q; 1-byte: lane 2i + q key i at dims 8q.
  const int vg = (lane >> 4) & 1;
  const int vi = kEb == 2 ? (lane & 15) >> 2 : (lane & 15) >> 1;
  const int v_key = kEb == 2 ? 4 * h + vi : (vi & 3) + 4 * h + 2 * (vi & 4);
  const int v_chunk = kEb == 2 ? 2 * vg + ((lane & 3) >> 1) : vg;
  // A swizzled chunk's offset is linear in the chunk under xor: chunk 2 st + h of
  // K is base ^ st << 5, V's 32-dim block b is base ^ b << 6 (1-byte: << 5), and 8
  // keys on (16-bit) flips one more bit; 16 and 32 keys on do not reach the swizzle.
  const int k_base = T::offset(kg * TK + c, h);
  const int v_base = T::offset(kg * TK + v_key, v_chunk) + 8 * (lane & 1);
  struct VRaw {
    uint32_t w[kEb == 2 ? 4 : 2];
  };
  auto v_read = [&](int nb, int half, int b) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    char* const at = lds_v + (32 * nb + 16 * half) * T::kRow;
    VRaw r;
    if constexpr (kEb == 2) {
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + (v_base ^ b << 6))));
      const u32x2 up = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + (v_base ^ b << 6 ^ 32) + 8 * T::kRow)));
      r.w[0] = lo[0];
      r.w[1] = lo[1];
      r.w[2] = up[0];
      r.w[3] = up[1];
    } else {
      const i32x2 x = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(at + (v_base ^ b << 5)));
      r.w[0] = (uint32_t)x[0];
      r.w[1] = (uint32_t)x[1];
    }
    return r;
  };
  auto v_operand = [&](const VRaw& r) {
    if constexpr (kEb == 2)
      return __builtin_bit_cast(Op16<CT>, u32x4{r.w[0], r.w[1], r.w[2], r.w[3]});
    else
      return codes_to_f16<KV_DT>(r.w[0], r.w[1]);
  };

  // ---- a tile's steps ----
  constexpr int kReads = kEb == 2 ? 8 : 4;  // 16-byte reads of a key block's K
  struct KOps {
    u32x4 w[kReads];
  };
  struct VOps {
    VRaw w[2][4];
  };
  auto k_read = [&](int nb, KOps& k) {
#pragma unroll
    for (int j = 0; j < kReads; ++j)
      k.w[j] = *reinterpret_cast<const u32x4*>(lds_k + (k_base ^ j << 5) + 32 * nb * T::kRow);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto qk = [&](const KOps& k) {
    f32x16 s = f32x16{};
#pragma unroll
    for (int st = 0; st < 8; ++st) {
      if constexpr (kEb == 2)
        s = mfma32<CT>(__builtin_bit_cast(Op16<CT>, k.w[st]), qop[st], s);
      else
        s = mfma32<CT>(codes_to_f16<KV_DT>(k.w[st >> 1][2 * (st & 1)], k.w[st >> 1][2 * (st & 1) + 1]), qop[st], s);
    }
    return s;
  };
  const float* const ks = sc + (PAIR && hi ? 3 * TK : 0) + 4 * h;
  // scores of key block nb: K scales, -inf where the row does not see, and the
  // running maximum (with what is already summed, and the pending P of the block
  // before, brought to it)
  auto s_max = [&](f32x16& s, int nb, bool masked, uint32_t see, f32x16& pending, auto has_pending) {
    if constexpr (kTok) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(ks + 32 * nb + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * g + e] *= x[e];
      }
    }
    if (masked) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = (see >> e) & 1 ? s[e] : kNegInf;
    }
    float mx;
    if constexpr (kTok) {
      // of what P times its V scale comes to
      mx = kNegInf;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(ks + 2 * TK + 32 * nb + 8 * g);
        float t[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) t[j] = __builtin_fmaf(s[4 * g + j], score_mul, x[j]);
        mx = max3(max3(mx, t[0], t[1]), t[2], t[3]);
      }
      mx = fmaxf(mx, other_half(mx));
      mx = fmaxf(mx - kLift, kNegBig);
    } else {
      float my = max3(s[3], s[4], s[5]);
      mx = max3(s[0], s[1], s[2]);
#pragma unroll
      for (int e = 6; e < 14; e += 4) {
        mx = max3(mx, s[e], s[e + 1]);
        my = max3(my, s[e + 2], s[e + 3]);
      }
      mx = max3(mx, s[14], s[15]);
      mx = max3(mx, my, my);
      mx = fmaxf(mx, other_half(mx));
      mx = fmaxf(__builtin_fmaf(mx, score_mul, -kLift), kNegBig);
    }
    const float m_new = mx > m_run + kRescaleSlack ? mx : m_run;
    if (__builtin_amdgcn_ballot_w64(m_new != m_run)) {
      // (before the first visible key there is nothing to rescale but marks)
      const float alpha = m_run == kNegBig ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      if constexpr (kTok) l_run = mul_exp2(l_run, m_run - m_new);
      else l_run *= alpha;
      m_run = m_new;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] *= alpha;
      if constexpr (decltype(has_pending)::value) {
#pragma unroll
        for (int e = 0; e < 16; ++e) pending[e] *= alpha;
      }
    }
  };
  auto s_exp = [&](f32x16& s, int nb, bool masked, uint32_t see) {
    float sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      f32x4 x;
      if constexpr (kTok) x = *reinterpret_cast<const f32x4*>(ks + TK + 32 * nb + 8 * g);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * g + j;
        s[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e], score_mul, -m_run));
        sum[g & 1] += s[e];
        if constexpr (kTok) {
          s[e] *= x[j];
          if (masked) s[e] = (see >> e) & 1 ? s[e] : 0.0f;
        }
      }
    }
    l_run += sum[0] + sum[1];
  };
  auto v_block = [&](int nb, VOps& v) {
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int b = 0; b < 4; ++b) v.w[half][b] = v_read(nb, half, b);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto pv = [&](const VOps& v, const f32x16& p) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      Op16<CT> ph, pl;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (CT == MKV_DTYPE_BF16)
          ph[j] = (__bf16)p[8 * half + j];
        else
          ph[j] = (_Float16)p[8 * half + j];
      }
      if constexpr (CT == MKV_DTYPE_BF16) {
        // bf16 holds P to 8 bits: a second term carries the rest, so that a
        // row whose weight sits on few keys is as exact as decode's.  p - hi is
        // one dot product a value: hi_pair . (-1, 0) or (0, -1), + p
        uint32_t lo_bits = 0x0000bf80u, hi_bits = 0xbf800000u;
        asm volatile("" : "+s"(lo_bits), "+s"(hi_bits));
        const bf16x2 neg_lo = __builtin_bit_cast(bf16x2, lo_bits), neg_hi = __builtin_bit_cast(bf16x2, hi_bits);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const bf16x2 hp = {ph[j], ph[j + 1]};
          pl[j] = (__bf16)__builtin_amdgcn_fdot2_f32_bf16(hp, neg_lo, p[8 * half + j], false);
          pl[j + 1] = (__bf16)__builtin_amdgcn_fdot2_f32_bf16(hp, neg_hi, p[8 * half + j + 1], false);
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[b] = mfma32<CT>(v_operand(v.w[half][b]), ph, acc[b]);
      if constexpr (CT == MKV_DTYPE_BF16) {
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[b] = mfma32<CT>(v_operand(v.w[half][b]), pl, acc[b]);
      }
    }
  };
  // N MFMAs with V vector operations after each: what the scheduler is asked for
  // where a key block's products stand beside the other's softmax
  auto mix = [&](auto n_tag, auto v_tag) {
#pragma unroll
    for (int i = 0; i < decltype(n_tag)::value; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x402, decltype(v_tag)::value, 0);
    }
  };

  for (int kb = kb0, turn = 0; kb < k1; kb += NK, turn ^= 1) {
    const int key0 = kg * TK;  // this wave's keys of the tile
    wait_vm<kDma>();  // K is here, V may be on its way
    if constexpr (kShared) meet();
    uint32_t present = 0;
    if constexpr (kShared) {
#pragma unroll
      for (int u = 0; u < TK / 16; ++u) present |= uniform(slots[turn * (NK / 16) + key0 / 16 + u]) >= 0 ? 1u << u : 0u;
    } else {
#pragma unroll
      for (int u = 0; u < kSubs; ++u) present |= left[u] > 0 ? 1u << u : 0u;
    }
    if constexpr (kTok) {
#pragma unroll
      for (int i = 0; i < kScLoads; ++i) {
        const int at = lane + 64 * i, which = at / TK, to = at + (which >> 1) * TK;
        sc[to] = sc_raw[i];
        if (which & 1) sc[to + TK] = scale_log2(sc_raw[i]);
      }
    }
    // ---- what this lane's row sees of keys that are not all prefix: element
    // e of key block nb is key 32 nb + 8 (e >> 2) + 4h + (e & 3) ----
    const bool drafted = kb + key0 + TK > prefix;
    const bool masked = drafted || kb + key0 + TK > k1 || present != (1u << TK / 16) - 1;
    uint32_t seen[NB] = {};
    if (masked) {
      uint32_t few = 0;  // a mask narrower than a word
      if (drafted && row_ok && a.mask_cols < 4)
        for (int j = 0; j < a.mask_cols; ++j) few |= mask_row[j] ? 0xffu << 8 * j : 0u;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int kl = 32 * nb + 8 * g + 4 * h, t = kb + key0 + kl;
          const int j0 = t - prefix;  // the four keys' first column
          uint32_t x = 0;
          if (row_ok && j0 > -4 && j0 < a.mask_cols) {
            const int at = a.mask_cols < 4 ? 0 : min(max(j0, 0), a.mask_cols - 4);
            x = few;
            if (a.mask_cols >= 4) __builtin_memcpy(&x, mask_row + at, 4);
            x = j0 >= at ? x >> 8 * (j0 - at) : x << 8 * (at - j0);
          }
          const bool here = (present >> (kl >> 4)) & 1;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool vis = here && t + e < k1 && (j0 + e < 0 || (x >> 8 * e & 0xffu) != 0);
            seen[nb] |= vis ? 1u << (4 * g + e) : 0u;
          }
        }
      }
    }


    // ---- S^T = K Q^T of the first key block; all of K is read ----
    KOps k_ops[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) k_read(nb, k_ops[nb]);
    f32x16 s[NB];
    s[0] = qk(k_ops[0]);
    // ---- V is here; the next tile's K goes where this one's was ----
    wait_vm<0>();
    entry_use(kb + NK, e_ahead);
    if constexpr (kShared) {
      if (lane == 0) {
#pragma unroll
        for (int u = 0; u < kSubs; ++u) slots[(turn ^ 1) * (NK / 16) + sub0 / 16 + u] = left[u] > 0 ? slot[u] : -1;
      }
      meet();
    } else {
      wait_lds();
    }
    load_scales(kb + NK, turn ^ 1);
    dma(a.k, lds_k);
    if (kShared ? kb + NK > prefix : drafted) {
      bool found = false;
      constexpr int kScan = kShared ? NK * T::kChunks / kThreads : TK * T::kChunks / 64;
      for (int i = 0; i < kScan; ++i) {
        const int at = kShared ? i * kThreads + tid : kg * TK * T::kChunks + i * 64 + lane;
        const u32x4 v = *reinterpret_cast<const u32x4*>(lds_v + 16 * at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if constexpr (kEb == 2) found |= not_finite2<CT>(v[j]);
          // (e4m3: S.1111.111 alone)
          else if constexpr (KV_DT != kKvI8PerToken)
            found |= (((v[j] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }
      }
      if (kShared ? __syncthreads_or(found) : __builtin_amdgcn_ballot_w64(found) != 0) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          f32x16 marks = f32x16{};
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              Op16<CT> vt = v_operand(v_read(nb, half, b)), sees;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float one = !masked || ((seen[nb] >> (8 * half + j)) & 1) ? 1.0f : 0.0f;
                if constexpr (CT == MKV_DTYPE_BF16) {
                  vt[j] = (__bf16)mark_of((float)vt[j]);
                  sees[j] = (__bf16)one;
                } else {
                  vt[j] = (_Float16)mark_of((float)vt[j]);
                  sees[j] = (_Float16)one;
                }
              }
              marks = mfma32<CT>(vt, sees, marks);
            }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[b][e] += marked_value(marks[e]);
        }
        if constexpr (kShared) meet();
        for (int i = 0; i < kScan * 4; ++i) {
          const int at = kShared ? i * kThreads + tid : kg * TK * T::kChunks * 4 + i * 64 + lane;
          uint32_t* v = reinterpret_cast<uint32_t*>(lds_v) + at;
          uint32_t x = *v;
          if constexpr (kEb == 2) {
            constexpr uint32_t e = CT == MKV_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
            if ((x & e) == e) x &= 0xffff0000u;
            if (((x >> 16) & e) == e) x &= 0xffffu;
          } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if ((x >> 8 * j & 0x7fu) == 0x7fu) x &= ~(0xffu << 8 * j);
          }
          *v = x;
        }
        if constexpr (kShared) meet();
        else wait_lds();
      }
    }

    // ---- softmax and O^T += V^T P^T: the second block's K Q^T beside the first's
    // exponentials, the first's P V beside the second's ----
    VOps v_ops[NB];
    s_max(s[0], 0, masked, seen[0], s[0], std::false_type{});
    v_block(0, v_ops[0]);
    if constexpr (NB == 2) {
      s[1] = qk(k_ops[1]);
      s_exp(s[0], 0, masked, seen[0]);
      mix(std::integral_constant<int, 8>{}, std::integral_constant<int, kEb == 2 ? 6 : 10>{});
      // (held here: the compiler would sink the exponentials to their use, behind
      // the branches below and out of the MFMAs' shadow)
      asm volatile("" : "+v"(s[0]), "+v"(l_run));
      s_max(s[1], 1, masked, seen[NB - 1], s[0], std::true_type{});
      v_block(1, v_ops[NB - 1]);
      pv(v_ops[0], s[0]);
      s_exp(s[1], 1, masked, seen[NB - 1]);
      mix(std::integral_constant<int, CT == MKV_DTYPE_BF16 ? 16 : 8>{}, std::integral_constant<int, CT == MKV_DTYPE_BF16 ? 4 : 10>{});
      __builtin_amdgcn_sched_barrier(0);
    } else {
      s_exp(s[0], 0, masked, seen[0]);
    }
    // ---- all of V is read: the next tile's goes where it was ----
    if constexpr (kShared) meet();
    else wait_lds();
    e_ahead = entry_load(kb + 2 * NK);
    dma(a.v, lds_v);
    pv(v_ops[NB - 1], s[NB - 1]);
  }
  wait_vm<0>();
  if (zeroes) zero_rows_past(a, w);

  // ---- the key groups' results: each group sums its share of the dims ----
  float l = l_run + other_half(l_run);
  constexpr int kMine = 4 / KG;  // 32-dim blocks: kMine * kg ..
  f32x16 res[kMine];
  if constexpr (KG > 1) {
    if (h == 0) join_ml[wave * 32 + c] = f32x2{m_run, l};
    meet();  // (all reads of the tiles are done, too)
    float m = kNegBig;
    f32x2 ml[KG];
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      ml[g] = join_ml[(g * R + rg) * 32 + c];
      m = fmaxf(m, ml[g][0]);
    }
    const float f = __builtin_amdgcn_exp2f(m_run - m);
    m_run = m;
    l = 0.0f;
#pragma unroll
    for (int g = 0; g < KG; ++g)
      l += kTok ? mul_exp2(ml[g][1], ml[g][0] - m) : ml[g][1] * __builtin_amdgcn_exp2f(ml[g][0] - m);
    // a 4 KB block to each group's summands from the others
    auto at = [&](int to, int i, int from) {  // (from != to; i: the block of the group's)
      const int n = ((to * kMine + i) * (KG - 1) + from - (from > to)) * R + rg;
      return reinterpret_cast<u32x4*>((n < kBuf / 4096 ? lds_k : lds_v - kBuf) + n * 4096) + lane;
    };
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      acc[b] *= f;
      if (b / kMine != kg) {
        u32x4* const o = at(b / kMine, b % kMine, kg);
#pragma unroll
        for (int e = 0; e < 16; e += 4)
          o[e * 16] = u32x4{__float_as_uint(acc[b][e]), __float_as_uint(acc[b][e + 1]), __float_as_uint(acc[b][e + 2]),
                            __float_as_uint(acc[b][e + 3])};
      }
    }
    meet();
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
      f32x16 mine = acc[i];
#pragma unroll
      for (int g = 1; g < KG; ++g) mine = kg == g ? acc[g * kMine + i] : mine;
      res[i] = f32x16{};
#pragma unroll
      for (int g = 0; g < KG; ++g) {  // (in the groups' order for each)
        if (g == kg) {
          res[i] += mine;
        } else {
          const u32x4* const o = at(kg, i, g);
#pragma unroll
          for (int e = 0; e < 16; ++e) res[i][e] += __uint_as_float(o[(e & 12) * 16][e & 3]);
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < kMine; ++i) res[i] = acc[i];
  }
  if (!row_ok) return;
  if (split) {
    const int64_t at = ((int64_t)place.unit * a.num_kv_heads + w.kvh) * a.row_cap + row;
    float* o = a.ws_o + at * kHeadDim + 32 * kMine * kg + 4 * h;
#pragma unroll
    for (int i = 0; i < kMine; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        st16(o + 32 * i + 2 * e, u32x4{__float_as_uint(res[i][e]), __float_as_uint(res[i][e + 1]),
                                       __float_as_uint(res[i][e + 2]), __float_as_uint(res[i][e + 3])});
    if (h == 0 && kg == 0) *reinterpret_cast<f32x2*>(a.ws_ml + 2 * at) = f32x2{m_run, l};
    return;
  }
  float norm = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  if constexpr (KV_DT == MKV_DTYPE_FP8E4M3) norm *= load_uniform_f32(a.v_scale);
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    const int b = kMine * kg + i;
    if (PAIR && (b >> 1) != (int)hi) continue;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float x[4] = {res[i][e] * norm, res[i][e + 1] * norm, res[i][e + 2] * norm, res[i][e + 3] * norm};
      store4(a.out, a.q_dtype, q_off + 32 * (PAIR ? b & 1 : b) + 2 * e + 4 * h, x);
    }
  }
}

template <int KV_DT, int R, int KG, bool PAIR>
__global__ __launch_bounds__(64 * R * KG) __attribute__((amdgpu_waves_per_eu(2))) void tree_attention_kernel(TreeArgs a) {
  tree_attention_body<KV_DT, R, KG, PAIR>(a);
}

// Rows of sequences in several splits: half a wave two rows, four dims a lane.
// Z waves of a workgroup share the splits of their rows.
template <int Z>
constexpr int kJoinRows = 16 / Z;  // a workgroup
MKV_DEV float half_max(float x) {  // of the 32 lanes
  auto get = [&](auto ctrl) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x = fmaxf(x, get(std::integral_constant<int, 0xB1>{}));   // lane ^ 1, ^ 2, then within 8, 16
  x = fmaxf(x, get(std::integral_constant<int, 0x4E>{}));
  x = fmaxf(x, get(std::integral_constant<int, 0x141>{}));
  x = fmaxf(x, get(std::integral_constant<int, 0x140>{}));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int UNIT, int Z, int KV_DT, bool PAIR>
MKV_DEV void tree_join_body(const TreeArgs& a) {
  constexpr int kAhead = 4;  // splits whose loads are in flight
  Place place;
  place.kvh = blockIdx.x % a.num_kv_heads;
  const int n = Units<UNIT>(a).of_sequence(blockIdx.x / a.num_kv_heads, place);
  if (n <= 1) return;
  const Work w = find_work(a, place);
  const int c = threadIdx.x & 31, wave = uniform(threadIdx.x >> 6);
  const int row0 = blockIdx.y * kJoinRows<Z> + 2 * ((wave / Z) * 2 + (threadIdx.x >> 5 & 1));
  if (blockIdx.y * kJoinRows<Z> >= w.rows || (Z == 1 && row0 >= w.rows)) return;
  const bool one = row0 < w.rows, two = row0 + 1 < w.rows;
  const int64_t at = ((int64_t)place.unit * a.num_kv_heads + w.kvh) * a.row_cap + (one ? row0 : 0),
                step = (int64_t)a.num_kv_heads * a.row_cap;
  const float* const ml = a.ws_ml + 2 * at;
  const float* const o = a.ws_o + at * kHeadDim + 4 * c;
  f32x2 x_ml[2][kAhead];
  f32x4 x_o[2][kAhead];
  auto load = [&](int z0) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int64_t i = min(z0 + j, n - 1) * step;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        x_ml[r][j] = *reinterpret_cast<const f32x2*>(ml + 2 * (i + (r && two)));
        x_o[r][j] = *reinterpret_cast<const f32x4*>(o + (i + (r && two)) * kHeadDim);
      }
    }
  };
  load(wave % Z * kAhead);
  float m[2] = {kNegBig, kNegBig}, l[2] = {0.0f, 0.0f};
  f32x4 sum[2] = {};
  for (int z = c; z < n; z += 32) {  // the largest maximum first, a lane a split
    m[0] = fmaxf(m[0], ml[2 * z * step]);
    m[1] = fmaxf(m[1], ml[2 * (z * step + two)]);
  }
  m[0] = half_max(m[0]);
  m[1] = half_max(m[1]);
  for (int z0 = wave % Z * kAhead; z0 < n; z0 += Z * kAhead) {
    if (z0 >= Z * kAhead) load(z0);
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (z0 + j < n) {
          const float f = __builtin_amdgcn_exp2f(x_ml[r][j][0] - m[r]);
          l[r] += kPerTokenScale<KV_DT> ? mul_exp2(x_ml[r][j][1], x_ml[r][j][0] - m[r]) : x_ml[r][j][1] * f;
          sum[r] += x_o[r][j] * f;
        }
      }
  }
  if constexpr (Z > 1) {
    __shared__ f32x4 part[Z - 1][2][64];
    __shared__ float part_l[Z - 1][2][64];
    const int lane = threadIdx.x & 63;
    if (wave > 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        part[wave - 1][r][lane] = sum[r];
        part_l[wave - 1][r][lane] = l[r];
      }
    }
    __syncthreads();
    if (wave > 0 || !one) return;
#pragma unroll
    for (int z = 1; z < Z; ++z)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        sum[r] += part[z - 1][r][lane];
        l[r] += part_l[z - 1][r][lane];
      }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    if (r && !two) return;
    float norm = l[r] > 0.0f ? 1.0f / l[r] : l[r] == 0.0f ? 0.0f : l[r];
    if constexpr (KV_DT == MKV_DTYPE_FP8E4M3) norm *= load_uniform_f32(a.v_scale);
    bool hi = false;
    const int64_t off = row_offset<PAIR>(a, w, row0 + r, hi);
    if (PAIR && (c >= 16) != hi) continue;
    const float x[4] = {sum[r][0] * norm, sum[r][1] * norm, sum[r][2] * norm, sum[r][3] * norm};
    store4(a.out, a.q_dtype, off + 4 * (PAIR ? c & 15 : c), x);
  }
}
// (KV_DT: FP8 per tensor, FP8 per token and head for both formats with such
// scales, fp32 for the rest)
template <int UNIT, int Z, int KV_DT, bool PAIR>
__global__ __launch_bounds__(256) void tree_join_kernel(TreeArgs a) {
  tree_join_body<UNIT, Z, KV_DT, PAIR>(a);
}

// fp32 caches: products and sums in fp32 on the 32x32x2 fp32 MFMA, one row group
// of 32 rows and four key groups, each of which loads its own 32 keys of a tile and
// meets the others at the end alone.  Lane (c, h) supplies K[key c][64h + st] and
// q[row c][64h + st] at step st, and for O^T its own keys' P again.  A tile's 128
// MFMAs a wave (8192 cycles) and its 128 KB a CU take about as long as each other:
// K and V have a buffer each, whose next tile goes out as soon as its last operands
// are read, and one workgroup fills a CU's LDS (60 sequences of 300-800 keys with 16
// drafted tokens, 8 KV heads: 102 us, 2.9 TB/s; with one buffer and four barriers a
// tile 248 us).
// LDS rows of 512 bytes, 16-byte chunk i at i ^ swz(key): one-to-one on 16 keys (K
// operands), and keys 4 apart in the two halves of 256 bytes (V's).
template <bool PAIR>
MKV_DEV void tree_attention_f32_body(const TreeArgs& a) {
  constexpr int KG = 4, TK = 32, NK = TK * KG, kRow = 4 * kHeadDim, kDma = TK * kRow / 1024, kSubs = TK / 16;
  __shared__ __align__(16) char lds_k[NK * kRow], lds_v[NK * kRow];
  const int tid = threadIdx.x, lane = tid & 63, kg = uniform(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  Place place;
  if (!find_place<NK>(a, place)) return;
  const int len = place.len;
  const Work w = find_work(a, place);
  if (place.rb == 0 && place.z == 0 && w.kvh == 0) zero_rows_past(a, w);
  if (place.rb * 32 >= w.rows) return;
  const int kb0 = place.z * len, k1 = (int)min((int64_t)kb0 + len, (int64_t)w.ctx);
  const int prefix = (int)min(w.prefix, (int64_t)0x7fffffff);
  const bool split = w.ctx > len;
  const int row = place.rb * 32 + c;
  const bool row_ok = row < w.rows;
  bool hi = false;
  const int64_t q_off = row_offset<PAIR>(a, w, row_ok ? row : 0, hi);
  const float score_mul = a.sm_scale * kLog2e;
  float qv[64];
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    const u32x4 v = ld16(reinterpret_cast<const float*>(a.q) + q_off + (PAIR ? 0 : 64 * h) + i);  // (within q for any row)
#pragma unroll
    for (int j = 0; j < 4; ++j) qv[i + j] = __uint_as_float(v[j]);
  }

  // ---- loads of tiles, as above: two keys a load, a sub-tile of 16 keys never
  // across a block ----
  const int64_t row_bytes = (int64_t)a.num_kv_heads * kRow;
  const int64_t head_bytes = (int64_t)w.kvh * kRow;
  const int own0 = kg * TK;
  auto swz = [](int key) { return (key & 3) | (key & 4) << 1 | (key & 8) >> 1; };
  uint32_t voff[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) voff[i] = (uint32_t)((2 * i + h) * row_bytes) + 16 * (c ^ swz(2 * i + h));
  int32_t slot[kSubs], left[kSubs];
  const int32_t* bt_row = a.idx.block_tables + (int64_t)w.seq * a.idx.bt_stride;
  auto entry_load = [&](int kb) -> int32_t {
    const int blk = (kb + own0 + 16 * h) >> a.idx.bs_log2;
    return bt_row[min(blk, a.idx.max_blocks - 1)];
  };
  auto entry_use = [&](int kb, int32_t e) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      const int t = kb + own0 + 16 * u;
      const int phys = __builtin_amdgcn_readlane(e, 32 * u);
      const bool ok = t < k1 && phys >= 0 && phys < (int)a.idx.num_blocks;
      slot[u] = ok ? (phys << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : 0;
      left[u] = ok ? min(k1 - t, 16) : 0;
    }
  };
  auto dma = [&](const char* pool, char* buf) {
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(pool + slot[u] * row_bytes + head_bytes), (short)0,
          left[u] > 0 ? (int)((left[u] - 1) * row_bytes + kRow) : 0, 0x00020000);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            r, (__attribute__((address_space(3))) void*)(buf + (own0 + u * 16) * kRow + i * 1024), 16, voff[i], 0, 0, 0);
    }
  };
  int32_t e_ahead = 0;
  if (kb0 < k1) {
    e_ahead = entry_load(kb0);
    const int32_t e_next = entry_load(kb0 + NK);
    entry_use(kb0, e_ahead);
    e_ahead = e_next;
    dma(a.k, lds_k);
    dma(a.v, lds_v);
  }
  const bool mine = row_ok && (!PAIR || h == (int)hi);
#pragma unroll
  for (int i = 0; i < 64; ++i) qv[i] = mine ? qv[i] : 0.0f;

  const uint8_t* mask_row = a.mask + (w.q0 + (row_ok ? row / a.group : 0)) * a.mask_stride;
  const int k_base = (own0 + c) * kRow + ((16 * h ^ swz(c)) << 4);
  const int v_base = (own0 + 4 * h) * kRow + (((c >> 2) ^ 8 * h) << 4) + 4 * (c & 3);
  f32x16 acc[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) acc[b] = f32x16{};
  float m_run = kNegBig, l_run = 0.0f;
  for (int kb = kb0; kb < k1; kb += NK) {
    wait_vm<kDma>();  // K is here, V may be on its way
    uint32_t present = 0;
#pragma unroll
    for (int u = 0; u < kSubs; ++u) present |= left[u] > 0 ? 1u << u : 0u;
    const bool drafted = kb + own0 + TK > prefix;
    uint32_t seen = 0xffffu;  // element e is key 8 (e >> 2) + 4h + (e & 3)
    if (drafted || kb + own0 + TK > k1 || present != (1u << kSubs) - 1) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int kl = 8 * (e >> 2) + 4 * h + (e & 3), t = kb + own0 + kl, j = t - prefix;
        bool vis = t < k1 && ((present >> (kl >> 4)) & 1);
        if (vis && j >= 0) vis = row_ok && j < a.mask_cols && mask_row[j] != 0;
        seen &= vis ? 0xffffu : ~(1u << e);
      }
    }
    u32x4 kw[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) kw[i] = *reinterpret_cast<const u32x4*>(lds_k + (k_base ^ i << 4));
    f32x16 s = f32x16{}, s2 = f32x16{};
#pragma unroll
    for (int i = 0; i < 16; ++i) {
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kw[i][j]), qv[4 * i + j], s, 0, 0, 0);
        s2 = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kw[i][j + 1]), qv[4 * i + j + 1], s2, 0, 0, 0);
      }
    }
    // ---- V is here; the next tile's K goes where this one's was ----
    wait_vm<0>();
    entry_use(kb + NK, e_ahead);
    wait_lds();
    dma(a.k, lds_k);
    float v[4][16];
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int b = 0; b < 4; ++b)
        v[b][e] = *reinterpret_cast<const float*>(lds_v + (v_base ^ (8 * b ^ (e & 3) ^ (e & 4)) << 4) +
                                                  (8 * (e >> 2) + (e & 3)) * kRow);
    float mx = kNegInf;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[e] = (seen >> e) & 1 ? (s[e] + s2[e]) * score_mul : kNegInf;
      mx = fmaxf(mx, s[e]);
    }
    mx = fmaxf(fmaxf(mx, other_half(mx)), kNegBig);
    const float m_new = fmaxf(mx, m_run);
    if (__builtin_amdgcn_ballot_w64(m_new != m_run)) {
      const float alpha = m_run == kNegBig ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[b] *= alpha;
    }
    float p[16], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = __builtin_amdgcn_exp2f(s[e] - m_run);
      sum += p[e];
    }
    l_run += sum;
    // ---- all of V is read: the next tile's goes where it was ----
    wait_lds();
    e_ahead = entry_load(kb + 2 * NK);
    dma(a.v, lds_v);
    if (drafted) {
      bool found = false;
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) found |= not_finite(v[b][e]);
      if (__builtin_amdgcn_ballot_w64(found)) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          f32x16 marks = f32x16{};
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            marks = __builtin_amdgcn_mfma_f32_32x32x2f32(mark_of(v[b][e]), (seen >> e) & 1 ? 1.0f : 0.0f, marks, 0, 0, 0);
            v[b][e] = not_finite(v[b][e]) ? 0.0f : v[b][e];
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[b][e] += marked_value(marks[e]);
        }
      }
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
#pragma unroll
      for (int b = 0; b < 4; ++b) acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[b][e], p[e], acc[b], 0, 0, 0);
  }
  wait_vm<0>();
  __syncthreads();
  float* part = reinterpret_cast<float*>(lds_k);
  static_assert((KG - 1) * 64 * 66 * 4 <= NK * kRow, "the join fits the tile");
  if (kg > 0) {
    float* o = part + (kg - 1) * 64 * 66;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[(16 * b + e) * 64 + lane] = acc[b][e];
    o[64 * 64 + lane] = m_run;
    o[65 * 64 + lane] = l_run;
  }
  __syncthreads();
  if (kg > 0) return;
  for (int g = 1; g < KG; ++g) {
    const float* o = part + (g - 1) * 64 * 66;
    const float m = o[64 * 64 + lane], l = o[65 * 64 + lane];
    const float m_new = fmaxf(m, m_run);
    const float fa = __builtin_amdgcn_exp2f(m_run - m_new), fb = __builtin_amdgcn_exp2f(m - m_new);
    m_run = m_new;
    l_run = l_run * fa + l * fb;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][e] = acc[b][e] * fa + o[(16 * b + e) * 64 + lane] * fb;
  }
  const float l = l_run + other_half(l_run);
  if (!row_ok) return;
  float norm = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  const int64_t at = ((int64_t)place.unit * a.num_kv_heads + w.kvh) * a.row_cap + row;
  if (split && h == 0) {
    a.ws_ml[2 * at] = m_run;
    a.ws_ml[2 * at + 1] = l;
  }
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    if (PAIR && !split && (b >> 1) != (int)hi) continue;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float f = split ? 1.0f : norm;
      const float x[4] = {acc[b][e] * f, acc[b][e + 1] * f, acc[b][e + 2] * f, acc[b][e + 3] * f};
      if (split)
        store4(a.ws_o, MKV_DTYPE_F32, at * kHeadDim + 32 * b + 2 * e + 4 * h, x);
      else
        store4(a.out, MKV_DTYPE_F32, q_off + 32 * (PAIR ? b & 1 : b) + 2 * e + 4 * h, x);
    }
  }
}

template <bool PAIR>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(1))) void tree_attention_f32_kernel(TreeArgs a) {
  tree_attention_f32_body<PAIR>(a);
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

// The form of a launch, from sizes the host knows.
struct Plan {
  int row_groups;  // 32-row groups of a workgroup
  int row_blocks;
  int row_cap;
  int unit;        // keys of a tile
  int shares;
  int min_split;
  bool splits;
  int64_t units;   // at most
};

Plan make_plan(int num_seqs, int64_t total_q, int kernel_kv_heads, int kernel_group, int mask_cols, int64_t capacity,
               bool f32) {
  Plan p;
  const int64_t toks = mask_cols < total_q ? mask_cols : total_q;
  const int64_t rows = toks * kernel_group;
  p.row_groups = f32 || rows <= 32 ? 1 : rows <= 64 ? 2 : 4;
  p.row_blocks = (int)((rows + 32 * p.row_groups - 1) / (32 * p.row_groups));
  if (p.row_blocks < 1) p.row_blocks = 1;
  p.row_cap = p.row_blocks * 32 * p.row_groups;
  p.unit = p.row_groups == 4 ? 64 : 128;
  // Workgroups that run at once: two a CU (fp32: one).  Where the sequences leave
  // some free, their keys are dealt out so that all fit one round (a sequence's last
  // split may be short: num_seqs shares are kept back); where they do not fit a
  // round, in pieces of a quarter round; many sequences split only those of more
  // than twice the mean.
  const int64_t slots = f32 ? 256 : 512;
  const int64_t round = slots / ((int64_t)kernel_kv_heads * p.row_blocks) > 0 ? slots / ((int64_t)kernel_kv_heads * p.row_blocks) : 1;
  int64_t shares;
  if (num_seqs <= round)
    shares = round - num_seqs > round / 4 ? round - num_seqs : round / 4;
  else if (num_seqs < 4 * round)
    shares = 4 * round - num_seqs > round ? 4 * round - num_seqs : round;
  else
    shares = num_seqs / 2;
  p.shares = (int)(shares < 1 ? 1 : shares);
  p.min_split = num_seqs * 4 <= round ? 128 : num_seqs * 2 <= round ? 256 : 1024;
  const int64_t most = (capacity + p.min_split - 1) / p.min_split;
  // Short block tables are not split at all: a second launch and the partial
  // results cost more than the tiles one after another where the host's calls follow
  // each other (one sequence, 8 KV heads, bf16: 16 rows of 700 keys 13.4 us against
  // 17.6, of 1000 15.2 against 17.5; 64 rows of 380 15.8 against 16.9, of 500 17.7
  // against 17.0; 128 rows of 250 16.5 against 16.8, of 380 19.7 against 17.0; fp32 at
  // 250 keys 21.1 against 19.3), and for many sequences anyhow (60 of 16 rows and
  // 300-800 keys: bf16 30.4 against 33.2, FP8 20.4 against 23.5; one of 700 in a graph
  // 13.1 against 12.1).  By the table's width: the contexts are on the device.
  const int64_t whole = f32 ? 128 : p.row_groups == 1 ? 1024 : p.row_groups == 2 ? 384 : 256;
  p.splits = most > 1 && capacity > whole;
  p.units = !p.splits ? num_seqs : num_seqs + shares < num_seqs * most ? num_seqs + shares : num_seqs * most;
  return p;
}

size_t workspace_of(const Plan& p, int kernel_kv_heads) {
  return p.splits ? (size_t)p.units * kernel_kv_heads * p.row_cap * (kHeadDim + 2) * sizeof(float) : 0;
}

template <int KV_DT, bool PAIR>
int launch_tree(const TreeArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.units * a.num_kv_heads * p.row_blocks));
  if constexpr (KV_DT == MKV_DTYPE_F32) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_f32_kernel<PAIR>), grid, dim3(256), 0, s, a);
  } else {
    switch (p.row_groups) {
      case 1: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 1, 4, PAIR>), grid, dim3(256), 0, s, a); break;
      case 2: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 2, 2, PAIR>), grid, dim3(256), 0, s, a); break;
      default: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 4, 1, PAIR>), grid, dim3(256), 0, s, a); break;
    }
  }
  if (hipError_t e = hipGetLastError()) return (int)e;
  if (p.splits) {
    constexpr int kFormat = kPerTokenScale<KV_DT> ? kKvFp8PerToken : KV_DT == MKV_DTYPE_FP8E4M3 ? KV_DT : MKV_DTYPE_F32;
    // (few sequences in many splits each: the waves share them)
    auto join = [&](auto unit, auto z) {
      constexpr int kUnit = decltype(unit)::value, kZ = decltype(z)::value;
      const dim3 jgrid((unsigned)(a.num_seqs * a.num_kv_heads), (unsigned)((p.row_cap + kJoinRows<kZ> - 1) / kJoinRows<kZ>));
      hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_join_kernel<kUnit, kZ, kFormat, PAIR>), jgrid, dim3(256), 0, s, a);
    };
    using I1 = std::integral_constant<int, 1>;
    using I4 = std::integral_constant<int, 4>;
    const bool many = p.units >= 8 * (int64_t)a.num_seqs && p.row_cap <= 4096;
    if (p.unit == 128)
      many ? join(std::integral_constant<int, 128>{}, I4{}) : join(std::integral_constant<int, 128>{}, I1{});
    else
      many ? join(std::integral_constant<int, 64>{}, I4{}) : join(std::integral_constant<int, 64>{}, I1{});
    return (int)hipGetLastError();
  }
  return MKV_OK;
}

constexpr int64_t kMaxRows = 65535 * 16 - 255;
constexpr int64_t kMaxGrid = 0xffffff;  // workgroups of 256 threads: below 2^32 threads

int check_tree(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
               int max_blocks, int mask_cols) {
  if (num_seqs < 0 || total_q < 0 || total_q > 0x7fffffff || num_heads <= 0 || num_kv_heads <= 0 || max_blocks < 0 ||
      mask_cols < 0)
    return MKV_ERR_BAD_SHAPE;
  if (head_dim != 128 && !(head_dim == 64 && num_kv_heads % 2 == 0)) return MKV_ERR_UNSUPPORTED_HEAD_DIM;
  const int g = num_heads / num_kv_heads;
  if (num_heads % num_kv_heads || g < 1 || g > (head_dim == 64 ? 8 : 16)) return MKV_ERR_UNSUPPORTED_GROUP;
  if (log2_exact(block_size) < 4) return MKV_ERR_BAD_BLOCK_SIZE;
  if ((int64_t)num_seqs * num_kv_heads > 0x7fffffff || (int64_t)max_blocks * block_size > 0x7fff0000)
    return MKV_ERR_BAD_SHAPE;
  // (a KV head's rows of a sequence: the join's grid)
  if ((mask_cols < total_q ? mask_cols : total_q) * g * (head_dim == 64 ? 2 : 1) > kMaxRows) return MKV_ERR_BAD_SHAPE;
  return MKV_OK;
}

Plan plan_of(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
             int max_blocks, int mask_cols, int kv_dtype, int& kernel_kv_heads) {
  const int pair = head_dim == 64 ? 2 : 1;
  const int kv = num_kv_heads / pair, g = num_heads / num_kv_heads * pair;
  kernel_kv_heads = kv;
  return make_plan(num_seqs, total_q, kv, g, mask_cols, (int64_t)max_blocks * block_size, kv_dtype == MKV_DTYPE_F32);
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_paged_tree_workspace_size(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads,
                                                int head_dim, int block_size, int max_blocks, int mask_cols,
                                                int kv_dtype) {
  if (check_tree(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols)) return 0;
  int kv;
  const Plan p = plan_of(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols, kv_dtype, kv);
  return workspace_of(p, kv);
}

extern "C" int mkv_paged_tree(void* out, const void* q, int q_dtype, const void* k_cache, const void* v_cache,
                              int kv_dtype, int64_t num_blocks, const float* k_scale, const float* v_scale,
                              int kv_scale_mode, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                              const void* context_lens, int context_lens_dtype, const int32_t* cu_seqlens_q,
                              const uint8_t* tree_mask, int64_t mask_stride, int mask_cols, int num_seqs,
                              int64_t total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
                              float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_tree(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols)) return st;
  // (token rows and, within 16 of them, bytes are counted in 32 bits)
  if (num_blocks < 0 || num_blocks * block_size > 0x7fffffff || num_kv_heads > (1 << 16)) return MKV_ERR_BAD_SHAPE;
  if (num_seqs == 0 || total_q == 0) return MKV_OK;
  const bool code = kv_dtype == MKV_DTYPE_FP8E4M3 || kv_dtype == MKV_DTYPE_I8;
  const bool token = code && kv_scale_mode == MKV_SCALE_PER_TOKEN_HEAD;
  if (kv_scale_mode != MKV_SCALE_PER_TENSOR && kv_scale_mode != MKV_SCALE_PER_TOKEN_HEAD) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (code ? q_dtype != MKV_DTYPE_BF16 && q_dtype != MKV_DTYPE_F16 : q_dtype != kv_dtype) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (kv_dtype == MKV_DTYPE_I8 && !token) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (!out || !q || !k_cache || !v_cache || !context_lens || !cu_seqlens_q || (max_blocks && !block_tables) ||
      (mask_cols && !tree_mask) || (code && (!k_scale || !v_scale)))
    return MKV_ERR_NULL_POINTER;
  if (context_lens_dtype != MKV_INDEX_I32 && context_lens_dtype != MKV_INDEX_I64) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (bt_stride < max_blocks || mask_stride < 0) return MKV_ERR_BAD_STRIDE;
  if ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) |
       reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(workspace)) & 15u)
    return MKV_ERR_MISALIGNED;
  int kv;
  const Plan p = plan_of(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols, kv_dtype, kv);
  if (p.units * kv * p.row_blocks > kMaxGrid) return MKV_ERR_BAD_SHAPE;
  if (workspace_of(p, kv) > workspace_bytes || (p.splits && !workspace)) return MKV_ERR_WORKSPACE_TOO_SMALL;
  const int pair = head_dim == 64 ? 2 : 1;
  TreeArgs a;
  a.out = out;
  a.q = q;
  a.k = reinterpret_cast<const char*>(k_cache);
  a.v = reinterpret_cast<const char*>(v_cache);
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.idx = PagedIndex{block_tables, bt_stride, max_blocks, num_blocks, log2_exact(block_size),
                     (int64_t)num_kv_heads * head_dim};
  a.ctx = context_lens;
  a.ctx_i64 = context_lens_dtype == MKV_INDEX_I64;
  a.cu = cu_seqlens_q;
  a.mask = tree_mask;
  a.mask_stride = mask_stride;
  a.mask_cols = mask_cols;
  a.num_seqs = num_seqs;
  a.total_q = total_q;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads / pair;
  a.scale_heads = num_kv_heads;
  a.group = num_heads / num_kv_heads * pair;
  a.q_dtype = q_dtype;
  a.sm_scale = sm_scale;
  a.splits = p.splits;
  a.shares = p.shares;
  a.min_split = p.min_split;
  a.row_cap = p.row_cap;
  a.row_blocks = p.row_blocks;
  a.ws_o = reinterpret_cast<float*>(workspace);
  a.ws_ml = a.ws_o + (size_t)p.units * kv * p.row_cap * kHeadDim;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const int fmt = token ? 0x100 | kv_dtype : kv_dtype;
#define MKV_TREE(F) \
  case F: return pair == 2 ? launch_tree<F, true>(a, p, s) : launch_tree<F, false>(a, p, s);
  switch (fmt) {
    MKV_TREE(MKV_DTYPE_F32)
    MKV_TREE(MKV_DTYPE_BF16)
    MKV_TREE(MKV_DTYPE_F16)
    MKV_TREE(MKV_DTYPE_FP8E4M3)
    MKV_TREE(kKvFp8PerToken)
    MKV_TREE(kKvI8PerToken)
    default: return MKV_ERR_UNSUPPORTED_DTYPE;
  }
#undef MKV_TREE
}
