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
// the running maximum moves only when a tile exceeds it by more than 2^8: P
// stays within 2^8 (exact in range in bf16 and fp16) and most tiles rescale
// nothing; any offset of the maximum cancels in the normalisation
constexpr float kRescaleSlack = 8.0f;

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
  int max_splits;    // 1: no partial results
  int target;        // workgroups that fill the GPU
  int min_split;     // keys
  int row_blocks;
  float* ws_o;       // partials: (seq, kv head, split, row cap, 128)
  float* ws_ml;      // (seq, kv head, split, row cap, 2)
  int row_cap;
};

// The share of a sequence that a split takes, the same for every sequence: the
// batch's keys over the workgroups that fill the GPU, in whole tiles.  At most
// max_splits for the longest.
template <int UNIT>
MKV_DEV int split_keys(const TreeArgs& a) {
  const int lane = threadIdx.x & 63;
  const int64_t cap = (int64_t)a.idx.max_blocks << a.idx.bs_log2;
  float sum = 0.0f;  // (a rule of thumb's accuracy, the same in every wave)
  int longest = 0;
  for (int s = lane; s < a.num_seqs; s += 64) {
    const int64_t c = min(max(load_index(a.ctx, s, a.ctx_i64), (int64_t)0), cap);
    sum += (float)c;
    longest = max(longest, (int)c);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    sum += __shfl_xor(sum, o);
    longest = max(longest, __shfl_xor(longest, o));
  }
  const float share = sum * (float)(a.num_kv_heads * a.row_blocks) / (float)a.target;
  int len = (int)fminf(share, 1.0e9f);
  len = max(max(len, a.min_split), (longest + a.max_splits - 1) / a.max_splits);
  len = (len + UNIT - 1) / UNIT * UNIT;
  return uniform(len);
}

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

// LDS tiles: 256-byte key rows of 16-bit elements in 16-byte chunks, chunk c of
// key at position c ^ swz(key).  swz is one-to-one on 16 keys (K operand reads:
// 16 keys, one chunk) and moves four neighbouring keys to the four 64-byte
// quarters of a row (transposed V reads: four keys, 32 dims), so both go without
// bank conflicts.
MKV_DEV int swz(int key) { return ((key & 3) << 2) | ((key >> 2) & 3); }
MKV_DEV int tile_offset(int key, int chunk) { return key * 256 + ((chunk ^ swz(key)) << 4); }

// Values that are not finite.  A drafted token that a row does not see weighs
// P = 0 there, and 0 * inf or 0 * NaN would still reach the row's output: where a
// tile of drafted tokens holds such values, the products take zeros in their
// place, and a product of marks with what each row sees says which outputs they
// belong to.  Marks of up to 64 keys add up without mixing.
constexpr float kMarkPos = 1.0f, kMarkNeg = 256.0f, kMarkNan = 32768.0f;
MKV_DEV float mark_of(float x) {
  return x != x ? kMarkNan : x == __builtin_huge_valf() ? kMarkPos : x == -__builtin_huge_valf() ? kMarkNeg : 0.0f;
}
MKV_DEV float marked_value(float n) {  // n > 0
  const bool nan = n >= kMarkNan;
  n -= kMarkNan * floorf(n * (1.0f / kMarkNan));
  const bool neg = n >= kMarkNeg, pos = n != kMarkNeg * floorf(n * (1.0f / kMarkNeg));
  return nan || (neg && pos) ? __builtin_nanf("") : pos ? __builtin_huge_valf() : -__builtin_huge_valf();
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

MKV_DEV Work find_work(const TreeArgs& a, int item) {
  Work w;
  w.kvh = item % a.num_kv_heads;
  w.seq = item / a.num_kv_heads;
  const int64_t q0 = min(max((int64_t)a.cu[w.seq], (int64_t)0), a.total_q);
  const int64_t q1 = min(max((int64_t)a.cu[w.seq + 1], q0), a.total_q);
  const int64_t c = max(load_index(a.ctx, w.seq, a.ctx_i64), (int64_t)0);
  w.q0 = q0;
  w.rows = (int)min(q1 - q0, (int64_t)a.mask_cols) * a.group;
  w.prefix = max(c - (q1 - q0), (int64_t)0);
  w.ctx = (int)min(c, (int64_t)a.idx.max_blocks << a.idx.bs_log2);
  return w;
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

template <int KV_DT, int R, int KG, bool PAIR>
__global__ __launch_bounds__(64 * R * KG) void tree_attention_kernel(TreeArgs a) {
  constexpr int CT = kOperand<KV_DT>;
  constexpr bool kTok = kPerTokenScale<KV_DT>;
  constexpr int kThreads = 64 * R * KG;
  constexpr int TK = KG == 1 ? 64 : 32;   // keys a wave takes of a tile
  constexpr int NK = TK * KG;             // keys of a tile
  constexpr int NB = TK / 32;
  constexpr int kEb = DTypeInfo<KV_DT>::kBytes;
  constexpr int kChunks = kHeadDim * kEb / 16;         // 16-byte chunks of a cached row
  constexpr int kKeysPerLoad = kThreads / kChunks;     // keys of one load of the workgroup
  constexpr int kLoads = NK / kKeysPerLoad;            // loads a thread, for K and for V each
  static_assert(NK % kKeysPerLoad == 0 && kLoads >= 1, "a tile is whole loads");
  constexpr int kJoinBytes = (KG - 1) * R * 64 * 66 * 4;
  constexpr int kTileBytes = 2 * NK * 256;
  __shared__ __align__(16) char lds[kTileBytes > kJoinBytes ? kTileBytes : kJoinBytes];
  __shared__ float sc[kTok ? (PAIR ? 4 : 2) * NK : 1];  // K then V scales, for each head of a pair
  char* const lds_k = lds;
  char* const lds_v = lds + NK * 256;

  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const int rg = wave % R, kg = wave / R;
  const int c = lane & 31, h = lane >> 5;
  const Work w = find_work(a, blockIdx.x);
  const int len = a.max_splits > 1 ? split_keys<NK>(a) : 0x7fffffff / NK * NK;
  const int64_t k0 = (int64_t)blockIdx.z * len;
  if (blockIdx.y == 0 && blockIdx.z == 0 && w.kvh == 0) zero_rows_past(a, w);
  if ((blockIdx.z > 0 && k0 >= w.ctx) || (int)blockIdx.y * 32 * R >= w.rows) return;
  const int kb0 = (int)k0, k1 = (int)min(k0 + len, (int64_t)w.ctx);
  const bool split = w.ctx > len;

  // ---- q: this lane's row, dims 16 s + 8 h .. + 7 of step s ----
  const int row = blockIdx.y * 32 * R + rg * 32 + c;
  const bool row_ok = row < w.rows;
  bool hi = false;
  const int64_t q_off = row_offset<PAIR>(a, w, row_ok ? row : 0, hi);
  float score_mul = a.sm_scale * kLog2e;
  Op16<CT> qop[8];
  {
    float x[8][8];
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const bool mine = row_ok && (!PAIR || (s >> 2) == (int)hi);
      const int d = 16 * (PAIR ? s & 3 : s) + 8 * h;
      u32x4 v{0, 0, 0, 0};
      if (mine) v = ld16(reinterpret_cast<const uint16_t*>(a.q) + q_off + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (a.q_dtype == MKV_DTYPE_BF16) {
          x[s][2 * j] = __uint_as_float(v[j] << 16);
          x[s][2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
        } else {
          x[s][2 * j] = f16_bits_to_f32(v[j] & 0xffffu);
          x[s][2 * j + 1] = f16_bits_to_f32(v[j] >> 16);
        }
        top = fmaxf(top, fmaxf(fabsf(x[s][2 * j]), fabsf(x[s][2 * j + 1])));
      }
    }
    // the loop keeps raw scores and wants score_mul > 0: a negative scale
    // moves its sign into q, a zero one makes q zero
    float f = 1.0f;
    if (!(score_mul > 0.0f) && score_mul == score_mul) {
      f = score_mul < 0.0f ? -1.0f : 0.0f;
      score_mul = score_mul < 0.0f ? -score_mul : 1.0f;
    }
    if constexpr (CT == MKV_DTYPE_F16) {
      // a row's q times a power of two: a bf16 q in fp16 is exact but for
      // elements below 2^-24 of the row's largest
      top = fmaxf(top, other_half(top));
      if (top > 0.0f && top < __builtin_huge_valf()) {
        const int e = ilogbf(top);
        f *= ldexpf(1.0f, 8 - e);
        score_mul *= ldexpf(1.0f, e - 8);
      }
    }
#pragma unroll
    for (int s = 0; s < 8; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if constexpr (CT == MKV_DTYPE_BF16)
          qop[s][j] = (__bf16)(x[s][j] * f);
        else
          qop[s][j] = (_Float16)(x[s][j] * f);
      }
  }
  if constexpr (KV_DT == MKV_DTYPE_FP8E4M3) score_mul *= load_uniform_f32(a.k_scale);

  const int64_t row_bytes = (int64_t)a.num_kv_heads * kHeadDim * kEb;
  const int64_t head_bytes = (int64_t)w.kvh * kHeadDim * kEb;
  const uint8_t* mask_row = a.mask + (w.q0 + (row_ok ? row / a.group : 0)) * a.mask_stride;

  f32x16 acc[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) acc[b] = f32x16{};
  float m_run = kNegBig, l_run = 0.0f;

  // ---- staging: 16 keys never straddle a block ----
  constexpr int kSubs = NK / 16;
  u32x4 st_k[kLoads], st_v[kLoads];
  const int ld_key = tid / kChunks, ld_ch = tid % kChunks;
  uint32_t present = 0, present_next = 0;
  constexpr int kScales = (PAIR ? 4 : 2) * NK, kScLoads = (kScales + kThreads - 1) / kThreads;
  float st_sc[kScLoads];
  auto load_tile = [&](int kb) {
    present_next = 0;
    int64_t slot[kSubs];
#pragma unroll
    for (int u = 0; u < kSubs; ++u) {
      const int t = kb + 16 * u;
      const int64_t phys = t < k1 ? a.idx.physical_block(w.seq, t >> a.idx.bs_log2) : -1;
      present_next |= phys >= 0 ? 1u << u : 0u;
      slot[u] = phys < 0 ? -1 : (phys << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1));
    }
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int key = u * kKeysPerLoad + ld_key;
      int64_t s = -1;
#pragma unroll
      for (int j = 0; j < kSubs; ++j)
        if (key >> 4 == j) s = slot[j];
      st_k[u] = st_v[u] = u32x4{0, 0, 0, 0};
      if (s >= 0 && kb + key < k1) {
        const int64_t o = (s + (key & 15)) * row_bytes + head_bytes + 16 * ld_ch;
        st_k[u] = ld16(a.k + o);
        st_v[u] = ld16(a.v + o);
      }
    }
    if constexpr (kTok) {
      constexpr int kHeads = PAIR ? 2 : 1;
#pragma unroll
      for (int i = 0; i < kScLoads; ++i) {
        // K head 0, V head 0, K head 1, V head 1
        const int key = (tid + i * kThreads) % NK, which = (tid + i * kThreads) / NK;
        int64_t s = -1;
#pragma unroll
        for (int j = 0; j < kSubs; ++j)
          if (key >> 4 == j) s = slot[j];
        st_sc[i] = 0.0f;
        if (which < 2 * kHeads && s >= 0 && kb + key < k1)
          st_sc[i] = ((which & 1) ? a.v_scale : a.k_scale)[(s + (key & 15)) * a.scale_heads + w.kvh * kHeads + (which >> 1)];
      }
    }
  };
  auto convert = [&](u32x4 v, u32x4& lo, u32x4& hi16) {  // 16 codes -> 16 exact fp16
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a0, a1;
      if constexpr (KV_DT == kKvI8PerToken) {
        a0 = __builtin_bit_cast(uint32_t, i8x2_to_f16x2<false>(v[j]));
        a1 = __builtin_bit_cast(uint32_t, i8x2_to_f16x2<true>(v[j]));
      } else {
        a0 = __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<false>(v[j]));
        a1 = __builtin_bit_cast(uint32_t, fp8x2_to_f16x2<true>(v[j]));
      }
      if (j < 2) {
        lo[2 * j] = a0;
        lo[2 * j + 1] = a1;
      } else {
        hi16[2 * j - 4] = a0;
        hi16[2 * j - 3] = a1;
      }
    }
  };
  auto store_tile = [&]() {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int key = u * kKeysPerLoad + ld_key;
      if constexpr (kEb == 2) {
        *reinterpret_cast<u32x4*>(lds_k + tile_offset(key, ld_ch)) = st_k[u];
        *reinterpret_cast<u32x4*>(lds_v + tile_offset(key, ld_ch)) = st_v[u];
      } else {
        u32x4 lo, hi16;
        convert(st_k[u], lo, hi16);
        *reinterpret_cast<u32x4*>(lds_k + tile_offset(key, 2 * ld_ch)) = lo;
        *reinterpret_cast<u32x4*>(lds_k + tile_offset(key, 2 * ld_ch + 1)) = hi16;
        convert(st_v[u], lo, hi16);
        *reinterpret_cast<u32x4*>(lds_v + tile_offset(key, 2 * ld_ch)) = lo;
        *reinterpret_cast<u32x4*>(lds_v + tile_offset(key, 2 * ld_ch + 1)) = hi16;
      }
    }
    if constexpr (kTok) {
#pragma unroll
      for (int i = 0; i < kScLoads; ++i)
        if (tid + i * kThreads < kScales) sc[tid + i * kThreads] = st_sc[i];
    }
  };

  // transposed V reads: lane 4i + q of a 16-lane group reads key 4h + i at dims
  // 16 (lane >> 4 & 1) + 4q of the block, and receives V[4h + 0..3][its dim]
  const int vi = (lane & 15) >> 2, vq = lane & 3, vg = (lane >> 4) & 1;

  if (kb0 < k1) load_tile(kb0);
  for (int kb = kb0; kb < k1; kb += NK) {
    __syncthreads();
    store_tile();
    present = present_next;
    __syncthreads();
    if (kb + NK < k1) load_tile(kb + NK);

    const int key0 = kg * TK;  // this wave's keys of the tile
    typedef short i16x8 __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
    auto v_operand = [&](int nb, int half, int b) {
      const int key = key0 + 32 * nb + 16 * half + 4 * h + vi;
      const int chunk = 4 * b + 2 * vg + (vq >> 1), sub = 8 * (vq & 1);
      const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_v + tile_offset(key, chunk) + sub));
      const i16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(lds_v + tile_offset(key + 8, chunk) + sub));
      const i16x8 vt = {lo[0], lo[1], lo[2], lo[3], up[0], up[1], up[2], up[3]};
      return __builtin_bit_cast(Op16<CT>, vt);
    };
    // ---- what this lane's row sees of a tile that is not all prefix: element
    // e of key block nb is key 32 nb + 8 (e >> 2) + 4h + (e & 3) ----
    const bool masked = kb + NK > min(w.prefix, (int64_t)k1) || present != (1u << kSubs) - 1;
    uint32_t seen[NB] = {};
    if (masked) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int kl = key0 + 32 * nb + 8 * (e >> 2) + 4 * h + (e & 3);
          const int64_t j = kb + kl - w.prefix;
          bool vis = kb + kl < k1 && ((present >> (kl >> 4)) & 1);
          if (vis && j >= 0) vis = row_ok && j < a.mask_cols && mask_row[j] != 0;
          seen[nb] |= vis ? 1u << e : 0u;
        }
      }
      if (kb + NK > w.prefix) {
        bool found = false;
        for (int i = tid; i < NK * 16; i += kThreads) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(lds_v + 16 * i);
#pragma unroll
          for (int j = 0; j < 4; ++j) found |= not_finite2<CT>(v[j]);
        }
        if (__syncthreads_or(found)) {
          for (int b = 0; b < 4; ++b) {
            f32x16 marks = f32x16{};
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                Op16<CT> vt = v_operand(nb, half, b), sees;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  const float one = (seen[nb] >> (8 * half + j)) & 1 ? 1.0f : 0.0f;
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
            for (int bb = 0; bb < 4; ++bb)
#pragma unroll
              for (int e = 0; e < 16; ++e)
                if (bb == b && marks[e] > 0.0f) acc[bb][e] += marked_value(marks[e]);
          }
          __syncthreads();
          for (int i = tid; i < NK * 64; i += kThreads) {
            uint32_t* v = reinterpret_cast<uint32_t*>(lds_v) + i;
            constexpr uint32_t e = CT == MKV_DTYPE_BF16 ? 0x7f80u : 0x7c00u;
            uint32_t x = *v;
            if ((x & e) == e) x &= 0xffff0000u;
            if (((x >> 16) & e) == e) x &= 0xffffu;
            *v = x;
          }
          __syncthreads();
        }
      }
    }
    f32x16 s[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      s[nb] = f32x16{};
      const int key = key0 + 32 * nb + c;
#pragma unroll
      for (int st = 0; st < 8; ++st) {
        const u32x4 kw = *reinterpret_cast<const u32x4*>(lds_k + tile_offset(key, 2 * st + h));
        s[nb] = mfma32<CT>(__builtin_bit_cast(Op16<CT>, kw), qop[st], s[nb]);
      }
    }
    const float* ks = sc + (PAIR && hi ? 2 * NK : 0) + key0;
    if constexpr (kTok) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[nb][e] *= ks[32 * nb + 8 * (e >> 2) + 4 * h + (e & 3)];
    }
    if (masked) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[nb][e] = (seen[nb] >> e) & 1 ? s[nb][e] : kNegInf;
    }
    float mx = kNegInf;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[nb][e]);
    mx = fmaxf(mx, other_half(mx));
    mx = fmaxf(mx * score_mul, kNegBig);
    const float m_new = mx > m_run + kRescaleSlack ? mx : m_run;
    // (before the first visible key there is nothing to rescale but marks)
    const float alpha = m_run == kNegBig ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    l_run *= alpha;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f)) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[b][e] *= alpha;
    }
    float p[NB][16];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        p[nb][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][e], score_mul, -m_new));
        l_run += p[nb][e];
        if constexpr (kTok) {
          p[nb][e] *= ks[NK + 32 * nb + 8 * (e >> 2) + 4 * h + (e & 3)];
          if (masked) p[nb][e] = (seen[nb] >> e) & 1 ? p[nb][e] : 0.0f;
        }
      }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        Op16<CT> ph, pl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = p[nb][8 * half + j];
          if constexpr (CT == MKV_DTYPE_BF16) {
            // bf16 holds P to 8 bits: a second term carries the rest, so that
            // a row whose weight sits on few keys is as exact as decode's
            ph[j] = (__bf16)x;
            pl[j] = (__bf16)(x - (float)ph[j]);
          } else {
            ph[j] = (_Float16)x;
          }
        }
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const Op16<CT> vt = v_operand(nb, half, b);
          acc[b] = mfma32<CT>(vt, ph, acc[b]);
          if constexpr (CT == MKV_DTYPE_BF16) acc[b] = mfma32<CT>(vt, pl, acc[b]);
        }
      }
  }

  // ---- the key groups' results, joined in the first one's waves ----
  if constexpr (KG > 1) {
    __syncthreads();
    float* part = reinterpret_cast<float*>(lds);
    if (kg > 0) {
      float* o = part + ((kg - 1) * R + rg) * 64 * 66;
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
      const float* o = part + ((g - 1) * R + rg) * 64 * 66;
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
  }
  const float l = l_run + other_half(l_run);
  if (!row_ok) return;
  if (split) {
    const int64_t at = ((int64_t)blockIdx.x * a.max_splits + blockIdx.z) * a.row_cap + row;
    float* o = a.ws_o + at * kHeadDim;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        st16(o + 32 * b + 2 * e + 4 * h, u32x4{__float_as_uint(acc[b][e]), __float_as_uint(acc[b][e + 1]),
                                              __float_as_uint(acc[b][e + 2]), __float_as_uint(acc[b][e + 3])});
    if (h == 0) {
      a.ws_ml[2 * at] = m_run;
      a.ws_ml[2 * at + 1] = l;
    }
    return;
  }
  float norm = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  if constexpr (KV_DT == MKV_DTYPE_FP8E4M3) norm *= load_uniform_f32(a.v_scale);
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    if (PAIR && (b >> 1) != (int)hi) continue;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const float x[4] = {acc[b][e] * norm, acc[b][e + 1] * norm, acc[b][e + 2] * norm, acc[b][e + 3] * norm};
      store4(a.out, a.q_dtype, q_off + 32 * (PAIR ? b & 1 : b) + 2 * e + 4 * h, x);
    }
  }
}

// Rows of sequences in several splits: a wave a row, two dims a lane.
constexpr int kJoinWaves = 4;
template <int UNIT, bool FP8, bool PAIR>
__global__ __launch_bounds__(64 * kJoinWaves) void tree_join_kernel(TreeArgs a) {
  const Work w = find_work(a, blockIdx.x);
  const int len = split_keys<UNIT>(a);
  const int n = (w.ctx + len - 1) / len;
  if (n <= 1) return;
  const int lane = threadIdx.x & 63;
  const int row = blockIdx.y * kJoinWaves + uniform(threadIdx.x >> 6);
  if (row >= w.rows) return;
  const int64_t at = (int64_t)blockIdx.x * a.max_splits * a.row_cap + row;
  float m = kNegBig, l = 0.0f, x = 0.0f, y = 0.0f;
  for (int z = 0; z < n; ++z) {
    const int64_t i = at + (int64_t)z * a.row_cap;
    const float mz = a.ws_ml[2 * i], lz = a.ws_ml[2 * i + 1];
    const float* o = a.ws_o + i * kHeadDim + 2 * lane;
    const float m_new = fmaxf(m, mz);
    const float fa = __builtin_amdgcn_exp2f(m - m_new), fb = __builtin_amdgcn_exp2f(mz - m_new);
    m = m_new;
    l = l * fa + lz * fb;
    x = x * fa + o[0] * fb;
    y = y * fa + o[1] * fb;
  }
  float norm = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
  if constexpr (FP8) norm *= load_uniform_f32(a.v_scale);
  bool hi = false;
  int64_t off = row_offset<PAIR>(a, w, row, hi);
  int d = 2 * lane;
  if constexpr (PAIR) {
    if ((d >= 64) != hi) return;
    d &= 63;
  }
  off += d;
  if (a.q_dtype == MKV_DTYPE_F32) {
    reinterpret_cast<float*>(a.out)[off] = x * norm;
    reinterpret_cast<float*>(a.out)[off + 1] = y * norm;
  } else {
    const uint32_t b0 = a.q_dtype == MKV_DTYPE_BF16 ? f32_to_bf16_bits(x * norm) : f32_to_f16_bits(x * norm);
    const uint32_t b1 = a.q_dtype == MKV_DTYPE_BF16 ? f32_to_bf16_bits(y * norm) : f32_to_f16_bits(y * norm);
    *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.out) + off) = b0 | b1 << 16;
  }
}

// fp32 caches: products and sums in fp32 on the 32x32x2 fp32 MFMA, one row
// group of 32 rows and four key groups.  Lane (c, h) supplies K[key c][64h + st]
// and q[row c][64h + st] at step st, and for O^T its own keys' P again.
template <bool PAIR>
__global__ __launch_bounds__(256) void tree_attention_f32_kernel(TreeArgs a) {
  constexpr int KG = 4, NK = 128, kRow = 528;  // 512-byte rows, 16 bytes apart in the banks
  __shared__ __align__(16) char lds[NK * kRow];
  const int tid = threadIdx.x, lane = tid & 63, kg = uniform(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const Work w = find_work(a, blockIdx.x);
  const int len = a.max_splits > 1 ? split_keys<NK>(a) : 0x7fffffff / NK * NK;
  const int64_t k0 = (int64_t)blockIdx.z * len;
  if (blockIdx.y == 0 && blockIdx.z == 0 && w.kvh == 0) zero_rows_past(a, w);
  if ((blockIdx.z > 0 && k0 >= w.ctx) || (int)blockIdx.y * 32 >= w.rows) return;
  const int kb0 = (int)k0, k1 = (int)min(k0 + len, (int64_t)w.ctx);
  const bool split = w.ctx > len;
  const int row = blockIdx.y * 32 + c;
  const bool row_ok = row < w.rows;
  bool hi = false;
  const int64_t q_off = row_offset<PAIR>(a, w, row_ok ? row : 0, hi);
  const float score_mul = a.sm_scale * kLog2e;
  float qv[64];
#pragma unroll
  for (int i = 0; i < 64; i += 4) {
    u32x4 v{0, 0, 0, 0};
    if (row_ok && (!PAIR || h == (int)hi)) v = ld16(reinterpret_cast<const float*>(a.q) + q_off + (PAIR ? 0 : 64 * h) + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) qv[i + j] = __uint_as_float(v[j]);
  }
  const int64_t row_elems = (int64_t)a.num_kv_heads * kHeadDim;
  const uint8_t* mask_row = a.mask + (w.q0 + (row_ok ? row / a.group : 0)) * a.mask_stride;
  f32x16 acc[4];
#pragma unroll
  for (int b = 0; b < 4; ++b) acc[b] = f32x16{};
  float m_run = kNegBig, l_run = 0.0f;
  for (int kb = kb0; kb < k1; kb += NK) {
    uint32_t present = 0;
    int64_t slot[NK / 16];
#pragma unroll
    for (int u = 0; u < NK / 16; ++u) {
      const int t = kb + 16 * u;
      const int64_t phys = t < k1 ? a.idx.physical_block(w.seq, t >> a.idx.bs_log2) : -1;
      present |= phys >= 0 ? 1u << u : 0u;
      slot[u] = phys < 0 ? -1 : (phys << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1));
    }
    auto stage = [&](const char* pool) {
#pragma unroll
      for (int u = 0; u < NK / 8; ++u) {  // 8 keys of 32 chunks a load
        const int key = 8 * u + (tid >> 5);
        u32x4 v{0, 0, 0, 0};
        if (slot[u >> 1] >= 0 && kb + key < k1)
          v = ld16(pool + ((slot[u >> 1] + (key & 15)) * row_elems + w.kvh * kHeadDim + 4 * (tid & 31)) * 4);
        *reinterpret_cast<u32x4*>(lds + key * kRow + 16 * (tid & 31)) = v;
      }
    };
    __syncthreads();
    stage(a.k);
    __syncthreads();
    f32x16 s = f32x16{};
    const int key0 = 32 * kg;
#pragma unroll
    for (int i = 0; i < 64; i += 4) {
      const u32x4 kw = *reinterpret_cast<const u32x4*>(lds + (key0 + c) * kRow + 256 * h + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) s = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kw[j]), qv[i + j], s, 0, 0, 0);
    }
    __syncthreads();
    stage(a.v);
    __syncthreads();
    float mx = kNegInf;
    uint32_t seen = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const int kl = key0 + 8 * (e >> 2) + 4 * h + (e & 3);
      const int64_t j = kb + kl - w.prefix;
      bool vis = kb + kl < k1 && ((present >> (kl >> 4)) & 1);
      if (vis && j >= 0) vis = row_ok && j < a.mask_cols && mask_row[j] != 0;
      s[e] = vis ? s[e] * score_mul : kNegInf;
      seen |= vis ? 1u << e : 0u;
      mx = fmaxf(mx, s[e]);
    }
    mx = fmaxf(fmaxf(mx, other_half(mx)), kNegBig);
    const float m_new = fmaxf(mx, m_run);
    const float alpha = m_run == kNegBig ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
    m_run = m_new;
    l_run *= alpha;
#pragma unroll
    for (int b = 0; b < 4; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[b][e] *= alpha;
    float p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = __builtin_amdgcn_exp2f(s[e] - m_new);
      l_run += p[e];
    }
    auto v_at = [&](int e, int b) {
      return *reinterpret_cast<const float*>(lds + (key0 + 8 * (e >> 2) + 4 * h + (e & 3)) * kRow + 4 * (32 * b + c));
    };
    bool found = false;
    if (kb + key0 + 32 > w.prefix) {
      for (int i = 0; i < 16; ++i) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(lds + (key0 + 2 * i + h) * kRow + 16 * c);
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= not_finite(__uint_as_float(v[j]));
      }
    }
    const bool dirty = __builtin_amdgcn_ballot_w64(found) != 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        float v = v_at(e, b);
        if (dirty && not_finite(v)) v = 0.0f;
        acc[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, p[e], acc[b], 0, 0, 0);
      }
    }
    if (dirty) {
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        f32x16 marks = f32x16{};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          marks = __builtin_amdgcn_mfma_f32_32x32x2f32(mark_of(v_at(e, b)), (seen >> e) & 1 ? 1.0f : 0.0f, marks, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (marks[e] > 0.0f) acc[b][e] += marked_value(marks[e]);
      }
    }
  }
  __syncthreads();
  float* part = reinterpret_cast<float*>(lds);
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
  const int64_t at = ((int64_t)blockIdx.x * a.max_splits + blockIdx.z) * a.row_cap + row;
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
  int target;
  int min_split;
  int max_splits;
};

Plan make_plan(int num_seqs, int64_t total_q, int kernel_kv_heads, int kernel_group, int mask_cols, int64_t capacity,
               bool f32) {
  Plan p;
  const int64_t toks = mask_cols < total_q ? mask_cols : total_q;
  const int64_t rows = toks * kernel_group;
  p.row_groups = f32 || rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
  p.row_blocks = (int)((rows + 32 * p.row_groups - 1) / (32 * p.row_groups));
  if (p.row_blocks < 1) p.row_blocks = 1;
  p.row_cap = p.row_blocks * 32 * p.row_groups;
  p.unit = p.row_groups == 1 ? 128 : 64;
  p.target = p.row_groups == 8 ? 512 : 1024;
  p.min_split = 128;
  const int64_t items = (int64_t)num_seqs * kernel_kv_heads * p.row_blocks;
  // twice the even share: the longest sequences of a ragged batch
  int64_t s = items > 0 ? 2 * (p.target + items - 1) / items : 1;
  const int64_t most = (capacity + p.min_split - 1) / p.min_split;
  if (items >= 2 * p.target) s = 1;
  if (s > most) s = most;
  p.max_splits = (int)(s < 1 ? 1 : s);
  return p;
}

size_t workspace_of(const Plan& p, int64_t items) {
  return p.max_splits > 1 ? (size_t)items * p.max_splits * p.row_cap * (kHeadDim + 2) * sizeof(float) : 0;
}

template <int KV_DT, bool PAIR>
int launch_tree(const TreeArgs& a, const Plan& p, hipStream_t s) {
  const dim3 grid((unsigned)(a.num_seqs * a.num_kv_heads), (unsigned)p.row_blocks, (unsigned)p.max_splits);
  if constexpr (KV_DT == MKV_DTYPE_F32) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_f32_kernel<PAIR>), grid, dim3(256), 0, s, a);
  } else {
    switch (p.row_groups) {
      case 1: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 1, 4, PAIR>), grid, dim3(256), 0, s, a); break;
      case 2: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 2, 2, PAIR>), grid, dim3(256), 0, s, a); break;
      case 4: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 4, 1, PAIR>), grid, dim3(256), 0, s, a); break;
      default: hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_attention_kernel<KV_DT, 8, 1, PAIR>), grid, dim3(512), 0, s, a); break;
    }
  }
  if (hipError_t e = hipGetLastError()) return (int)e;
  if (p.max_splits > 1) {
    constexpr bool kFp8 = KV_DT == MKV_DTYPE_FP8E4M3;
    const dim3 jgrid(grid.x, (unsigned)((p.row_cap + kJoinWaves - 1) / kJoinWaves));
    if (p.unit == 128)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_join_kernel<128, kFp8, PAIR>), jgrid, dim3(64 * kJoinWaves), 0, s, a);
    else
      hipLaunchKernelGGL(HIP_KERNEL_NAME(tree_join_kernel<64, kFp8, PAIR>), jgrid, dim3(64 * kJoinWaves), 0, s, a);
    return (int)hipGetLastError();
  }
  return MKV_OK;
}

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
  return MKV_OK;
}

Plan plan_of(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
             int max_blocks, int mask_cols, int kv_dtype, int64_t& items) {
  const int pair = head_dim == 64 ? 2 : 1;
  const int kv = num_kv_heads / pair, g = num_heads / num_kv_heads * pair;
  items = (int64_t)num_seqs * kv;
  return make_plan(num_seqs, total_q, kv, g, mask_cols, (int64_t)max_blocks * block_size, kv_dtype == MKV_DTYPE_F32);
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_paged_tree_workspace_size(int num_seqs, int64_t total_q, int num_heads, int num_kv_heads,
                                                int head_dim, int block_size, int max_blocks, int mask_cols,
                                                int kv_dtype) {
  if (check_tree(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols)) return 0;
  int64_t items;
  const Plan p = plan_of(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols, kv_dtype, items);
  return workspace_of(p, items);
}

extern "C" int mkv_paged_tree(void* out, const void* q, int q_dtype, const void* k_cache, const void* v_cache,
                              int kv_dtype, int64_t num_blocks, const float* k_scale, const float* v_scale,
                              int kv_scale_mode, const int32_t* block_tables, int64_t bt_stride, int max_blocks,
                              const void* context_lens, int context_lens_dtype, const int32_t* cu_seqlens_q,
                              const uint8_t* tree_mask, int64_t mask_stride, int mask_cols, int num_seqs,
                              int64_t total_q, int num_heads, int num_kv_heads, int head_dim, int block_size,
                              float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_tree(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols)) return st;
  if (num_blocks < 0 || num_blocks > 0x7fffffff) return MKV_ERR_BAD_SHAPE;
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
  int64_t items;
  const Plan p = plan_of(num_seqs, total_q, num_heads, num_kv_heads, head_dim, block_size, max_blocks, mask_cols, kv_dtype, items);
  if (p.row_blocks > 65535 || p.max_splits > 65535) return MKV_ERR_BAD_SHAPE;
  if (workspace_of(p, items) > workspace_bytes || (p.max_splits > 1 && !workspace)) return MKV_ERR_WORKSPACE_TOO_SMALL;
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
  a.max_splits = p.max_splits;
  a.target = p.target;
  a.min_split = p.min_split;
  a.row_blocks = p.row_blocks;
  a.row_cap = p.row_cap;
  a.ws_o = reinterpret_cast<float*>(workspace);
  a.ws_ml = a.ws_o + (size_t)items * p.max_splits * p.row_cap * kHeadDim;
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
