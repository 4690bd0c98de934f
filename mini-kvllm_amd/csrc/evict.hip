// Eviction from the paged cache by accumulated attention weight: every layer and KV
// head keeps `budget` tokens of a sequence longer than that, the first `sinks`, the
// last `recent` and, between them, those of the largest weight (the earlier of equal
// ones), moved to the sequence's front in their order.
//
// evict_select_kernel finds the kept tokens' slots, a workgroup a (layer, sequence,
// KV head): the weight that the last kept one has by a radix search over the weights'
// order (11, 11 and 10 bits, histograms in LDS), then their places by ballots.  Whole
// numbers throughout, so the result is one only.
// evict_move_kernel moves the rows, HBM bound: each kept row is read and written once.
// A kept token's source never lies ahead of its destination, so a workgroup that takes
// one head's rows in order, each batch of rows in registers before any of it is
// written, moves them in place: a later source is behind everything written so far.
// 60 sequences of 300-800 tokens cut to 256 in 8 layers: 32 us and 208 (where nearly
// every row moves, 1 GB, 4.8 TB/s); two of 49k and 66k cut to 8192 in 4 layers, scales
// beside them: keys 11 us, selection 61, rows 137.
#include <type_traits>

#include "mkv_device.hpp"

namespace mkv {
namespace {

// (lambdas whose arrays have to stay in registers)
#define MKV_INLINE __attribute__((always_inline))

constexpr int kMaxTensors = 128;  // a launch's tensors, their addresses in the kernel arguments
constexpr int kBins = 2048;
// Keys of long tables in the workspace: those of as many layers (of one layer's sequences,
// if need be) as this many bytes hold, of one sequence at least.  The table's width, which
// may be far past the lengths, sets their size: 28 layers of 60 sequences and 8 heads under
// tables of 131,072 tokens would be 6.6 GiB together (300-800 tokens cut to 256: 1.46 ms
// with all of that, 1.63 a layer at a time; under tables of 1024 tokens 0.83).
constexpr size_t kMaxKeyBytes = (size_t)256 << 20;

struct EvictArgs {
  PagedIndex idx;
  const void* lens;
  int lens_i64;
  int batch, heads;
  int budget, sinks, recent;
  int64_t* new_lens;
  int32_t* slots;   // workspace: (layers, batch, heads, budget), the kept tokens' slots in order
  uint32_t* keys;   // workspace: (layers, sequences, heads, key_stride) of a launch, for long tables
  int64_t key_stride;
};
struct Weights {
  const float* base[kMaxTensors];
};
struct Moved {
  char* base[kMaxTensors];
  int32_t head_bytes[kMaxTensors];
  int32_t layer[kMaxTensors];
};

// Unsigned order of the weights: NaN above +inf, the two zeros alike, never 0.
MKV_DEV uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  const uint32_t o = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : o;
}

// Tokens of a sequence that its table holds.
MKV_DEV int length_of(const EvictArgs& a, int b, int64_t& len) {
  len = max(load_index(a.lens, b, a.lens_i64), (int64_t)0);
  return (int)min(len, (int64_t)a.idx.max_blocks << a.idx.bs_log2);
}
// Slot of token t, -1 outside the pool.
MKV_DEV int slot_of(const EvictArgs& a, int b, int t) {
  const int32_t p = a.idx.block_tables[(int64_t)b * a.idx.bt_stride + (t >> a.idx.bs_log2)];
  return p >= 0 && p < a.idx.num_blocks ? (p << a.idx.bs_log2) + (t & ((1 << a.idx.bs_log2) - 1)) : -1;
}
// A launch's layers from `layer` on and sequences from `seq` on.
struct Slice {
  int layer, layers, seq, seqs;
};
// Workgroups of one (layer, sequence) lie 8 apart, on one XCD: its heads share the
// weights' cache lines.  (layer and b: within the slice)
MKV_DEV bool place_of(const EvictArgs& a, const Slice& s, int i, int& layer, int& b, int& h) {
  const int group = i / (8 * a.heads), in = i % (8 * a.heads);
  const int pair = group * 8 + in % 8;
  h = in / 8;
  layer = pair / s.seqs;
  b = pair % s.seqs;
  return layer < s.layers;
}

// The weights' keys of long tables, transposed to a row a head: four heads a load
// where their number allows it.
__global__ __launch_bounds__(256) void evict_keys_kernel(EvictArgs a, Weights w, Slice of) {
  const int b = of.seq + blockIdx.y, layer = blockIdx.z;
  int64_t len;
  const int n = length_of(a, b, len);
  if (n <= a.budget) return;
  uint32_t* const out = a.keys + ((int64_t)layer * of.seqs + blockIdx.y) * a.heads * a.key_stride;
  const bool wide = a.heads % 4 == 0 && (reinterpret_cast<uintptr_t>(w.base[layer]) & 15) == 0;
  for (int t = blockIdx.x * 256 + threadIdx.x; t < n; t += gridDim.x * 256) {
    const int s = slot_of(a, b, t);
    const float* row = w.base[layer] + (int64_t)max(s, 0) * a.heads;
    if (wide) {
      for (int h = 0; h < a.heads; h += 4) {
        const u32x4 v = ld16(row + h);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[(h + e) * a.key_stride + t] = s >= 0 ? order_of(__uint_as_float(v[e])) : 0u;
      }
    } else {
      for (int h = 0; h < a.heads; ++h) out[h * a.key_stride + t] = s >= 0 ? order_of(row[h]) : 0u;
    }
  }
}

// The keys of a (layer, sequence, KV head), four tokens a lane at a time: each wave has
// a run of consecutive tokens, kHeld of its vectors in registers, the rest (of rows
// longer than they take) in memory.
template <int T, int HELD>
struct Keys {
  static constexpr int kWaves = T / 64;
  u32x4 held[HELD];
  const u32x4* more;  // the row in memory
  int first, num;     // the wave's first token, and its vectors
  MKV_DEV int token(int j) const { return first + 256 * j + 4 * (threadIdx.x & 63); }
  MKV_DEV Keys(int n, int wave) {
    num = (n + 256 * kWaves - 1) / (256 * kWaves);
    first = wave * num * 256;
  }
  // f(vector j's keys, its first token)
  template <class F>
  MKV_DEV void each(int n, F f) const {
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (j < num && first + 256 * j < n) f(held[j], token(j));
    // (lanes behind the row's end: its last vector, masked)
    for (int j = HELD; j < num && first + 256 * j < n; ++j) f(more[min(token(j), n - 1) / 4], token(j));
  }
};

// KEYS: from the transposed keys; else from the weights themselves (up to HELD vectors
// a wave: 256 T / 64 HELD tokens).
// COPIES of the histograms, lanes by turns, lessen what meets at one address: long rows
// 74 us with one and a wave's common key counted ahead, 61 with four and plain atomics
// (1, 8, 16: 64, 63, 68); short ones 35 and, with one and plain atomics, 32 (2: 34).
// Weights that are all alike, as before the first step, meet at one address whatever the
// copies: 87 for the 61, in a call that then moves no row.
template <int T, int HELD, bool KEYS, int COPIES>
__global__ __launch_bounds__(T) void evict_select_kernel(EvictArgs a, Weights w, Slice of) {
  constexpr int kWaves = T / 64;
  __shared__ __align__(16) int hist[kBins * COPIES];
  __shared__ int scan[kWaves], found[2], part_kept[kWaves], part_equal[kWaves];
  int layer, in, h;
  if (!place_of(a, of, blockIdx.x, layer, in, h)) return;
  const int b = of.seq + in;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  int64_t len;
  const int n = length_of(a, b, len);
  if (of.layer + layer == 0 && h == 0 && tid == 0) a.new_lens[b] = min(len, (int64_t)a.budget);
  if (n <= a.budget) return;
  const int64_t at = ((int64_t)(of.layer + layer) * a.batch + b) * a.heads + h;
  Keys<T, HELD> keys(n, wave);
  if constexpr (KEYS) {
    // (rows are a multiple of four long; what lies behind the last token is masked)
    keys.more = reinterpret_cast<const u32x4*>(a.keys + (((int64_t)layer * of.seqs + in) * a.heads + h) * a.key_stride);
#pragma unroll
    for (int j = 0; j < HELD; ++j) keys.held[j] = j < keys.num && keys.token(j) < n ? keys.more[keys.token(j) / 4] : u32x4{0, 0, 0, 0};
  } else {
    keys.more = nullptr;
    int slot[HELD];  // (four tokens lie in one block)
#pragma unroll
    for (int j = 0; j < HELD; ++j)
      if (j < keys.num) slot[j] = a.idx.block_tables[(int64_t)b * a.idx.bt_stride + (min(keys.token(j), n - 1) >> a.idx.bs_log2)];
    float x[HELD][4];
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (j >= keys.num) continue;
      const bool there = slot[j] >= 0 && slot[j] < a.idx.num_blocks;
      const int64_t s = ((int64_t)(there ? slot[j] : 0) << a.idx.bs_log2) + (keys.token(j) & ((1 << a.idx.bs_log2) - 1));
      if (!there) slot[j] = -1;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[j][e] = w.base[layer][(s + e) * a.heads + h];
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (j >= keys.num) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) keys.held[j][e] = slot[j] >= 0 ? order_of(x[j][e]) : 0u;
    }
  }
  const int first = a.sinks, last = n - a.recent;  // the middle: [first, last)
  int want = a.budget - a.sinks - a.recent;        // of it are kept
  uint32_t least = 0xffffffffu;                    // the smallest key kept; `want` of those equal to it
  if (want > 0) {
    least = 0;
    constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      constexpr int kNone = 32;
      const int shift = kShift[pass], bins = 1 << kBits[pass], upper = pass == 0 ? kNone : kShift[pass > 0 ? pass - 1 : 0];
      for (int i = tid; i < kBins * COPIES; i += T) hist[i] = 0;
      __syncthreads();
      const uint32_t above = pass == 0 ? 0u : least >> upper;
      keys.each(n, [&](const u32x4& v, int t) MKV_INLINE {
        // (most vectors lie in the middle whole)
        const int t0 = uniform(t - 4 * lane);
        const bool whole = t0 >= first && t0 + 256 <= last;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool in = (whole || (t + e >= first && t + e < last)) && (pass == 0 || v[e] >> upper == above);
          const int d = (int)(v[e] >> shift) & (bins - 1);
          if (in) atomicAdd(&hist[d * COPIES + lane % COPIES], 1);
        }
      });
      __syncthreads();
      // the bin in which the want-th largest lies; thread tid has bins from the top
      constexpr int kPer = kBins / T;
      int c[kPer], own = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        c[j] = 0;
#pragma unroll
        for (int i = 0; i < COPIES; ++i) c[j] += hist[(kBins - 1 - (tid * kPer + j)) * COPIES + i];
        own += c[j];
      }
      int upto = own;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 63) scan[wave] = upto;
      __syncthreads();
      int before = upto - own;
      for (int v = 0; v < wave; ++v) before += scan[v];
      if (before < want && want <= before + own) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
          if (before < want && want <= before + c[j]) {
            found[0] = kBins - 1 - (tid * kPer + j);
            found[1] = before;
          }
          before += c[j];
        }
      }
      __syncthreads();
      least |= (uint32_t)found[0] << shift;
      want -= found[1];
    }
  }
  // ---- the kept tokens' places, in order ----
  int kept = 0, equal = 0;  // of the lane
  keys.each(n, [&](const u32x4& v, int t) MKV_INLINE {
    const int t0 = uniform(t - 4 * lane);
    if (t0 >= first && t0 + 256 <= last) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kept += v[e] > least;
        equal += v[e] == least;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = t + e < n, mid = in && t + e >= first && t + e < last;
        kept += (in && !mid) || (mid && v[e] > least);
        equal += mid && v[e] == least;
      }
    }
  });
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    kept += __shfl_xor(kept, o);
    equal += __shfl_xor(equal, o);
  }
  if (lane == 0) {
    part_kept[wave] = kept;
    part_equal[wave] = equal;
  }
  __syncthreads();
  int to = 0, tied = 0;  // kept, and equal ones, ahead of this wave's run
  for (int v = 0; v < wave; ++v) {
    to += part_kept[v] + min(max(want - tied, 0), part_equal[v]);
    tied += part_equal[v];
  }
  int32_t* const out = a.slots + at * a.budget;
  const uint64_t below = (1ull << lane) - 1;
  keys.each(n, [&](const u32x4& v, int t) MKV_INLINE {
    // equal tokens ahead of the lane's, then the kept ones
    bool eq[4], keep[4];
    int eq_ahead = tied, eq_all = 0, eq_own = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      eq[e] = t + e < n && t + e >= first && t + e < last && v[e] == least;
      const uint64_t ball = __builtin_amdgcn_ballot_w64(eq[e]);
      eq_ahead += __popcll(ball & below);
      eq_all += __popcll(ball);
    }
    int place = to, all = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool in = t + e < n, mid = in && t + e >= first && t + e < last;
      keep[e] = (in && !mid) || (mid && v[e] > least) || (eq[e] && eq_ahead + eq_own < want);
      eq_own += eq[e];
      const uint64_t ball = __builtin_amdgcn_ballot_w64(keep[e]);
      place += __popcll(ball & below);
      all += __popcll(ball);
    }
    const int s = slot_of(a, b, min(t, n - 1));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (keep[e] && place < a.budget) out[place] = s >= 0 ? s + e : -1;
      place += keep[e];
    }
    to += all;
    tied += eq_all;
  });
}

// Rows of one head (X a 16- or 4-byte item, `units` of them a row), or of all heads
// together (heads_together: 4 bytes a head).  The next batch's slots are on their way
// while this one's rows are.
constexpr int kItems = 8;  // a thread's, in registers
constexpr int kMaxHeadBytes = 64 * kItems * 4;  // (a row of the smallest workgroup's 4-byte items)
template <typename X, int T>
MKV_DEV void move_rows(const EvictArgs& a, char* base, int64_t token_bytes, int units, int b, const int32_t* slots,
                       int64_t head_stride, bool heads_together) {
  const int mask = (1 << a.idx.bs_log2) - 1;
  const int32_t* bt = a.idx.block_tables + (int64_t)b * a.idx.bt_stride;
  const int per = max(T * kItems / units, 1);  // rows of a batch
  int row[kItems], col[kItems], from[kItems], to[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) {
    const int item = i * T + (int)threadIdx.x;
    row[i] = item / units;
    col[i] = item - row[i] * units;
  }
  auto look_up = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = min(j0 + row[i], a.budget - 1);
      from[i] = slots[(heads_together ? col[i] * head_stride : 0) + j];
      to[i] = bt[j >> a.idx.bs_log2];
    }
  };
  look_up(0);
  for (int j0 = 0; j0 < a.budget; j0 += per) {
    X v[kItems];
    int d[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int j = j0 + row[i];
      const bool ok = row[i] < per && j < a.budget && from[i] >= 0 && to[i] >= 0 && to[i] < a.idx.num_blocks;
      d[i] = ok ? (to[i] << a.idx.bs_log2) + (j & mask) : -1;
      if (d[i] == from[i]) d[i] = -1;
      if (d[i] >= 0) v[i] = *reinterpret_cast<const X*>(base + from[i] * token_bytes + col[i] * (int)sizeof(X));
    }
    if (j0 + per < a.budget) look_up(j0 + per);
    // every row of the batch has been read before any is written
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (T > 64) __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (d[i] >= 0) *reinterpret_cast<X*>(base + d[i] * token_bytes + col[i] * (int)sizeof(X)) = v[i];
  }
}

template <int T>
__global__ __launch_bounds__(T) void evict_move_kernel(EvictArgs a, Moved m, int slices) {
  // (the last tensors, of 4 bytes a head, first: theirs are the longest turns)
  const int h = blockIdx.x / slices, slice = blockIdx.x % slices, b = blockIdx.y, t = gridDim.z - 1 - blockIdx.z;
  int64_t len;
  if (length_of(a, b, len) <= a.budget) return;
  const int64_t bytes = m.head_bytes[t], token = bytes * a.heads;
  const int64_t lists = ((int64_t)m.layer[t] * a.batch + b) * a.heads;
  const int32_t* slots = a.slots + (lists + h) * a.budget;
  char* const base = m.base[t];
  if (bytes == 4) {
    // (few sequences: two heads a workgroup)
    const int share = T > 256 ? 2 : a.heads;
    if (h % share == 0 && slice == 0)
      move_rows<uint32_t, T>(a, base + 4 * h, token, min(share, a.heads - h), b, slots, a.budget, true);
  } else if (bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {
    // a slice: an even share of the row's 16-byte items
    const int units = (int)(bytes / 16), share = (units + slices - 1) / slices, c0 = slice * share;
    if (c0 < units)
      move_rows<u32x4, T>(a, base + h * bytes + 16 * c0, token, min(share, units - c0), b, slots, 0, false);
  } else if (slice == 0) {
    move_rows<uint32_t, T>(a, base + h * bytes, token, (int)(bytes / 4), b, slots, 0, false);
  }
}

int log2_exact(int64_t v) {
  if (v <= 0 || (v & (v - 1))) return -1;
  int l = 0;
  while (((int64_t)1 << l) < v) ++l;
  return l;
}

// Of a table: a grid's stride past them, 2^18 (evict_keys_kernel), stays within 32 bits.
constexpr int64_t kMaxTokens = 0x7ff00000;
int64_t capacity_of(int max_blocks, int block_size) { return (int64_t)max_blocks * block_size; }

// The forms of the selection by the table's width: tokens that a workgroup of 256
// threads holds (8 vectors a wave); wider ones go by transposed keys.
constexpr int kHeldVectors = 8;
constexpr int kHeldTokens = 256 * 4 * kHeldVectors;
bool needs_keys(int64_t cap) { return cap > kHeldTokens; }
int64_t key_stride_of(int64_t cap) { return (cap + 3) / 4 * 4; }
// The layers and sequences of a selection's launch, at most: even shares.
struct Share {
  int layers, seqs;
};
Share share_of(int num_layers, int batch, int heads, int64_t cap) {
  Share s{num_layers < kMaxTensors ? num_layers : kMaxTensors, batch};
  if (needs_keys(cap)) {
    const size_t one = (size_t)heads * key_stride_of(cap) * 4, fit = kMaxKeyBytes > one ? kMaxKeyBytes / one : 1;
    const size_t layers = fit / batch < (size_t)s.layers ? fit / batch : s.layers;
    if (layers) {
      const int turns = (int)((num_layers + layers - 1) / layers);
      s.layers = (num_layers + turns - 1) / turns;
    } else {
      const int turns = (int)((batch + fit - 1) / fit);
      s = Share{1, (batch + turns - 1) / turns};
    }
  }
  return s;
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_evict_tokens_workspace_size(int num_layers, int batch, int num_kv_heads, int block_size,
                                                  int max_blocks, int budget) {
  if (num_layers <= 0 || batch <= 0 || num_kv_heads <= 0 || max_blocks <= 0 || block_size <= 0 || budget <= 0) return 0;
  const size_t lists = (size_t)num_layers * batch * num_kv_heads, cap = (size_t)capacity_of(max_blocks, block_size);
  const Share s = share_of(num_layers, batch, num_kv_heads, cap);
  return ((lists * budget + 3) / 4 * 4 + (needs_keys(cap) ? (size_t)s.layers * s.seqs * num_kv_heads * key_stride_of(cap) : 0)) * 4;
}

extern "C" int mkv_evict_tokens(const void* const* tensors, const int64_t* head_bytes, const int* layer_of,
                                int num_tensors, const void* const* weights, int num_layers, int64_t num_pages,
                                int block_size, int num_kv_heads, const int32_t* block_tables, int64_t bt_stride,
                                int max_blocks, const void* seq_lens, int seq_lens_dtype, int batch, int budget,
                                int sinks, int recent, int64_t* new_lens, void* workspace, size_t workspace_bytes,
                                void* stream) {
  if (num_tensors < 0 || num_layers < 0 || num_kv_heads <= 0 || num_kv_heads > 1024 || batch < 0 || batch > 65535 ||
      num_pages < 0 || max_blocks < 0 || budget <= 0 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > budget)
    return MKV_ERR_BAD_SHAPE;
  const int bs_log2 = log2_exact(block_size);
  if (bs_log2 < 2) return MKV_ERR_BAD_BLOCK_SIZE;
  if (num_pages > (0x7fffffff >> bs_log2) || capacity_of(max_blocks, block_size) > kMaxTokens) return MKV_ERR_BAD_SHAPE;
  if (seq_lens_dtype != MKV_INDEX_I32 && seq_lens_dtype != MKV_INDEX_I64) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (batch == 0 || num_layers == 0) return MKV_OK;
  if ((num_tensors && (!tensors || !head_bytes || !layer_of)) || !weights || !block_tables || !seq_lens || !new_lens ||
      !workspace)
    return MKV_ERR_NULL_POINTER;
  if (bt_stride < max_blocks) return MKV_ERR_BAD_STRIDE;
  for (int t = 0; t < num_tensors; ++t) {
    if (!tensors[t]) return MKV_ERR_NULL_POINTER;
    if (head_bytes[t] <= 0 || head_bytes[t] % 4 || head_bytes[t] > kMaxHeadBytes || layer_of[t] < 0 || layer_of[t] >= num_layers)
      return MKV_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(tensors[t]) & 3) return MKV_ERR_MISALIGNED;
  }
  for (int l = 0; l < num_layers; ++l) {
    if (!weights[l]) return MKV_ERR_NULL_POINTER;
    if (reinterpret_cast<uintptr_t>(weights[l]) & 3) return MKV_ERR_MISALIGNED;
  }
  if ((reinterpret_cast<uintptr_t>(workspace) & 15) != 0) return MKV_ERR_MISALIGNED;
  const int64_t cap = capacity_of(max_blocks, block_size);
  const int64_t pairs = ((int64_t)(num_layers < kMaxTensors ? num_layers : kMaxTensors) * batch + 7) / 8 * 8;
  if (pairs * num_kv_heads > 0x3fffff || (int64_t)num_layers * batch * num_kv_heads > 0x7fffffff) return MKV_ERR_BAD_SHAPE;
  if (workspace_bytes < mkv_evict_tokens_workspace_size(num_layers, batch, num_kv_heads, block_size, max_blocks, budget))
    return MKV_ERR_WORKSPACE_TOO_SMALL;
  // (the move reads the old lengths behind the selection's new ones)
  const char *const old_at = static_cast<const char*>(seq_lens), *const new_at = reinterpret_cast<const char*>(new_lens);
  if (old_at < new_at + 8 * (int64_t)batch && new_at < old_at + (seq_lens_dtype == MKV_INDEX_I64 ? 8 : 4) * (int64_t)batch)
    return MKV_ERR_BAD_SHAPE;
  EvictArgs a;
  a.idx = PagedIndex{block_tables, bt_stride, max_blocks, num_pages, bs_log2, 0};
  a.lens = seq_lens;
  a.lens_i64 = seq_lens_dtype == MKV_INDEX_I64;
  a.batch = batch;
  a.heads = num_kv_heads;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.new_lens = new_lens;
  a.slots = reinterpret_cast<int32_t*>(workspace);
  a.keys = reinterpret_cast<uint32_t*>(a.slots + ((size_t)num_layers * batch * num_kv_heads * budget + 3) / 4 * 4);
  a.key_stride = key_stride_of(cap);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  const Share share = share_of(num_layers, batch, num_kv_heads, cap);
  for (int l0 = 0; l0 < num_layers; l0 += share.layers) {
    const int layers = num_layers - l0 < share.layers ? num_layers - l0 : share.layers;
    Weights w;
    for (int l = 0; l < layers; ++l) w.base[l] = reinterpret_cast<const float*>(weights[l0 + l]);
    for (int b0 = 0; b0 < batch; b0 += share.seqs) {
      const Slice of{l0, layers, b0, batch - b0 < share.seqs ? batch - b0 : share.seqs};
      const dim3 grid((unsigned)(((int64_t)layers * of.seqs + 7) / 8 * 8 * num_kv_heads));
      if (needs_keys(cap)) {
        const unsigned x = (unsigned)((cap + 255) / 256 < 1024 ? (cap + 255) / 256 : 1024);
        hipLaunchKernelGGL(evict_keys_kernel, dim3(x, (unsigned)of.seqs, (unsigned)layers), dim3(256), 0, s, a, w, of);
        if (hipError_t e = hipGetLastError()) return (int)e;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(evict_select_kernel<1024, 16, true, 4>), grid, dim3(1024), 0, s, a, w, of);
      } else {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(evict_select_kernel<256, kHeldVectors, false, 1>), grid, dim3(256), 0, s, a, w, of);
      }
      if (hipError_t e = hipGetLastError()) return (int)e;
    }
  }
  for (int t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    const int n = num_tensors - t0 < kMaxTensors ? num_tensors - t0 : kMaxTensors;
    Moved m;
    for (int t = 0; t < n; ++t) {
      m.base[t] = reinterpret_cast<char*>(const_cast<void*>(tensors[t0 + t]));
      m.head_bytes[t] = (int32_t)head_bytes[t0 + t];
      m.layer[t] = layer_of[t0 + t];
    }
    // Workgroups: one a (tensor, sequence, head), or of few of them larger ones, a
    // slice of the row each (64 bytes at least): what is in flight has to cover the
    // memory's latency, 16 KB a CU and more.
    const int64_t whole = (int64_t)num_kv_heads * batch * n;
    auto move = [&](auto threads, int slices) {
      constexpr int T = decltype(threads)::value;
      hipLaunchKernelGGL(HIP_KERNEL_NAME(evict_move_kernel<T>), dim3((unsigned)(num_kv_heads * slices), (unsigned)batch, (unsigned)n),
                         dim3(T), 0, s, a, m, slices);
    };
    if (whole >= 2048)
      move(std::integral_constant<int, 256>{}, 1);
    else
      move(std::integral_constant<int, 1024>{}, whole >= 512 ? 1 : 2);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  return MKV_OK;
}
