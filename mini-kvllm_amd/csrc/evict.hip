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
#include <type_traits>

#include "mkv_device.hpp"

namespace mkv {
namespace {

constexpr int kMaxTensors = 64;  // a launch's tensors, their addresses in the kernel arguments
constexpr int kBins = 2048;
constexpr int kLdsKeys = 8192;   // capacities up to this keep their keys in LDS

struct EvictArgs {
  PagedIndex idx;
  const void* lens;
  int lens_i64;
  int batch, heads;
  int budget, sinks, recent;
  int64_t* new_lens;
  int32_t* slots;   // workspace: (layers, batch, heads, budget), the kept tokens' slots in order
  uint32_t* keys;   // workspace: (layers, batch, heads, key_stride), for long tables
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
MKV_DEV uint32_t key_at(const EvictArgs& a, const float* w, int b, int h, int t) {
  const int s = slot_of(a, b, t);
  return s >= 0 ? order_of(w[(int64_t)s * a.heads + h]) : 0u;
}

// Workgroups of one (layer, sequence) lie 8 apart, on one XCD: its heads share the
// weights' cache lines.
MKV_DEV bool place_of(const EvictArgs& a, int layers, int i, int& layer, int& b, int& h) {
  const int group = i / (8 * a.heads), in = i % (8 * a.heads);
  const int pair = group * 8 + in % 8;
  h = in / 8;
  layer = pair / a.batch;
  b = pair % a.batch;
  return layer < layers;
}

// The weights' keys of long tables, transposed to a row a head.
__global__ __launch_bounds__(256) void evict_keys_kernel(EvictArgs a, Weights w, int layer0) {
  const int b = blockIdx.y, layer = blockIdx.z;
  int64_t len;
  const int n = length_of(a, b, len);
  if (n <= a.budget) return;
  uint32_t* const out = a.keys + (int64_t)((layer0 + layer) * a.batch + b) * a.heads * a.key_stride;
  for (int t = blockIdx.x * 256 + threadIdx.x; t < n; t += gridDim.x * 256) {
    const int s = slot_of(a, b, t);
    const float* row = w.base[layer] + (int64_t)max(s, 0) * a.heads;
    for (int h = 0; h < a.heads; ++h) out[h * a.key_stride + t] = s >= 0 ? order_of(row[h]) : 0u;
  }
}

template <int T, bool LDS>
__global__ __launch_bounds__(T) void evict_select_kernel(EvictArgs a, Weights w, int layer0, int layers) {
  extern __shared__ uint32_t lds_keys[];
  __shared__ int hist[kBins];
  __shared__ int scan[T / 64], found[2], part_kept[T / 64], part_equal[T / 64];
  int layer, b, h;
  if (!place_of(a, layers, blockIdx.x, layer, b, h)) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int64_t len;
  const int n = length_of(a, b, len);
  if (layer0 + layer == 0 && h == 0 && tid == 0) a.new_lens[b] = min(len, (int64_t)a.budget);
  if (n <= a.budget) return;
  const int64_t at = ((int64_t)(layer0 + layer) * a.batch + b) * a.heads + h;
  const uint32_t* keys = LDS ? lds_keys : a.keys + at * a.key_stride;
  if constexpr (LDS) {
    constexpr int kAhead = 4;  // (their loads in one round trip)
    for (int t0 = tid; t0 < n; t0 += T * kAhead) {
      uint32_t k[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) k[j] = t0 + j * T < n ? key_at(a, w.base[layer], b, h, t0 + j * T) : 0u;
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (t0 + j * T < n) lds_keys[t0 + j * T] = k[j];
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
      const int shift = kShift[pass], bins = 1 << kBits[pass];
      __syncthreads();
      for (int i = tid; i < kBins; i += T) hist[i] = 0;
      __syncthreads();
      const uint32_t above = pass == 0 ? 0u : least >> kShift[pass > 0 ? pass - 1 : 0];
      for (int t0 = first; t0 < last; t0 += T) {
        const int t = t0 + tid;
        const uint32_t k = t < last ? keys[t] : 0u;
        const bool in = t < last && (pass == 0 || k >> kShift[pass > 0 ? pass - 1 : 0] == above);
        const int d = (int)(k >> shift) & (bins - 1);
        // (many alike: one addition for the wave)
        const uint64_t mine = __builtin_amdgcn_ballot_w64(in);
        if (mine == 0) continue;
        const int d0 = __builtin_amdgcn_readlane(d, __builtin_ctzll(mine));
        if (__builtin_amdgcn_ballot_w64(in && d == d0) == mine) {
          if (lane == __builtin_ctzll(mine)) atomicAdd(&hist[d0], __popcll(mine));
        } else if (in) {
          atomicAdd(&hist[d], 1);
        }
      }
      __syncthreads();
      // the bin in which the want-th largest lies; thread tid has bins from the top
      constexpr int kPer = kBins / T;
      int c[kPer], own = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        c[j] = hist[kBins - 1 - (tid * kPer + j)];
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
  } else {
    __syncthreads();
  }
  // ---- the kept tokens' places: a run of tokens a wave ----
  constexpr int kWaves = T / 64;
  const int run = (n + 64 * kWaves - 1) / (64 * kWaves) * 64;
  const int t_lo = wave * run, t_hi = min(n, t_lo + run);
  int kept = 0, equal = 0;
  for (int t0 = t_lo; t0 < t_hi; t0 += 64) {
    const int t = t0 + lane;
    const bool in = t < t_hi, mid = in && t >= first && t < last;
    const uint32_t k = mid ? keys[t] : 0u;
    kept += __popcll(__builtin_amdgcn_ballot_w64((in && !mid) || (mid && k > least)));
    equal += __popcll(__builtin_amdgcn_ballot_w64(mid && k == least));
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
  for (int t0 = t_lo; t0 < t_hi; t0 += 64) {
    const int t = t0 + lane;
    const bool in = t < t_hi, mid = in && t >= first && t < last;
    const uint32_t k = mid ? keys[t] : 0u;
    const bool eq = mid && k == least;
    const uint64_t eqs = __builtin_amdgcn_ballot_w64(eq), below = (1ull << lane) - 1;
    const bool keep = (in && !mid) || (mid && k > least) || (eq && tied + __popcll(eqs & below) < want);
    const uint64_t keeps = __builtin_amdgcn_ballot_w64(keep);
    const int place = to + __popcll(keeps & below);
    if (keep && place < a.budget) out[place] = slot_of(a, b, t);
    to += __popcll(keeps);
    tied += __popcll(eqs);
  }
}

// Rows of one head (X a 16- or 4-byte item, `units` of them a row from `col0` on), or
// of all heads together (heads_together: 4 bytes a head).
constexpr int kItems = 8;  // a thread's, in registers
constexpr int kMaxHeadBytes = 64 * kItems * 4;  // (a row of the smallest workgroup's 4-byte items)
template <typename X, int T>
MKV_DEV void move_rows(const EvictArgs& a, char* base, int64_t token_bytes, int64_t off, int units, int b,
                       const int32_t* slots, int64_t head_stride, bool heads_together) {
  const int mask = (1 << a.idx.bs_log2) - 1;
  const int32_t* bt = a.idx.block_tables + (int64_t)b * a.idx.bt_stride;
  const int per = max(T * kItems / units, 1);  // rows of a batch
  for (int j0 = 0; j0 < a.budget; j0 += per) {
    const int rows = min(per, a.budget - j0);
    X v[kItems];
    char* to[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      const int item = i * T + (int)threadIdx.x;
      const int r = item / units, c = item - r * units;
      to[i] = nullptr;
      if (r < rows) {
        const int j = j0 + r;
        const int s = slots[(heads_together ? c * head_stride : 0) + j];
        const int p = bt[j >> a.idx.bs_log2];
        if (s >= 0 && p >= 0 && p < a.idx.num_blocks) {
          const int d = (p << a.idx.bs_log2) + (j & mask);
          if (d != s) {
            to[i] = base + d * token_bytes + off + c * (int64_t)sizeof(X);
            v[i] = *reinterpret_cast<const X*>(base + s * token_bytes + off + c * (int64_t)sizeof(X));
          }
        }
      }
    }
    // every row of the batch has been read before any is written
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if constexpr (T > 64) __syncthreads();
#pragma unroll
    for (int i = 0; i < kItems; ++i)
      if (to[i]) *reinterpret_cast<X*>(to[i]) = v[i];
  }
}

template <int T>
__global__ __launch_bounds__(T) void evict_move_kernel(EvictArgs a, Moved m, int slices) {
  const int h = blockIdx.x / slices, slice = blockIdx.x % slices, b = blockIdx.y, t = blockIdx.z;
  int64_t len;
  if (length_of(a, b, len) <= a.budget) return;
  const int64_t bytes = m.head_bytes[t], token = bytes * a.heads;
  const int64_t lists = ((int64_t)m.layer[t] * a.batch + b) * a.heads;
  const int32_t* slots = a.slots + (lists + h) * a.budget;
  char* const base = m.base[t];
  if (bytes == 4) {
    if (h == 0 && slice == 0) move_rows<uint32_t, T>(a, base, token, 0, a.heads, b, slots, a.budget, true);
  } else if (bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(base) & 15) == 0) {
    // a slice: an even share of the row's 16-byte items
    const int units = (int)(bytes / 16), share = (units + slices - 1) / slices, c0 = slice * share;
    if (c0 < units)
      move_rows<u32x4, T>(a, base, token, h * bytes + 16 * c0, min(share, units - c0), b, slots, 0, false);
  } else if (slice == 0) {
    move_rows<uint32_t, T>(a, base, token, h * bytes, (int)(bytes / 4), b, slots, 0, false);
  }
}

int log2_exact(int64_t v) {
  if (v <= 0 || (v & (v - 1))) return -1;
  int l = 0;
  while (((int64_t)1 << l) < v) ++l;
  return l;
}

int64_t capacity_of(int max_blocks, int block_size) { return (int64_t)max_blocks * block_size; }

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_evict_tokens_workspace_size(int num_layers, int batch, int num_kv_heads, int block_size,
                                                  int max_blocks, int budget) {
  if (num_layers <= 0 || batch <= 0 || num_kv_heads <= 0 || max_blocks <= 0 || block_size <= 0 || budget <= 0) return 0;
  const size_t lists = (size_t)num_layers * batch * num_kv_heads, cap = (size_t)capacity_of(max_blocks, block_size);
  return lists * ((size_t)budget + (cap > kLdsKeys ? cap : 0)) * 4;
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
  if (bs_log2 < 0) return MKV_ERR_BAD_BLOCK_SIZE;
  if (num_pages > (0x7fffffff >> bs_log2) || capacity_of(max_blocks, block_size) > 0x7fff0000) return MKV_ERR_BAD_SHAPE;
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
  if ((reinterpret_cast<uintptr_t>(workspace) & 3) != 0) return MKV_ERR_MISALIGNED;
  const int64_t cap = capacity_of(max_blocks, block_size);
  const int64_t pairs = ((int64_t)(num_layers < kMaxTensors ? num_layers : kMaxTensors) * batch + 7) / 8 * 8;
  if (pairs * num_kv_heads > 0x3fffff || (int64_t)num_layers * batch * num_kv_heads > 0x7fffffff) return MKV_ERR_BAD_SHAPE;
  if (workspace_bytes < mkv_evict_tokens_workspace_size(num_layers, batch, num_kv_heads, block_size, max_blocks, budget))
    return MKV_ERR_WORKSPACE_TOO_SMALL;
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
  a.keys = reinterpret_cast<uint32_t*>(a.slots + (size_t)num_layers * batch * num_kv_heads * budget);
  a.key_stride = cap;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  for (int l0 = 0; l0 < num_layers; l0 += kMaxTensors) {
    const int layers = num_layers - l0 < kMaxTensors ? num_layers - l0 : kMaxTensors;
    Weights w;
    for (int l = 0; l < layers; ++l) w.base[l] = reinterpret_cast<const float*>(weights[l0 + l]);
    const dim3 grid((unsigned)(((int64_t)layers * batch + 7) / 8 * 8 * num_kv_heads));
    if (cap > kLdsKeys) {
      const unsigned x = (unsigned)((cap + 255) / 256 < 256 ? (cap + 255) / 256 : 256);
      hipLaunchKernelGGL(evict_keys_kernel, dim3(x, (unsigned)batch, (unsigned)layers), dim3(256), 0, s, a, w, l0);
      if (hipError_t e = hipGetLastError()) return (int)e;
      hipLaunchKernelGGL(HIP_KERNEL_NAME(evict_select_kernel<1024, false>), grid, dim3(1024), 0, s, a, w, l0, layers);
    } else {
      hipLaunchKernelGGL(HIP_KERNEL_NAME(evict_select_kernel<256, true>), grid, dim3(256), (size_t)cap * 4, s, a, w, l0, layers);
    }
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  for (int t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    const int n = num_tensors - t0 < kMaxTensors ? num_tensors - t0 : kMaxTensors;
    Moved m;
    for (int t = 0; t < n; ++t) {
      m.base[t] = reinterpret_cast<char*>(const_cast<void*>(tensors[t0 + t]));
      m.head_bytes[t] = (int32_t)head_bytes[t0 + t];
      m.layer[t] = layer_of[t0 + t];
    }
    hipLaunchKernelGGL(HIP_KERNEL_NAME(evict_move_kernel<256>), dim3((unsigned)num_kv_heads, (unsigned)batch, (unsigned)n),
                       dim3(256), 0, s, a, m, 1);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  return MKV_OK;
}
