// Operations on the pages of the paged KV cache, over every layer's pools in
// one launch: whole-page copies, the compaction of accepted drafted tokens,
// and the page table's step (rows that fork, grow or are freed).
//
// All are moves of bytes and table entries: HBM bound where pages are copied
// (each byte read once and written once), latency bound in the table step.
// The pools' addresses travel in the kernel arguments (a scalar load each),
// so a program's 2 x layers tensors need no device-side pointer table.
#include "mkv_device.hpp"

namespace mkv {
namespace {

constexpr int kMaxTensors = 64;  // a launch's pools: 1 KB of kernel arguments

struct Pools {
  char* base[kMaxTensors];
  int64_t row_bytes[kMaxTensors];  // bytes of one token's row
};

// A workgroup copies kCopyBytes: four 16-byte loads a thread in flight ahead
// of their stores.
constexpr int kCopyThreads = 256;
constexpr int kCopyUnroll = 4;
constexpr int64_t kCopyBytes = (int64_t)kCopyThreads * kCopyUnroll * 16;

// bytes from s to d, both 4-byte aligned (16 with rows that are multiples of
// it): the chunk [lo, lo + kCopyBytes) of them.
MKV_DEV void copy_chunk(char* __restrict__ d, const char* __restrict__ s, int64_t lo, int64_t bytes, bool wide) {
  const int64_t hi = min(lo + kCopyBytes, bytes);
  if (wide) {
    u32x4 v[kCopyUnroll];
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j) {
      const int64_t o = lo + 16 * (j * kCopyThreads + (int)threadIdx.x);
      if (o < hi) v[j] = ld16_stream(s + o);
    }
#pragma unroll
    for (int j = 0; j < kCopyUnroll; ++j) {
      const int64_t o = lo + 16 * (j * kCopyThreads + (int)threadIdx.x);
      if (o < hi) __builtin_nontemporal_store(v[j], reinterpret_cast<u32x4*>(d + o));
    }
  } else {
    for (int64_t o = lo + 4 * (int)threadIdx.x; o < hi; o += 4 * kCopyThreads)
      *reinterpret_cast<uint32_t*>(d + o) = *reinterpret_cast<const uint32_t*>(s + o);
  }
}

// Page src[i] of every pool to page dst[i].  blockIdx.x: (tensor, chunk of a
// page), blockIdx.y strides over the pairs.
__global__ __launch_bounds__(kCopyThreads) void copy_pages_kernel(Pools p, int block_size, int chunks, int64_t num_pages,
                                                                 const void* __restrict__ src,
                                                                 const void* __restrict__ dst, int i64, int64_t pairs) {
  const int t = blockIdx.x / chunks;
  const int64_t lo = (int64_t)(blockIdx.x % chunks) * kCopyBytes;
  const int64_t bytes = p.row_bytes[t] * block_size;
  if (lo >= bytes) return;
  const bool wide = bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(p.base[t]) & 15) == 0;
  for (int64_t i = blockIdx.y; i < pairs; i += gridDim.y) {
    const int64_t a = load_index(src, i, i64), b = load_index(dst, i, i64);
    if (a < 0 || a >= num_pages || b < 0 || b >= num_pages || a == b) continue;
    copy_chunk(p.base[t] + b * bytes, p.base[t] + a * bytes, lo, bytes, wide);
  }
}

// ---------------------------------------------------------------------------
// Compaction: row prefix + accepted[b, j] of sequence b moves to prefix + j.
// A workgroup takes one sequence, a slice of the rows' columns and some of the
// pools, and holds all of the sequence's rows of a pool's slice in registers
// before it writes any, so rows may overlap in any order.  Several pools a
// workgroup share the look-up of the rows, which is a chain of three memory round
// trips (60 sequences, 56 pools: 29 us with one pool a workgroup).
// ---------------------------------------------------------------------------
constexpr int kMoveThreads = 256;
constexpr int kMoveItems = 8;                             // 16-byte items a thread holds
constexpr int kMaxMoves = kMoveThreads * kMoveItems;      // accepted offsets a sequence

// Columns of a slice (a power of two) for rows of `units` items, n rows.
__host__ MKV_DEV int slice_log2(int units, int n) {
  int l = 0;
  while ((1 << l) < units && (n << (l + 1)) <= kMaxMoves) ++l;
  return l;
}

template <typename T>
MKV_DEV void move_rows(char* base, const int64_t* src, const int64_t* dst, int n, int64_t row_bytes, int col0, int l2,
                       int units) {
  const int col = col0 + ((int)threadIdx.x & ((1 << l2) - 1));
  const bool mine = col < units;
  T v[kMoveItems];
  char* to[kMoveItems];
#pragma unroll
  for (int j = 0; j < kMoveItems; ++j) {
    const int e = (j * kMoveThreads + (int)threadIdx.x) >> l2;
    to[j] = nullptr;
    if (e < n && mine) {
      const int64_t s = src[e];
      if (s >= 0) {
        to[j] = base + dst[e] * row_bytes + (int64_t)col * sizeof(T);
        v[j] = *reinterpret_cast<const T*>(base + s * row_bytes + (int64_t)col * sizeof(T));
      }
    }
  }
  // every row of the slice has been read before any is written
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMoveItems; ++j)
    if (to[j]) *reinterpret_cast<T*>(to[j]) = v[j];
}

__global__ __launch_bounds__(kMoveThreads) __attribute__((amdgpu_waves_per_eu(5))) void compact_slots_kernel(
    Pools p, int num, int per_group, PagedIndex idx, const void* __restrict__ prefix, int prefix_i64,
    const void* __restrict__ accepted, int acc_i64, int64_t acc_stride, int n, int slices) {
  extern __shared__ int64_t slots[];  // [n] sources (-1: nothing to move), [n] destinations
  const int group = blockIdx.x / slices, slice = blockIdx.x % slices, b = blockIdx.y;
  const int64_t P = load_index(prefix, b, prefix_i64);
  for (int j = threadIdx.x; j < n; j += kMoveThreads) {
    const int64_t a = load_index(accepted, b * acc_stride + j, acc_i64);
    int64_t s = -1, d = -1;
    if (P >= 0 && P < ((int64_t)1 << 40) && a >= 0 && a != j && a < ((int64_t)1 << 40)) {
      const int64_t mask = ((int64_t)1 << idx.bs_log2) - 1;
      const int64_t ps = idx.physical_block(b, (P + a) >> idx.bs_log2), pd = idx.physical_block(b, (P + j) >> idx.bs_log2);
      if (ps >= 0 && pd >= 0) {
        s = (ps << idx.bs_log2) + ((P + a) & mask);
        d = (pd << idx.bs_log2) + ((P + j) & mask);
      }
    }
    slots[j] = s;
    slots[n + j] = d;
  }
  __syncthreads();
  for (int t = group * per_group; t < min(num, (group + 1) * per_group); ++t) {
    const int64_t row_bytes = p.row_bytes[t];
    const bool wide = row_bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(p.base[t]) & 15) == 0;
    const int units = (int)(row_bytes / (wide ? 16 : 4));
    const int l2 = slice_log2(units, n);
    if ((slice << l2) >= units) continue;
    if (wide)
      move_rows<u32x4>(p.base[t], slots, slots + n, n, row_bytes, slice << l2, l2, units);
    else
      move_rows<uint32_t>(p.base[t], slots, slots + n, n, row_bytes, slice << l2, l2, units);
  }
}

// ---------------------------------------------------------------------------
// The page table's step, one workgroup.  Whole numbers throughout: reference
// counts change by atomic additions, whose order does not matter, and fresh
// pages are the lowest-numbered free ones in row order, so the result is one
// only.  A second kernel copies the part-filled pages that it lists.
//
// Latency bound: a chain of memory round trips (parents; their lengths; the
// tables; the counts' additions; the counts; the stores), so what the steps hand
// on stays in LDS where it fits (tables of up to kLdsCells entries: 64 rows of 64
// pages in 7 us, where rows and fresh pages through memory took 16).
// ---------------------------------------------------------------------------
constexpr int kMaxRows = 1024;
constexpr int kAssignThreads = 1024;
constexpr int kCells = 4;     // table entries a thread looks at at once
constexpr int kScanPer = 16;  // reference counts a thread looks at in one sweep
constexpr int kLdsCells = 8192;

struct AssignArgs {
  int32_t* tables;
  int64_t bt_stride;
  int max_blocks;
  int64_t* seq_lens;
  int32_t* held;
  int32_t* refs;
  int64_t num_pages;
  int bs_log2;
  const void* parents;
  const void* tokens;
  int parents_i64, tokens_i64;
  uint8_t* granted;
  int rows;
  int32_t* new_tables;  // workspace: (rows, max_blocks), where they do not fit LDS
  int32_t* spare;       // workspace: rows * max_blocks fresh pages at most, likewise
  int32_t* copies;      // workspace: their number, then (source page, fresh page, live rows) each
};

// exclusive sum of v over the workgroup's threads in order; total in every thread
MKV_DEV int block_scan(int v, int* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kAssignThreads / 64; ++w) {
    const int c = lds[w];
    if (w < wave) before += c;
    total += c;
  }
  return before + x - v;
}
MKV_DEV void ref_add(const AssignArgs& a, int page, int by) {
  if (page >= 0 && page < a.num_pages)
    __hip_atomic_fetch_add(a.refs + page, by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
MKV_DEV int ref_get(const AssignArgs& a, int64_t page) {
  return __hip_atomic_load(a.refs + page, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// what this wave wrote is in memory (the workgroup's waves share the L1)
MKV_DEV void written() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <bool LDS>
__global__ __launch_bounds__(kAssignThreads) void assign_pages_kernel(AssignArgs a) {
  __shared__ int s_src[kMaxRows], s_keep[kMaxRows], s_held[kMaxRows], s_at[kMaxRows], s_start[kMaxRows], s_grow[kMaxRows];
  __shared__ __align__(16) int s_last[kMaxRows];
  __shared__ uint8_t s_copy[kMaxRows], s_drop[kMaxRows];
  __shared__ int s_scan[kAssignThreads / 64], s_listed;
  __shared__ int lds_tables[LDS ? kLdsCells : 1], lds_spare[LDS ? kLdsCells : 1];
  int* const fresh_tables = LDS ? lds_tables : a.new_tables;
  int* const spare = LDS ? lds_spare : a.spare;
  const int tid = threadIdx.x, R = a.rows, W = a.max_blocks;
  const int64_t bs = (int64_t)1 << a.bs_log2;
  // a thread a row
  int64_t new_len = 0;
  int want = 0, fill = 0, at = 0;
  bool valid = false, stays = false, gone = false, fits = false;
  if (tid == 0) s_listed = 0;
  if (tid < R) {
    const int64_t parent = load_index(a.parents, tid, a.parents_i64);
    const int64_t tok = a.tokens ? load_index(a.tokens, tid, a.tokens_i64) : 0;
    const int own_held = a.held[tid];
    valid = parent < R;
    gone = parent < 0;
    stays = parent == tid || !valid;
    const int src = gone || !valid ? tid : (int)parent;
    const int src_held = a.held[src];
    const int64_t len = a.seq_lens[src];
    const int old_held = min(max(own_held, 0), W);
    new_len = gone ? 0 : max(len, (int64_t)0);
    const int64_t need = (new_len + bs - 1) >> a.bs_log2;
    const int keep = gone ? 0 : stays ? old_held : (int)min(need, (int64_t)min(max(src_held, 0), W));
    const int64_t w = tok <= 0 ? 0 : (tok + bs - 1) >> a.bs_log2;
    fits = valid && w <= W;
    want = fits ? (int)w : 0;
    const int64_t last = new_len >> a.bs_log2;
    fill = last < keep ? (int)(new_len & (bs - 1)) : 0;
    at = (int)min(last, (int64_t)W);
    s_src[tid] = src;
    s_keep[tid] = keep;
    s_held[tid] = old_held;
    s_at[tid] = at;
    s_drop[tid] = stays;  // (for now: rows whose counts stay as they are)
  }
  __syncthreads();
  // the rows' new tables so far, and the counts of what is taken and let go
  // (kCells entries a thread at a time, their loads in one round trip)
  for (int i0 = tid; i0 < R * W; i0 += kAssignThreads * kCells) {
    int take[kCells], drop[kCells];
#pragma unroll
    for (int j = 0; j < kCells; ++j) {
      const int i = i0 + j * kAssignThreads;
      const int r = i < R * W ? i / W : 0, w = i < R * W ? i - r * W : W;
      take[j] = w < s_keep[r] ? a.tables[(int64_t)s_src[r] * a.bt_stride + w] : -1;
      drop[j] = w < s_held[r] && !s_drop[r] ? a.tables[(int64_t)r * a.bt_stride + w] : -1;
    }
#pragma unroll
    for (int j = 0; j < kCells; ++j) {
      const int i = i0 + j * kAssignThreads;
      if (i < R * W) {
        fresh_tables[i] = take[j];
        // (a page let go and taken again in the same place counts as before:
        // most of a beam's)
        if (!s_drop[i / W] && take[j] != drop[j]) {
          ref_add(a, take[j], 1);
          ref_add(a, drop[j], -1);
        }
      }
    }
  }
  written();
  __syncthreads();
  // a part-filled page that others hold too is copied by all but its first row;
  // rows without one have numbers that no other row shares
  int page = -1 - tid;
  if (tid < R && fill) {
    page = fresh_tables[tid * W + at];
    if (page < 0 || page >= a.num_pages) {
      page = -1 - tid;
      fill = 0;
    }
  }
  s_last[tid] = page;
  // (the counts: this row's page, and this thread's of the first sweep below)
  const int count = fill ? ref_get(a, page) : 0;
  uint32_t free_bits = 0;
  constexpr int kAgent = 16;  // sc1: coherent with the other CUs and with this one's atomics
  const __amdgpu_buffer_rsrc_t refs =
      __builtin_amdgcn_make_buffer_rsrc(a.refs, (short)0, (int)(a.num_pages * 4), 0x00020000);
  auto sweep = [&](int64_t p0) {
    // (16 bytes at a time, past the L1: the additions went past it; what lies
    // behind the last count reads 0 and is masked)
    free_bits = 0;
    const int64_t first = p0 + (int64_t)tid * kScanPer;
#pragma unroll
    for (int j = 0; j < kScanPer; j += 4) {
      const u32x4 c = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(refs, (int)((first + j) * 4), 0, kAgent));
#pragma unroll
      for (int e = 0; e < 4; ++e) free_bits |= c[e] == 0 && first + j + e < a.num_pages ? 1u << (j + e) : 0u;
    }
  };
  sweep(0);
  __syncthreads();
  int need = 0, grow = 0;
  bool copy = false;
  if (tid < R) {
    if (fill && count > 1) {
      int alike = 0, ahead = 0;
      for (int r0 = 0; r0 < R; r0 += 16) {  // (past the rows: numbers of their own)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const u32x4 v = *reinterpret_cast<const u32x4*>(s_last + r0 + j);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            alike += (int)v[e] == page;
            ahead += (int)v[e] == page && r0 + j + e < tid;
          }
        }
      }
      copy = ahead > 0 || count != alike;
    }
    grow = max(want - s_keep[tid], 0);
    need = fits ? (int)copy + grow : 0;
  }
  int total;
  const int start = block_scan(need, s_scan, total);
  // the lowest-numbered free pages, as many as are asked for
  int found = 0;
  for (int64_t p0 = 0; p0 < a.num_pages && found < total; p0 += kAssignThreads * kScanPer) {
    if (p0) sweep(p0);
    int here;
    int to = found + block_scan(__popc(free_bits), s_scan, here);
    while (free_bits && to < total) {
      const int j = __ffs(free_bits) - 1;
      free_bits &= free_bits - 1;
      spare[to++] = (int)(p0 + (int64_t)tid * kScanPer + j);
    }
    found += here;
  }
  if (!LDS) written();
  __syncthreads();
  if (tid < R) {
    const bool ok = fits && (need == 0 || start + need <= found);
    const bool drop = !ok && !stays;
    copy = copy && ok;
    grow = ok ? grow : 0;
    s_start[tid] = start + (copy ? 1 : 0);
    s_grow[tid] = grow;
    s_copy[tid] = copy;
    s_drop[tid] = drop;
    if (copy) {
      // (any order: the copies are apart)
      int32_t* c = a.copies + 1 + 3 * atomicAdd(&s_listed, 1);
      const int fresh = spare[start];
      c[0] = page;
      c[1] = fresh;
      c[2] = fill;
      ref_add(a, page, -1);
      ref_add(a, fresh, 1);
      s_last[tid] = fresh;
    }
    a.granted[tid] = ok;
    a.held[tid] = drop ? 0 : s_keep[tid] + grow;
    // (every row's length was read before the first barrier)
    a.seq_lens[tid] = drop ? 0 : new_len;
  }
  __syncthreads();
  if (tid == 0) a.copies[0] = s_listed;
  for (int i0 = tid; i0 < R * W; i0 += kAssignThreads * kCells) {
    int entry[kCells], add[kCells], sub[kCells];
#pragma unroll
    for (int j = 0; j < kCells; ++j) {
      const int i = i0 + j * kAssignThreads;
      add[j] = sub[j] = -1;
      entry[j] = 0;
      if (i < R * W) {
        const int r = i / W, w = i - r * W, keep = s_keep[r];
        if (w < keep)
          entry[j] = fresh_tables[i];
        else if (!s_drop[r] && w < keep + s_grow[r])
          entry[j] = add[j] = spare[s_start[r] + w - keep];
        if (s_drop[r]) {
          if (w < keep) sub[j] = entry[j];
          entry[j] = 0;
        } else if (s_copy[r] && w == s_at[r]) {
          entry[j] = s_last[r];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kCells; ++j) {
      const int i = i0 + j * kAssignThreads;
      ref_add(a, add[j], 1);
      ref_add(a, sub[j], -1);
      if (i < R * W) {
        const int r = i / W;
        a.tables[(int64_t)r * a.bt_stride + i - r * W] = entry[j];
      }
    }
  }
}

// The listed copies, blockIdx.y strides over them.
constexpr int kCopyRows = 16;
__global__ __launch_bounds__(kCopyThreads) void copy_listed_kernel(Pools p, int block_size, int chunks,
                                                                  const int32_t* __restrict__ copies) {
  const int n = copies[0];
  const int t = blockIdx.x / chunks;
  const int64_t lo = (int64_t)(blockIdx.x % chunks) * kCopyBytes;
  const int64_t page = p.row_bytes[t] * block_size;
  const bool wide = p.row_bytes[t] % 16 == 0 && (reinterpret_cast<uintptr_t>(p.base[t]) & 15) == 0;
  for (int i = blockIdx.y; i < n; i += gridDim.y) {
    const int32_t* c = copies + 1 + 3 * i;
    const int64_t bytes = p.row_bytes[t] * c[2];
    if (lo < bytes) copy_chunk(p.base[t] + c[1] * page, p.base[t] + c[0] * page, lo, bytes, wide);
  }
}

int log2_exact(int64_t v) {
  if (v <= 0 || (v & (v - 1))) return -1;
  int l = 0;
  while (((int64_t)1 << l) < v) ++l;
  return l;
}

// The tensors from t0 on as a launch's pools; the largest row in bytes.
int pools_at(const void* const* tensors, const int64_t* row_bytes, int num, int t0, Pools& p, int64_t& widest) {
  const int n = num - t0 < kMaxTensors ? num - t0 : kMaxTensors;
  widest = 0;
  for (int t = 0; t < n; ++t) {
    p.base[t] = reinterpret_cast<char*>(const_cast<void*>(tensors[t0 + t]));
    p.row_bytes[t] = row_bytes[t0 + t];
    widest = row_bytes[t0 + t] > widest ? row_bytes[t0 + t] : widest;
  }
  return n;
}

int check_pools(const void* const* tensors, const int64_t* row_bytes, int num, int64_t num_pages, int block_size) {
  if (num < 0 || num_pages < 0 || num_pages > 0x7fffffff || block_size <= 0 || block_size > (1 << 20))
    return MKV_ERR_BAD_SHAPE;
  if (num && (!tensors || !row_bytes)) return MKV_ERR_NULL_POINTER;
  for (int t = 0; t < num; ++t) {
    if (!tensors[t]) return MKV_ERR_NULL_POINTER;
    if (row_bytes[t] <= 0 || row_bytes[t] % 4 || row_bytes[t] > (1 << 24)) return MKV_ERR_BAD_SHAPE;
    if (reinterpret_cast<uintptr_t>(tensors[t]) & 3) return MKV_ERR_MISALIGNED;
  }
  return MKV_OK;
}

// A grid's first dimension in workgroups of 256 threads: below 2^32 threads.
constexpr int64_t kMaxGrid = 0xffffff;

// Whether a page's chunks of every tensor fit a launch's grid.
bool copies_fit(const int64_t* row_bytes, int num, int block_size) {
  int64_t widest = 0;
  for (int t = 0; t < num; ++t) widest = row_bytes[t] > widest ? row_bytes[t] : widest;
  const int n = num < kMaxTensors ? num : kMaxTensors;
  return (widest * block_size + kCopyBytes - 1) / kCopyBytes * n <= kMaxGrid;
}

bool index_ok(int dt) { return dt == MKV_INDEX_I32 || dt == MKV_INDEX_I64; }

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" int mkv_copy_pages(const void* const* tensors, const int64_t* row_bytes, int num_tensors, int64_t num_pages,
                              int block_size, const void* src, const void* dst, int index_dtype, int64_t pairs,
                              void* stream) {
  if (int st = check_pools(tensors, row_bytes, num_tensors, num_pages, block_size)) return st;
  if (pairs < 0) return MKV_ERR_BAD_SHAPE;
  if (!index_ok(index_dtype)) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (pairs == 0 || num_tensors == 0) return MKV_OK;
  if (!src || !dst) return MKV_ERR_NULL_POINTER;
  if (!copies_fit(row_bytes, num_tensors, block_size)) return MKV_ERR_BAD_SHAPE;
  for (int t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    Pools p;
    int64_t widest;
    const int n = pools_at(tensors, row_bytes, num_tensors, t0, p, widest);
    const int64_t chunks = (widest * block_size + kCopyBytes - 1) / kCopyBytes;
    hipLaunchKernelGGL(copy_pages_kernel, dim3((unsigned)(chunks * n), (unsigned)(pairs < 65535 ? pairs : 65535)),
                       dim3(kCopyThreads), 0, reinterpret_cast<hipStream_t>(stream), p, block_size, (int)chunks,
                       num_pages, src, dst, (int)(index_dtype == MKV_INDEX_I64), pairs);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  return MKV_OK;
}

extern "C" int mkv_compact_slots(const void* const* tensors, const int64_t* row_bytes, int num_tensors,
                                 int64_t num_pages, int block_size, const int32_t* block_tables, int64_t bt_stride,
                                 int max_blocks, const void* prefix_lens, int prefix_dtype, const void* accepted,
                                 int accepted_dtype, int64_t accepted_stride, int batch, int num_accepted,
                                 void* stream) {
  if (int st = check_pools(tensors, row_bytes, num_tensors, num_pages, block_size)) return st;
  if (batch < 0 || num_accepted < 0 || num_accepted > kMaxMoves || max_blocks < 0 || batch > 65535) return MKV_ERR_BAD_SHAPE;
  if (!index_ok(prefix_dtype) || !index_ok(accepted_dtype)) return MKV_ERR_UNSUPPORTED_DTYPE;
  const int bs_log2 = log2_exact(block_size);
  if (bs_log2 < 0) return MKV_ERR_BAD_BLOCK_SIZE;
  if (batch == 0 || num_accepted == 0 || num_tensors == 0) return MKV_OK;
  if (!block_tables || !prefix_lens || !accepted) return MKV_ERR_NULL_POINTER;
  if (bt_stride < max_blocks || accepted_stride < num_accepted) return MKV_ERR_BAD_STRIDE;
  PagedIndex idx{block_tables, bt_stride, max_blocks, num_pages, bs_log2, 0};
  Pools p;
  int n;
  int64_t widest, slices, per, groups;
  auto plan = [&](int t0) {  // the launch for the tensors from t0 on
    n = pools_at(tensors, row_bytes, num_tensors, t0, p, widest);
    slices = 1;
    for (int t = 0; t < n; ++t) {
      const bool wide = p.row_bytes[t] % 16 == 0 && (reinterpret_cast<uintptr_t>(p.base[t]) & 15) == 0;
      const int u = (int)(p.row_bytes[t] / (wide ? 16 : 4)), l2 = slice_log2(u, num_accepted);
      const int64_t c = ((int64_t)u + (1 << l2) - 1) >> l2;
      slices = c > slices ? c : slices;
    }
    // pools a workgroup: one while that leaves CUs free, at most eight
    per = (int64_t)n * slices * batch / 1024;
    per = per < 1 ? 1 : per > 8 ? 8 : per;
    groups = (n + per - 1) / per;
    return slices * groups <= kMaxGrid;
  };
  // (every launch fits, or none runs)
  for (int t0 = 0; t0 < num_tensors; t0 += kMaxTensors)
    if (!plan(t0)) return MKV_ERR_BAD_SHAPE;
  for (int t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    if (num_tensors > kMaxTensors) plan(t0);
    hipLaunchKernelGGL(compact_slots_kernel, dim3((unsigned)(slices * groups), (unsigned)batch), dim3(kMoveThreads),
                       (size_t)num_accepted * 16, reinterpret_cast<hipStream_t>(stream), p, n, (int)per, idx,
                       prefix_lens, (int)(prefix_dtype == MKV_INDEX_I64), accepted,
                       (int)(accepted_dtype == MKV_INDEX_I64), accepted_stride, num_accepted, (int)slices);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  return MKV_OK;
}

extern "C" size_t mkv_assign_pages_workspace_size(int rows, int max_blocks) {
  if (rows <= 0 || max_blocks < 0) return 0;
  const size_t cells = (size_t)rows * max_blocks;
  return ((cells > kLdsCells ? cells * 2 : 0) + (size_t)rows * 3 + 1) * sizeof(int32_t);
}

extern "C" int mkv_assign_pages(const void* const* tensors, const int64_t* row_bytes, int num_tensors,
                                int64_t num_pages, int block_size, int32_t* block_tables, int64_t bt_stride,
                                int max_blocks, int64_t* seq_lens, int32_t* held, int32_t* ref_counts,
                                const void* parents, int parents_dtype, const void* tokens, int tokens_dtype,
                                uint8_t* granted, int rows, void* workspace, size_t workspace_bytes, void* stream) {
  if (int st = check_pools(tensors, row_bytes, num_tensors, num_pages, block_size)) return st;
  if (rows < 0 || rows > kMaxRows || num_pages > (1 << 28) || max_blocks < 0 || (int64_t)rows * max_blocks > (1 << 28)) return MKV_ERR_BAD_SHAPE;
  if (!index_ok(parents_dtype) || (tokens && !index_ok(tokens_dtype))) return MKV_ERR_UNSUPPORTED_DTYPE;
  const int bs_log2 = log2_exact(block_size);
  if (bs_log2 < 0) return MKV_ERR_BAD_BLOCK_SIZE;
  if (rows == 0) return MKV_OK;
  if (!block_tables || !seq_lens || !held || !ref_counts || !parents || !granted || !workspace)
    return MKV_ERR_NULL_POINTER;
  if (bt_stride < max_blocks) return MKV_ERR_BAD_STRIDE;
  if (workspace_bytes < mkv_assign_pages_workspace_size(rows, max_blocks)) return MKV_ERR_WORKSPACE_TOO_SMALL;
  // (ahead of the table's step, which the copies complete)
  if (!copies_fit(row_bytes, num_tensors, block_size)) return MKV_ERR_BAD_SHAPE;
  int32_t* ws = reinterpret_cast<int32_t*>(workspace);
  const size_t cells = (size_t)rows * max_blocks;
  // (a row asks for a copy and at most max_blocks pages: a row whose page is
  // copied keeps at least that one)
  AssignArgs a{block_tables, bt_stride, max_blocks, seq_lens, held, ref_counts, num_pages, bs_log2, parents, tokens,
               (int)(parents_dtype == MKV_INDEX_I64), (int)(tokens_dtype == MKV_INDEX_I64), granted, rows, ws,
               ws + cells, cells > kLdsCells ? ws + 2 * cells : ws};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (cells > kLdsCells)
    hipLaunchKernelGGL(HIP_KERNEL_NAME(assign_pages_kernel<false>), dim3(1), dim3(kAssignThreads), 0, s, a);
  else
    hipLaunchKernelGGL(HIP_KERNEL_NAME(assign_pages_kernel<true>), dim3(1), dim3(kAssignThreads), 0, s, a);
  if (hipError_t e = hipGetLastError()) return (int)e;
  for (int t0 = 0; t0 < num_tensors; t0 += kMaxTensors) {
    Pools p;
    int64_t widest;
    const int n = pools_at(tensors, row_bytes, num_tensors, t0, p, widest);
    const int64_t chunks = (widest * block_size + kCopyBytes - 1) / kCopyBytes;
    hipLaunchKernelGGL(copy_listed_kernel, dim3((unsigned)(chunks * n), (unsigned)(rows < kCopyRows ? rows : kCopyRows)), dim3(kCopyThreads), 0, s, p,
                       block_size, (int)chunks, a.copies);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  return MKV_OK;
}
