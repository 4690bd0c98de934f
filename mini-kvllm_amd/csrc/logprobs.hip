// Log probabilities of given tokens, the entropy of each row's distribution
// and its top alternatives, from one pass over the logits.
//
//   m = max x, s = sum e^(x - m), t = sum e^(x - m) (x - m)
//   log p(i) = (x_i - m) - log s        entropy = log s - t / s
//
// Read bound: the pass over (rows, vocab) logits is all but a few bytes of the
// traffic.  Pass 1 gives a workgroup kChunk logits of one row (32 a thread, in
// registers), so that a single row still spreads over many CUs, and leaves per
// chunk (m, s, t), joined by the usual rescaling, and the maximum of each
// thread's 32 logits.  Pass 2, one workgroup a row, joins the chunks and finds
// the top k from those maxima: a value that at least k threads' maxima reach
// bounds the k-th largest logit from below, so only the threads' logits that
// reach it are read again (a few dozen of the vocabulary).  Selecting in pass 1
// would cost its workgroups as many VALU cycles again as the whole softmax.
#include "mkv_device.hpp"

namespace mkv {
namespace {

constexpr int kLpThreads = 256;
constexpr int kPer = 32;                      // logits a thread holds
constexpr int kChunk = kLpThreads * kPer;     // 8192
constexpr int kMaxTop = 64;
constexpr int kMaxSub = 128;                  // threads' shares that pass 2 reads again at most
constexpr int kMaxCand = kMaxSub * kPer;      // 4096 candidates

struct LpArgs {
  const void* logits;
  int64_t row_stride;
  int64_t rows;
  int vocab;
  int chunks;
  const void* ids;
  int ids_i64, num_ids;
  int64_t ids_stride;
  int top;
  float* logprobs;     // (rows, num_ids)
  float* entropy;      // (rows)
  float* top_logprobs; // (rows, top)
  int64_t* top_ids;    // (rows, top)
  float* stats;        // workspace: (rows, chunks, 4): m, s, t, unused
  float* maxima;       // workspace: (rows, chunks, 256)
};

// max that a NaN on either side wins (v_maximum3_f32)
MKV_DEV float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// unsigned order of logits: NaN above +inf, the two zeros alike; 0 for none
MKV_DEV uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
MKV_DEV uint64_t key_of(float x, int i) { return (uint64_t)order_of(x) << 32 | (uint32_t)~i; }

template <int DT>
MKV_DEV float logit_at(const char* row, int64_t i) {
  if constexpr (DT == MKV_DTYPE_F32) return reinterpret_cast<const float*>(row)[i];
  const uint32_t b = reinterpret_cast<const uint16_t*>(row)[i];
  return DT == MKV_DTYPE_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// The 16-byte pieces of a chunk: piece j of thread tid starts at logit
// first + (j * 256 + tid) * kVec, where first brings the pieces onto 16-byte
// boundaries (a row may start anywhere); pieces that cross an end of the row
// are read a logit at a time.
template <int DT>
struct Pieces {
  static constexpr int kVec = DT == MKV_DTYPE_F32 ? 4 : 8;
  static constexpr int kNum = kPer / kVec;
  MKV_DEV static int shift(const char* row) {
    return (int)((reinterpret_cast<uintptr_t>(row) & 15) / (16 / kVec));
  }
  MKV_DEV static int64_t start(int chunk, int j, int tid, int shift) {
    return (int64_t)chunk * kChunk + (j * kLpThreads + tid) * kVec - shift;
  }
  // x[0..kVec): -inf outside [0, vocab)
  MKV_DEV static void load(const char* row, int64_t i, int vocab, float* x) {
    if (i >= 0 && i + kVec <= vocab) {
      const u32x4 w = ld16(row + i * (16 / kVec));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (DT == MKV_DTYPE_F32) {
          x[e] = __uint_as_float(w[e]);
        } else if constexpr (DT == MKV_DTYPE_BF16) {
          x[2 * e] = __uint_as_float(w[e] << 16);
          x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        } else {
          x[2 * e] = f16_bits_to_f32(w[e] & 0xffffu);
          x[2 * e + 1] = f16_bits_to_f32(w[e] >> 16);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        x[e] = -__builtin_huge_valf();
        if (i + e >= 0 && i + e < vocab) x[e] = logit_at<DT>(row, i + e);
      }
    }
  }
};

// (m, s, t) of two parts; a part without logits has m = -inf, s = t = 0.
struct Stat {
  float m, s, t;
};
MKV_DEV Stat join(Stat a, Stat b) {
  const float m = maximum(a.m, b.m);
  // equal maxima need no factor (and equal infinities have no difference)
  const float da = a.m == m ? 0.0f : a.m - m, db = b.m == m ? 0.0f : b.m - m;
  const float fa = expf(da), fb = expf(db);
  Stat r;
  r.m = m;
  r.s = a.s * fa + b.s * fb;
  // (a factor of 0 belongs to a difference of -inf or below -104)
  r.t = (fa > 0.0f ? fa * (a.t + a.s * da) : 0.0f) + (fb > 0.0f ? fb * (b.t + b.s * db) : 0.0f);
  if (m != m) r.s = r.t = m;
  return r;
}

template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprobs_chunk_kernel(LpArgs a) {
  using P = Pieces<DT>;
  const int chunk = blockIdx.x, tid = threadIdx.x;
  const int64_t r = blockIdx.y + (int64_t)blockIdx.z * 32768;
  if (r >= a.rows) return;
  const char* row = reinterpret_cast<const char*>(a.logits) + r * a.row_stride * (16 / P::kVec);
  const int shift = P::shift(row);
  float x[kPer];
#pragma unroll
  for (int j = 0; j < P::kNum; ++j) P::load(row, P::start(chunk, j, tid, shift), a.vocab, x + j * P::kVec);
  float own = x[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) own = maximum(own, x[i]);
  if (a.top) a.maxima[(r * a.chunks + chunk) * kLpThreads + tid] = own;
  float m = own;
#pragma unroll
  for (int o = 32; o; o >>= 1) m = maximum(m, __shfl_xor(m, o));
  // the wave's sums around its own maximum; a wave without a finite one has
  // none (all -inf), or NaN (a NaN or +inf among its logits)
  Stat w{m, 0.0f, 0.0f};
  if (m != -__builtin_huge_valf()) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      // below e^-200 nothing is left in 32 bits; -inf lands there too
      const float d = maximum(x[i] - m, -200.0f);
      const float e = __builtin_amdgcn_exp2f(d * kLog2e);
      w.s += e;
      w.t = __builtin_fmaf(e, d, w.t);
    }
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    w.s += __shfl_xor(w.s, o);
    w.t += __shfl_xor(w.t, o);
  }
  __shared__ Stat part[kLpThreads / 64];
  if ((tid & 63) == 0) part[tid >> 6] = w;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int i = 1; i < kLpThreads / 64; ++i) w = join(w, part[i]);
    float* o = a.stats + (r * a.chunks + chunk) * 4;
    o[0] = w.m;
    o[1] = w.s;
    o[2] = w.t;
  }
}

// number of threads' true bits, times weight: the sum of v over the workgroup
MKV_DEV int block_count(int v, int* lds) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  int n = 0;
#pragma unroll
  for (int w = 0; w < kLpThreads / 64; ++w) n += lds[w];
  return n;
}

template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprobs_row_kernel(LpArgs a) {
  using P = Pieces<DT>;
  __shared__ Stat parts[kLpThreads / 64];
  __shared__ int counts[kLpThreads / 64];
  __shared__ uint64_t cand[kMaxCand];
  __shared__ int subs[kMaxSub];
  __shared__ int fill;
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x;
  const char* row = reinterpret_cast<const char*>(a.logits) + r * a.row_stride * (16 / P::kVec);
  // the given tokens' logits go out first
  float given = 0.0f;
  int64_t id = -1;
  if (tid < a.num_ids) {
    id = load_index(a.ids, r * a.ids_stride + tid, a.ids_i64);
    if (id >= 0 && id < a.vocab) given = logit_at<DT>(row, id);
  }
  Stat st{-__builtin_huge_valf(), 0.0f, 0.0f};
  for (int c = tid; c < a.chunks; c += kLpThreads) {
    const u32x4 v = ld16(a.stats + (r * a.chunks + c) * 4);
    st = join(st, Stat{__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2])});
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) st = join(st, Stat{__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.t, o)});
  if ((tid & 63) == 0) parts[tid >> 6] = st;
  __syncthreads();
  st = parts[0];
#pragma unroll
  for (int w = 1; w < kLpThreads / 64; ++w) st = join(st, parts[w]);
  const float m = st.m, log_s = logf(st.s);
  if (tid == 0) a.entropy[r] = log_s - st.t / st.s;
  for (int i = tid; i < a.num_ids; i += kLpThreads) {
    if (i >= kLpThreads) {
      id = load_index(a.ids, r * a.ids_stride + i, a.ids_i64);
      if (id >= 0 && id < a.vocab) given = logit_at<DT>(row, id);
    }
    a.logprobs[r * a.num_ids + i] = id < 0 ? 0.0f : id < a.vocab ? (given - m) - log_s : __builtin_nanf("");
  }
  if (a.top == 0) return;

  // ---- a threshold that k to kMaxSub threads' maxima reach ----
  const int k = a.top;
  const int shift = P::shift(row);
  const int subs_all = a.chunks * kLpThreads;
  const float* maxima = a.maxima + r * subs_all;
  // a thread of pass 1 without a logit of the row counts for nothing
  auto sub_key = [&](int i) -> uint32_t {
    const int64_t s = P::start(i / kLpThreads, 0, i % kLpThreads, shift);
    return s >= a.vocab || s + P::kVec <= 0 ? 0u : order_of(maxima[i]);
  };
  // (from 1, which every share with a logit reaches, to above the largest)
  uint32_t lo = 1, hi = 0xffffffffu;
  auto reach = [&](uint32_t t) {
    int n = 0;
    for (int i = tid; i < subs_all; i += kLpThreads) n += sub_key(i) >= t;
    return block_count(n, counts);
  };
  int n_sub = reach(lo);
  bool ties = false;
  if (n_sub > kMaxSub) {
    int n_hi = reach(hi);
    if (n_hi >= k) {  // (k NaNs or more)
      lo = hi;
      n_sub = n_hi;
    } else {
      // reach(lo) > kMaxSub, reach(hi) < k
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const int n = reach(mid);
        if (n >= k) {
          lo = mid;
          n_sub = n;
          if (n <= kMaxSub) break;
        } else {
          hi = mid;
        }
      }
    }
    ties = n_sub > kMaxSub;  // many shares with the same largest logit, lo
  }
  // ---- the logits that reach it: with ties those above it, then the first
  // that equal it, in the order of their places ----
  const uint32_t from = ties && lo != 0xffffffffu ? lo + 1 : ties ? 0xffffffffu : lo;
  if (tid == 0) fill = 0;
  __syncthreads();
  const bool above = !(ties && lo == 0xffffffffu);
  if (above) {
    for (int i = tid; i < subs_all; i += kLpThreads)
      if (sub_key(i) >= from) {
        const int at = atomicAdd(&fill, 1);
        if (at < kMaxSub) subs[at] = i;
      }
  }
  __syncthreads();
  const int num_sub = above ? min(fill, kMaxSub) : 0;
  __syncthreads();
  if (tid == 0) fill = 0;
  __syncthreads();
  for (int w = tid; w < num_sub * P::kNum; w += kLpThreads) {
    const int i = subs[w / P::kNum];
    const int64_t s = P::start(i / kLpThreads, w % P::kNum, i % kLpThreads, shift);
    float x[P::kVec];
    P::load(row, s, a.vocab, x);
#pragma unroll
    for (int e = 0; e < P::kVec; ++e)
      if (s + e >= 0 && s + e < a.vocab && order_of(x[e]) >= from) {
        const int at = atomicAdd(&fill, 1);
        if (at < kMaxCand) cand[at] = key_of(x[e], (int)(s + e));
      }
  }
  __syncthreads();
  int n = min(fill, kMaxCand);
  if (ties) {
    // fewer than k may lie above: the first that equal lo, piece by piece
    int have = n;
    for (int64_t base = 0; base < a.vocab && have < k; base += kLpThreads) {
      const int64_t i = base + tid;
      const float x = i < a.vocab ? logit_at<DT>(row, i) : 0.0f;
      const bool hit = i < a.vocab && order_of(x) == lo;
      const uint64_t ball = __builtin_amdgcn_ballot_w64(hit);
      const int lane = tid & 63;
      int before = __popcll(ball & ((1ull << lane) - 1));
      __syncthreads();
      if (lane == 0) counts[tid >> 6] = __popcll(ball);
      __syncthreads();
      int all = 0;
#pragma unroll
      for (int w = 0; w < kLpThreads / 64; ++w) {
        if (w < (tid >> 6)) before += counts[w];
        all += counts[w];
      }
      if (hit && have + before < k) cand[have + before] = key_of(x, (int)i);
      have += min(all, k - have);
    }
    n = max(n, have);
    __syncthreads();
  }
  // ---- fewer candidates, by their (unlike) keys ----
  uint64_t least = 0;
  if (n > kLpThreads) {
    uint64_t low = 0, high = ~0ull;  // low is reached by k or more, high by fewer
    while (high - low > 1) {
      const uint64_t mid = low + (high - low) / 2;
      int c = 0;
      for (int i = tid; i < n; i += kLpThreads) c += cand[i] >= mid;
      c = block_count(c, counts);
      if (c >= k) {
        low = mid;
        if (c <= kLpThreads) break;
      } else {
        high = mid;
      }
    }
    least = low;
  }
  // ---- a candidate's place is the number of larger ones ----
  for (int i = tid; i < n; i += kLpThreads) {
    const uint64_t key = cand[i];
    if (key < least) continue;
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > key;
    if (rank < k) {
      const int at = (int)~(uint32_t)key;
      a.top_ids[r * k + rank] = at;
      a.top_logprobs[r * k + rank] = (logit_at<DT>(row, at) - m) - log_s;
    }
  }
}

int chunks_of(int vocab) { return (int)(((int64_t)vocab + 7 + kChunk - 1) / kChunk); }

template <int DT>
int launch_logprobs(const LpArgs& a, hipStream_t s) {
  const int64_t y = a.rows < 32768 ? a.rows : 32768;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_chunk_kernel<DT>),
                     dim3(a.chunks, (unsigned)y, (unsigned)((a.rows + 32767) / 32768)), dim3(kLpThreads), 0, s, a);
  if (hipError_t e = hipGetLastError()) return (int)e;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_row_kernel<DT>), dim3((unsigned)a.rows), dim3(kLpThreads), 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_token_logprobs_workspace_size(int64_t rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0) return 0;
  return (size_t)rows * chunks_of(vocab) * (4 + (top > 0 ? kLpThreads : 0)) * sizeof(float);
}

extern "C" int mkv_token_logprobs(float* logprobs, float* entropy, float* top_logprobs, int64_t* top_ids,
                                  const void* logits, int64_t row_stride, int dtype, int64_t rows, int vocab,
                                  const void* ids, int64_t ids_stride, int num_ids, int ids_dtype, int top,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  if (rows < 0 || rows > 0x3fffffff || vocab <= 0 || vocab > 0x7ffffff0 || num_ids < 0 || top < 0 || top > kMaxTop ||
      top > vocab)
    return MKV_ERR_BAD_SHAPE;
  if (rows == 0) return MKV_OK;
  if (!logits || !entropy || (num_ids && (!ids || !logprobs)) || (top && (!top_logprobs || !top_ids)) || !workspace)
    return MKV_ERR_NULL_POINTER;
  if (num_ids && ids_dtype != MKV_INDEX_I32 && ids_dtype != MKV_INDEX_I64) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (row_stride < vocab || (num_ids && ids_stride < num_ids)) return MKV_ERR_BAD_STRIDE;
  const int size = dtype == MKV_DTYPE_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % size || reinterpret_cast<uintptr_t>(workspace) & 15) return MKV_ERR_MISALIGNED;
  if (workspace_bytes < mkv_token_logprobs_workspace_size(rows, vocab, top)) return MKV_ERR_WORKSPACE_TOO_SMALL;
  LpArgs a;
  a.logits = logits;
  a.row_stride = row_stride;
  a.rows = rows;
  a.vocab = vocab;
  a.chunks = chunks_of(vocab);
  a.ids = ids;
  a.ids_i64 = ids_dtype == MKV_INDEX_I64;
  a.num_ids = num_ids;
  a.ids_stride = ids_stride;
  a.top = top;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_logprobs = top_logprobs;
  a.top_ids = top_ids;
  a.stats = reinterpret_cast<float*>(workspace);
  a.maxima = a.stats + (size_t)rows * a.chunks * 4;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case MKV_DTYPE_F32: return launch_logprobs<MKV_DTYPE_F32>(a, s);
    case MKV_DTYPE_BF16: return launch_logprobs<MKV_DTYPE_BF16>(a, s);
    case MKV_DTYPE_F16: return launch_logprobs<MKV_DTYPE_F16>(a, s);
    default: return MKV_ERR_UNSUPPORTED_DTYPE;
  }
}
