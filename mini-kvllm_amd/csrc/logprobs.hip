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
// thread's 32 logits as a key in unsigned order (16 bits for 16-bit logits).
// Pass 2, one workgroup a row, joins the chunks and finds the top k from those
// maxima, held in registers: a value that at least k of them reach bounds the k-th
// largest logit from below, so only the threads' logits that reach it are read
// again (a few dozen of the vocabulary).  Selecting in pass 1 would cost
// its workgroups as many VALU cycles again as the whole softmax.
//
// A vocabulary that one workgroup holds (up to 8185) takes one launch: a workgroup
// a row, one wave where 2041 logits or fewer leave no work for four (4096 rows of 2000
// bf16 logits, top 64: 19 us against 59 in two launches; 8 or 16 waves a row for
// larger vocabularies were slower than two launches at any number of rows).
#include <type_traits>

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
  void* maxima;        // workspace: (rows, chunks, 256) keys, each row 16-byte aligned
};

// A workgroup a row: rows past a grid's first dimension (below 2^32 threads) go on in
// the second.
constexpr int64_t kGridRows = (int64_t)1 << 22;
MKV_DEV int64_t row_of_grid() { return blockIdx.x + blockIdx.y * kGridRows; }
inline dim3 grid_of_rows(int64_t rows) {
  return dim3((unsigned)(rows < kGridRows ? rows : kGridRows), (unsigned)((rows + kGridRows - 1) / kGridRows));
}

// max that a NaN on either side wins (v_maximum3_f32)
MKV_DEV float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Unsigned order of logits: NaN above +inf, the two zeros alike; 0 for none.  A
// 16-bit logit's order is the upper half of it (fp16's by its own bits).
MKV_DEV uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
  const uint32_t o = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : o;
}
MKV_DEV float value_of(uint32_t order) {
  return __uint_as_float(order >> 31 ? order & 0x7fffffffu : ~order);  // (~0: a NaN)
}
MKV_DEV uint64_t key_of(float x, int i) { return (uint64_t)order_of(x) << 32 | (uint32_t)~i; }

// Sums and maxima over the wave by DPP moves and lane swaps (no LDS round trips).
template <class F>
MKV_DEV float wave_all(float x, F f) {
  // (x as it is rounded: a product fused into the first sum would differ from
  // lane to lane)
  asm volatile("" : "+v"(x));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xf, 0xf, false)));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xf, 0xf, false)));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xf, 0xf, false)));
  x = f(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xf, 0xf, false)));
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
MKV_DEV float wave_sum(float x) {
  return wave_all(x, [](float a, float b) { return a + b; });
}
MKV_DEV float wave_max(float x) {
  return wave_all(x, [](float a, float b) { return maximum(a, b); });
}

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
  using Key = typename std::conditional<DT == MKV_DTYPE_F32, uint32_t, uint16_t>::type;
  // a logit's key: its order, for 16-bit logits in 16 bits
  MKV_DEV static uint32_t key(float x) {
    if constexpr (DT == MKV_DTYPE_F32) return order_of(x);
    if constexpr (DT == MKV_DTYPE_BF16) return order_of(x) >> 16;
    const uint32_t u = f32_to_f16_bits(x == 0.0f ? 0.0f : x);  // (exact)
    return x != x ? 0xffffu : (u & 0x8000u ? ~u : u | 0x8000u) & 0xffffu;
  }
  static constexpr int kVec = DT == MKV_DTYPE_F32 ? 4 : 8;
  static constexpr int kNum = kPer / kVec;
  template <int T>
  MKV_DEV static int64_t start_of(int j, int tid, int shift) {  // one chunk, of T threads
    return (j * T + tid) * kVec - shift;
  }
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
  if (a.top) {
    // (a thread without a logit of the row: 0)
    const bool none = P::start(chunk, 0, tid, shift) >= a.vocab;
    reinterpret_cast<typename P::Key*>(a.maxima)[(r * a.chunks + chunk) * kLpThreads + tid] =
        (typename P::Key)(none ? 0u : P::key(own));
  }
  const float m = wave_max(own);
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
  w.s = wave_sum(w.s);
  w.t = wave_sum(w.t);
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

// The row's keys, 16 bytes a thread at a time: up to kHeld vectors in registers
// (16-bit logits: vocabularies up to 262144; fp32: 131072), the rest from memory.
template <int DT>
struct Keys {
  using P = Pieces<DT>;
  static constexpr int kPerVec = 16 / sizeof(typename P::Key);
  static constexpr int kHeld = DT == MKV_DTYPE_F32 ? 16 : 4;
  const u32x4* src;
  int vecs;
  u32x4 held[kHeld];

  MKV_DEV static uint32_t get(const u32x4& v, int e) {
    if constexpr (DT == MKV_DTYPE_F32) return v[e];
    return e & 1 ? v[e >> 1] >> 16 : v[e >> 1] & 0xffffu;
  }
  MKV_DEV void load(const void* p, int num) {
    src = reinterpret_cast<const u32x4*>(p);
    vecs = num / kPerVec;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      const int at = j * kLpThreads + (int)threadIdx.x;
      held[j] = u32x4{0, 0, 0, 0};
      if (at < vecs) held[j] = src[at];
    }
  }
  // f(key, number of the share)
  template <class F>
  MKV_DEV void each(F f) const {
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
      if (j * kLpThreads >= vecs) break;
#pragma unroll
      for (int e = 0; e < kPerVec; ++e) f(get(held[j], e), (j * kLpThreads + (int)threadIdx.x) * kPerVec + e);
    }
    for (int at = kHeld * kLpThreads + (int)threadIdx.x; at - (int)threadIdx.x < vecs; at += kLpThreads) {
      const u32x4 v = at < vecs ? src[at] : u32x4{0, 0, 0, 0};
#pragma unroll
      for (int e = 0; e < kPerVec; ++e) f(get(v, e), at * kPerVec + e);
    }
  }
};

// Every thread's two keys, 2 W a lane, in every wave.
template <int W>
MKV_DEV void threads_bests(uint32_t a, uint32_t b, uint32_t (&bests)[2 * W]) {
  if constexpr (W > 1) {
    __shared__ uint32_t all[2][64 * W];
    all[0][threadIdx.x] = a;
    all[1][threadIdx.x] = b;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 2 * W; ++v) bests[v] = all[v / W][v % W * 64 + (threadIdx.x & 63)];
  } else {
    bests[0] = a;
    bests[1] = b;
  }
}
// Of these keys, one that k reach: the k-th largest or less, found a bit at a time
// by each wave for itself, without a barrier; 0 where fewer than k are above 0.
template <int BITS, int N>
MKV_DEV uint32_t kth_best(const uint32_t (&bests)[N], int k) {
  uint32_t least = 0;
  for (int bit = BITS - 1; bit >= 0; --bit) {
    const uint32_t mid = least | 1u << bit;
    int n = 0;
#pragma unroll
    for (int v = 0; v < N; ++v) n += __popcll(__builtin_amdgcn_ballot_w64(bests[v] >= mid));
    if (n >= k) least = mid;
    if (n == k) break;
  }
  return least;
}
// ... of the threads' keys, the larger of each thread's two where these are many
// enough: k of 64 W leave few logits above the bound (1024 rows of 151936, top 20:
// 70 us against 74; 4096 rows of 2000, top 64 the other way: 27 against 19).
template <int BITS, int N>
MKV_DEV uint32_t bound(const uint32_t (&bests)[N], int k) {
  if (k > 32) return kth_best<BITS>(bests, k);
  uint32_t larger[N / 2];
#pragma unroll
  for (int v = 0; v < N / 2; ++v) larger[v] = max(bests[v], bests[v + N / 2]);
  return kth_best<BITS>(larger, k);
}
template <int N>
MKV_DEV uint32_t largest(const uint32_t (&bests)[N]) {
  uint32_t hi = 0;
#pragma unroll
  for (int v = 0; v < N; ++v) hi = max(hi, bests[v]);
#pragma unroll
  for (int o = 32; o; o >>= 1) hi = max(hi, (uint32_t)__shfl_xor((int)hi, o));
  return hi;
}

template <int DT>
__global__ __launch_bounds__(kLpThreads) void logprobs_row_kernel(LpArgs a) {
  using P = Pieces<DT>;
  constexpr int kWaves = kLpThreads / 64;
  __shared__ uint32_t counts[2][kWaves];
  __shared__ uint64_t cand[kMaxCand];
  __shared__ int subs[kMaxSub];
  __shared__ int fill[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = row_of_grid();
  if (r >= a.rows) return;
  const char* row = reinterpret_cast<const char*>(a.logits) + r * a.row_stride * (16 / P::kVec);
  // the given tokens' logits and the keys go out first
  float given = 0.0f;
  int64_t id = -1;
  if (tid < a.num_ids) {
    id = load_index(a.ids, r * a.ids_stride + tid, a.ids_i64);
    if (id >= 0 && id < a.vocab) given = logit_at<DT>(row, id);
  }
  const int shares = a.chunks * kLpThreads;
  Keys<DT> keys;
  if (a.top) keys.load(reinterpret_cast<const typename P::Key*>(a.maxima) + r * shares, shares);
  if (tid < 2) fill[tid] = 0;
  // the chunks' sums, in every wave: a lane a chunk
  float m = -__builtin_huge_valf(), s = 0.0f, t = 0.0f;
  for (int c0 = 0; c0 < a.chunks; c0 += 64) {
    Stat st{-__builtin_huge_valf(), 0.0f, 0.0f};
    if (c0 + lane < a.chunks) {
      const u32x4 v = ld16(a.stats + (r * a.chunks + c0 + lane) * 4);
      st = Stat{__uint_as_float(v[0]), __uint_as_float(v[1]), __uint_as_float(v[2])};
    }
    const float top = maximum(m, wave_max(st.m));
    // equal maxima need no factor (and equal infinities have no difference)
    const float d = st.m == top ? 0.0f : st.m - top, f = expf(d);
    const float d0 = m == top ? 0.0f : m - top, f0 = expf(d0);
    const float tn = wave_sum(f > 0.0f ? f * (st.t + st.s * d) : 0.0f);
    t = (f0 > 0.0f ? f0 * (t + s * d0) : 0.0f) + tn;
    s = s * f0 + wave_sum(st.s * f);
    m = top;
  }
  if (m != m) s = t = m;
  const float log_s = logf(s);
  if (tid == 0) a.entropy[r] = log_s - t / s;
  for (int i = tid; i < a.num_ids; i += kLpThreads) {
    if (i >= kLpThreads) {
      id = load_index(a.ids, r * a.ids_stride + i, a.ids_i64);
      if (id >= 0 && id < a.vocab) given = logit_at<DT>(row, id);
    }
    a.logprobs[r * a.num_ids + i] = id < 0 ? 0.0f : id < a.vocab ? (given - m) - log_s : __builtin_nanf("");
  }
  if (a.top == 0) return;

  // ---- a threshold that k to kMaxSub shares' maxima reach ----
  const int k = a.top;
  const int shift = P::shift(row);
  int turn = 0;
  // the workgroup's sum of a count that each wave has in a scalar
  auto all = [&](uint32_t wave_count) -> int {
    if (lane == 0) counts[turn][wave] = wave_count;
    __syncthreads();
    uint32_t n = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) n += counts[turn][w];
    turn ^= 1;  // (the other half is free again: everyone has passed a barrier since)
    return (int)n;
  };
  auto reach = [&](uint32_t least) -> int {
    uint32_t n = 0;
    keys.each([&](uint32_t key, int) { n += __popcll(__builtin_amdgcn_ballot_w64(key >= least)); });
    return all(n);
  };
  // a bound of k shares, from the largest of the threads' even and odd ones
  uint32_t own[2] = {0, 0};
  keys.each([&](uint32_t key, int share) { own[share & 1] = max(own[share & 1], key); });
  uint32_t bests[2 * kWaves];
  threads_bests<kWaves>(own[0], own[1], bests);
  uint32_t lo = max(bound<8 * sizeof(typename P::Key)>(bests, k), 1u);  // (0: few threads have a share)
  int n_sub = reach(lo);
  if (n_sub > kMaxSub) {
    uint32_t hi = largest(bests);
    const int n_hi = reach(hi);
    if (n_hi >= k) {
      lo = hi;
      n_sub = n_hi;
    }
    // reach(lo) > kMaxSub, reach(hi) < k
    while (n_sub > kMaxSub && hi - lo > 1) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const int n = reach(mid);
      if (n >= k) {
        lo = mid;
        n_sub = n;
      } else {
        hi = mid;
      }
    }
  }
  // many shares with one largest logit, lo: the logits above it, then the first
  // that equal it, in the order of their places
  const bool ties = n_sub > kMaxSub;
  const uint32_t from = ties ? lo + 1 : lo;  // (32-bit keys: 0 past the last)
  if (from) {
    keys.each([&](uint32_t key, int share) {
      if (key >= from) {
        const int at = atomicAdd(&fill[0], 1);
        if (at < kMaxSub) subs[at] = share;
      }
    });
  }
  __syncthreads();
  const int num_sub = min(fill[0], kMaxSub);
  for (int w = tid; w < num_sub * P::kNum; w += kLpThreads) {
    const int i = subs[w / P::kNum];
    const int64_t at = P::start(i / kLpThreads, w % P::kNum, i % kLpThreads, shift);
    float x[P::kVec];
    P::load(row, at, a.vocab, x);
#pragma unroll
    for (int e = 0; e < P::kVec; ++e)
      if (at + e >= 0 && at + e < a.vocab && P::key(x[e]) >= from) {
        const int c = atomicAdd(&fill[1], 1);
        if (c < kMaxCand) cand[c] = key_of(x[e], (int)(at + e));
      }
  }
  __syncthreads();
  int n = min(fill[1], kMaxCand);
  if (ties) {
    // fewer than k may lie above
    int have = n;
    for (int64_t base = 0; base < a.vocab && have < k; base += kLpThreads) {
      const int64_t i = base + tid;
      const float x = i < a.vocab ? logit_at<DT>(row, i) : 0.0f;
      const bool hit = i < a.vocab && P::key(x) == lo;
      const uint64_t ball = __builtin_amdgcn_ballot_w64(hit);
      if (lane == 0) counts[turn][wave] = (uint32_t)__popcll(ball);
      __syncthreads();
      int before = __popcll(ball & ((1ull << lane) - 1)), found = 0;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += (int)counts[turn][w];
        found += (int)counts[turn][w];
      }
      turn ^= 1;
      if (hit && have + before < k) cand[have + before] = key_of(x, (int)i);
      have += min(found, k - have);
    }
    n = max(n, have);
    __syncthreads();
  }
  // ---- fewer candidates, by their (unlike) keys ----
  uint64_t least = 0;
  if (n > kLpThreads) {
    uint64_t low = 0, high = ~0ull;  // k or more reach low
    while (high - low > 1) {
      const uint64_t mid = low + (high - low) / 2;
      uint32_t c = 0;
      for (int i0 = 0; i0 < n; i0 += kLpThreads)
        c += __popcll(__builtin_amdgcn_ballot_w64(i0 + tid < n && cand[i0 + tid] >= mid));
      const int reached = all(c);
      if (reached >= k) {
        low = mid;
        if (reached <= kLpThreads) break;
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
      a.top_ids[r * k + rank] = (int)~(uint32_t)key;
      a.top_logprobs[r * k + rank] = (value_of((uint32_t)(key >> 32)) - m) - log_s;
    }
  }
}

// Rows that a workgroup of W waves holds, PER logits a thread.
constexpr int kFew = 256;  // candidates that are ranked against each other
template <int DT, int W, int PER>
__global__ __launch_bounds__(64 * W) void logprobs_whole_kernel(LpArgs a) {
  using P = Pieces<DT>;
  constexpr int T = 64 * W, kPieces = PER / P::kVec;
  __shared__ Stat part[W];
  __shared__ uint32_t counts[2][W];
  __shared__ uint64_t cand[kFew];
  __shared__ int fill;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t r = row_of_grid();
  if (r >= a.rows) return;
  const char* row = reinterpret_cast<const char*>(a.logits) + r * a.row_stride * (16 / P::kVec);
  const int shift = P::shift(row);
  float given = 0.0f;
  int64_t id = -1;
  if (tid < a.num_ids) {
    id = load_index(a.ids, r * a.ids_stride + tid, a.ids_i64);
    if (id >= 0 && id < a.vocab) given = logit_at<DT>(row, id);
  }
  float x[PER];
#pragma unroll
  for (int j = 0; j < kPieces; ++j) P::load(row, P::template start_of<T>(j, tid, shift), a.vocab, x + j * P::kVec);
  if (tid == 0) fill = 0;
  float own = x[0];
#pragma unroll
  for (int i = 1; i < PER; ++i) own = maximum(own, x[i]);
  Stat w{wave_max(own), 0.0f, 0.0f};  // as in the first pass
  if (w.m != -__builtin_huge_valf()) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const float d = maximum(x[i] - w.m, -200.0f);
      const float e = __builtin_amdgcn_exp2f(d * kLog2e);
      w.s += e;
      w.t = __builtin_fmaf(e, d, w.t);
    }
  }
  w.s = wave_sum(w.s);
  w.t = wave_sum(w.t);
  if constexpr (W > 1) {
    if (lane == 0) part[wave] = w;
    __syncthreads();
    w = part[0];
#pragma unroll
    for (int i = 1; i < W; ++i) w = join(w, part[i]);
  }
  const float m = w.m, s = m != m ? m : w.s, t = m != m ? m : w.t;
  const float log_s = logf(s);
  if (tid == 0) a.entropy[r] = log_s - t / s;
  for (int i = tid; i < a.num_ids; i += T) {
    if (i >= T) {
      id = load_index(a.ids, r * a.ids_stride + i, a.ids_i64);
      if (id >= 0 && id < a.vocab) given = logit_at<DT>(row, id);
    }
    a.logprobs[r * a.num_ids + i] = id < 0 ? 0.0f : id < a.vocab ? (given - m) - log_s : __builtin_nanf("");
  }
  if (a.top == 0) return;

  const int k = a.top;
  uint32_t key[PER], best[2] = {0, 0};  // (0: outside the row)
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int64_t at = P::template start_of<T>(i / P::kVec, tid, shift) + i % P::kVec;
    key[i] = at >= 0 && at < a.vocab ? P::key(x[i]) : 0u;
    best[i >= PER / 2] = max(best[i >= PER / 2], key[i]);
  }
  int turn = 0;
  auto total = [&](uint32_t n) -> int {  // over the waves
    if constexpr (W > 1) {
      if (lane == 0) counts[turn][wave] = n;
      __syncthreads();
      n = 0;
#pragma unroll
      for (int v = 0; v < W; ++v) n += counts[turn][v];
      turn ^= 1;  // (the other half is free again: everyone has passed a barrier since)
    }
    return (int)n;
  };
  // the number of the workgroup's keys that reach `from`
  auto reach = [&](uint32_t from) -> int {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      n += __popcll(__builtin_amdgcn_ballot_w64(key[i] >= from));
      asm volatile("" : "+s"(n));  // (one ballot's registers at a time)
    }
    return total(n);
  };
  // ---- a bound that k logits reach, from the largest of the threads' halves ----
  uint32_t bests[2 * W];
  threads_bests<W>(best[0], best[1], bests);
  uint32_t lo = max(bound<8 * sizeof(typename P::Key)>(bests, k), 1u);
  uint32_t chosen = 0;  // a bit a logit
#pragma unroll
  for (int i = 0; i < PER; ++i) chosen |= (uint32_t)(key[i] >= lo) << i;
  auto sum = [&](uint32_t bits) { return total((uint32_t)wave_sum((float)__popc(bits))); };
  int n = sum(chosen);
  auto place = [&](int i) { return (int)P::template start_of<T>(i / P::kVec, tid, shift) + i % P::kVec; };
  if (n > kFew) {
    // ---- many (equal ones, or few threads with logits): exactly k, by the k-th
    // largest of all keys, lo ----
    uint32_t hi = largest(bests);
    const int n_hi = reach(hi);
    if (n_hi >= k) {
      lo = hi;
      n = n_hi;
    }
    while (n > k && hi - lo > 1) {  // n reach lo, fewer than k reach hi
      const uint32_t mid = lo + (hi - lo) / 2;
      const int n_mid = reach(mid);
      if (n_mid >= k) {
        lo = mid;
        n = n_mid;
      } else {
        hi = mid;
      }
    }
    uint32_t above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      above |= (uint32_t)(key[i] > lo) << i;
      equal |= (uint32_t)(key[i] == lo) << i;
    }
    if (n > k) {
      // the first of the equal logits: those below place `end` (a thread's places
      // rise with i)
      auto below = [&](int end) {
        int c = 0;
#pragma unroll
        for (int j = 0; j < kPieces; ++j) c += min(max(end - place(j * P::kVec), 0), P::kVec);
        return equal & (uint32_t)((1ull << c) - 1);
      };
      const int need = k - sum(above);
      int begin = 0, end = a.vocab;  // fewer than need below begin, need or more below end
      while (end - begin > 1) {
        const int mid = begin + (end - begin) / 2;
        const int c = sum(below(mid));
        if (c >= need) end = mid;
        else begin = mid;
        if (c == need) break;
      }
      equal = below(end);
    }
    chosen = above | equal;
    n = k;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PER; ++i)
    if (chosen >> i & 1) {
      const int at = atomicAdd(&fill, 1);
      if (at < kFew) cand[at] = (uint64_t)place(i);
    }
  __syncthreads();
  // a candidate's place is the number of larger ones (its logit comes from the row
  // again: the logits' registers hold the keys since)
  for (int i = tid; i < n; i += T) cand[i] = key_of(logit_at<DT>(row, (int64_t)cand[i]), (int)cand[i]);
  __syncthreads();
  for (int i = tid; i < n; i += T) {
    const uint64_t mine = cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > mine;
    if (rank < k) {
      a.top_ids[r * k + rank] = (int)~(uint32_t)mine;
      a.top_logprobs[r * k + rank] = (value_of((uint32_t)(mine >> 32)) - m) - log_s;
    }
  }
}

int chunks_of(int vocab) { return (int)(((int64_t)vocab + 7 + kChunk - 1) / kChunk); }

template <int DT>
int launch_logprobs(const LpArgs& a, hipStream_t s) {
  if (a.chunks == 1) {
    const int64_t held = a.vocab + 7;  // (a row's start may leave 7 places empty)
    auto whole = [&](auto w, auto per) {
      constexpr int W = decltype(w)::value, kPerThread = decltype(per)::value;
      hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_whole_kernel<DT, W, kPerThread>), grid_of_rows(a.rows), dim3(64 * W), 0, s, a);
      return (int)hipGetLastError();
    };
    using I1 = std::integral_constant<int, 1>;
    using I4 = std::integral_constant<int, 4>;
    if (held <= 64 * 8) return whole(I1{}, std::integral_constant<int, 8>{});
    if (held <= 64 * kPer) return whole(I1{}, std::integral_constant<int, kPer>{});
    return whole(I4{}, std::integral_constant<int, kPer>{});
  }
  const int64_t y = a.rows < 32768 ? a.rows : 32768;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_chunk_kernel<DT>),
                     dim3(a.chunks, (unsigned)y, (unsigned)((a.rows + 32767) / 32768)), dim3(kLpThreads), 0, s, a);
  if (hipError_t e = hipGetLastError()) return (int)e;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(logprobs_row_kernel<DT>), grid_of_rows(a.rows), dim3(kLpThreads), 0, s, a);
  return (int)hipGetLastError();
}

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_token_logprobs_workspace_size(int64_t rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0) return 0;
  if (chunks_of(vocab) == 1) return 256;  // (not used: one launch)
  // (4 bytes a key: enough for every type)
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
