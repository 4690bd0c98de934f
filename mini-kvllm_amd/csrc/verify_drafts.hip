// Verification of drafted tokens against the target's distribution from given
// random numbers: the accepting half of speculative sampling, over chains and
// trees.
//
// At a node of the tree, p = softmax(logits / T) of its row; its children are
// tokens drawn from q = softmax(draft logits / T) of the same row, or given without
// a distribution (q one at the token).  In their order
//
//   child x is taken if u q(x) < p(x), else p <- max(0, p - q) / sum of it
//
// and the walk goes on at the child taken; where none is, the next token is
// argmax_v p(v) / E(v), E given exponential variates: a sample of what is left.
//
// After r rejections p is max(0, a p - b q) with two scalars (a stays 0 once it is:
// the recurrence is linear where it is positive), so no row is ever written, and a
// test is u < a ratio - b with ratio = p(x) / q(x).
//
// Read bound: the logits' rows, once, for their maxima and sums
// (verify_stats_kernel); the walk reads a few words a node (verify_walk_kernel, a
// workgroup a sequence), and the last row, its draft's and E are read once more
// (verify_draw_kernel; the walk's own for up to 8192 logits).  Only siblings of a
// rejected token in a tree with draft distributions cost more: each a pass over the two
// rows, by the sequence's one workgroup, for the sum of what is left (16 trees of 21
// nodes, four children each, over 151,936 bf16 logits: rows 30 us, walk 103, draw 10).
// 60 chains of 9 nodes over 151,936 bf16 logits and the draft's: 65 us (4.8 TB/s), 10 and
// 16.5; one chain of 5: 5, 6.5 and 8, latency.
// Sums are fp32 within a workgroup's 8192 logits.
#include <type_traits>

#include "mkv_device.hpp"

namespace mkv {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 32;                   // logits a thread holds
constexpr int kChunk = kThreads * kPer;    // 8192
constexpr int kWalkThreads = 1024;
constexpr int kMaxNodes = 1024;   // of a sequence
constexpr float kNegInf = -__builtin_huge_valf();

struct VerifyArgs {
  const char* logits;
  const char* draft;  // NULL: drafts without a distribution
  int64_t row_stride, draft_stride;  // elements
  int64_t total;
  int vocab, chunks;
  int group;          // lanes of the walk that join a row's chunks: a power of two
  const void* ids;
  const void* parents;  // NULL: chains
  int ids_i64, parents_i64;
  const int32_t* cu;
  int num_seqs;
  const float* uniforms;
  const float* noise;
  int64_t noise_stride;
  const float* temperatures;  // NULL: 1
  int max_nodes;
  int64_t* accepted;
  int64_t* num_accepted;
  int64_t* next;
  float* acceptance;
  f32x4* stats;   // workspace: (1 or 2) x (total, chunks): maximum, sum, the maximum's place
  struct DrawState* state;  // workspace: (num_seqs)
  int32_t* barred;          // workspace: (num_seqs, max_nodes) tokens that the draw leaves out
};

// What the draw needs of the walk's end.
struct DrawState {
  unsigned long long best;  // the race's leader: (what is left first, value, ~place)
  unsigned int arrived;     // workgroups that are done
  int draws;                // 0: the walk has the token already
  int64_t row;              // of logits
  float c;                  // log2(e) / T
  float p_max, p_mul;       // a / sum
  float q_max, q_mul;       // b / sum, 0: p alone
  int barred;               // tokens left out
};

MKV_DEV float maximum(float a, float b) { return __builtin_elementwise_maximum(a, b); }  // (NaN wins)

template <class X, class F>
MKV_DEV X wave_all(X x, F f) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x = f(x, __shfl_xor(x, o));
  return x;
}
MKV_DEV float wave_max(float x) { return wave_all(x, [](float a, float b) { return maximum(a, b); }); }
MKV_DEV float wave_sum(float x) { return wave_all(x, [](float a, float b) { return a + b; }); }

template <int DT>
constexpr int kSize = DTypeInfo<DT>::kBytes;

template <int DT>
MKV_DEV float element(const char* row, int64_t i) {
  if constexpr (DT == MKV_DTYPE_F32) return reinterpret_cast<const float*>(row)[i];
  const uint32_t b = reinterpret_cast<const uint16_t*>(row)[i];
  return DT == MKV_DTYPE_BF16 ? bf16_bits_to_f32(b) : f16_bits_to_f32(b);
}

// 16 bytes of a row from element i on (rows start anywhere: the load need not be
// aligned); -inf past its end.
template <int DT>
struct Piece {
  static constexpr int kVec = 16 / kSize<DT>;
  MKV_DEV static void load(const char* row, int64_t i, int vocab, float* x) {
    if (i + kVec <= vocab) {
      u32x4 w;
      __builtin_memcpy(&w, row + i * kSize<DT>, 16);
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
      for (int e = 0; e < kVec; ++e) x[e] = i + e < vocab ? element<DT>(row, i + e) : kNegInf;
    }
  }
};

// A sequence's rows, cut to what the call covers.
struct Nodes {
  int64_t first;
  int n;
};
MKV_DEV Nodes nodes_of(const VerifyArgs& a, int s) {
  const int64_t q0 = min(max((int64_t)a.cu[s], (int64_t)0), a.total);
  const int64_t q1 = min(max((int64_t)a.cu[s + 1], q0), a.total);
  return Nodes{q0, (int)min(q1 - q0, (int64_t)a.max_nodes)};
}
// log2(e) / T, above 0 (an infinite T: all alike but -inf); 0: greedy
MKV_DEV float slope_of(const VerifyArgs& a, int s) {
  const float t = a.temperatures ? a.temperatures[s] : 1.0f;
  return t > 1e-30f ? fmaxf(kLog2e / t, 1e-36f) : 0.0f;
}
MKV_DEV bool finite(float x) { return fabsf(x) < __builtin_huge_valf(); }
// e^((x - m) / T): 0 for -inf (m is finite, c above 0)
MKV_DEV float weight(float x, float m, float c) { return __builtin_amdgcn_exp2f((x - m) * c); }

template <int DT>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(VerifyArgs a) {
  using P = Piece<DT>;
  const int chunk = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  int64_t r = blockIdx.y + (int64_t)blockIdx.z * 32768;
  if (r >= a.total * (a.draft ? 2 : 1)) return;
  const bool draft = r >= a.total;
  const int64_t at = r;
  r -= draft ? a.total : 0;
  // the row's sequence: as many end at or ahead of it
  int seq = 0;
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    const int s = s0 + lane;
    seq += __popcll(__builtin_amdgcn_ballot_w64(s < a.num_seqs && a.cu[s + 1] <= r));
  }
  if (seq >= a.num_seqs) return;
  const Nodes nodes = nodes_of(a, seq);
  const int64_t node = r - nodes.first;
  if (node < 0 || node >= nodes.n) return;
  const float c = slope_of(a, seq);
  if (draft) {  // rows without children, and greedy sequences', are not looked at
    if (c == 0.0f) return;
    bool parent = false;
    if (a.parents) {
      for (int j = (int)node + 1 + tid; j < nodes.n; j += kThreads)
        parent |= load_index(a.parents, nodes.first + j, a.parents_i64) == node;
      parent = __syncthreads_or(parent);
    } else {
      parent = node + 1 < nodes.n;
    }
    if (!parent) return;
  }
  const char* row = draft ? a.draft + r * a.draft_stride * kSize<DT> : a.logits + r * a.row_stride * kSize<DT>;
  float x[kPer];
#pragma unroll
  for (int j = 0; j < kPer / P::kVec; ++j)
    P::load(row, (int64_t)chunk * kChunk + (j * kThreads + tid) * P::kVec, a.vocab, x + j * P::kVec);
  float m = x[0];
#pragma unroll
  for (int i = 1; i < kPer; ++i) m = maximum(m, x[i]);
  __shared__ float part_m[kThreads / 64], part_s[kThreads / 64];
  __shared__ int part_i[kThreads / 64];
  m = wave_max(m);
  if (lane == 0) part_m[tid >> 6] = m;
  __syncthreads();
  m = part_m[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) m = maximum(m, part_m[w]);
  float s = 0.0f;
  int place = 0x7fffffff;
  if (c == 0.0f || !finite(m)) {
    // the first of the largest (a NaN is larger than all)
#pragma unroll
    for (int i = kPer - 1; i >= 0; --i) {
      const int p = chunk * kChunk + ((i / P::kVec) * kThreads + tid) * P::kVec + i % P::kVec;
      if (p < a.vocab && (x[i] == m || x[i] != x[i])) place = p;
    }
    place = wave_all(place, [](int u, int v) { return min(u, v); });
  }
  if (c != 0.0f && finite(m)) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += weight(x[i], m, c);
    s = wave_sum(s);
  }
  if (lane == 0) {
    part_s[tid >> 6] = s;
    part_i[tid >> 6] = place;
  }
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) {
      s += part_s[w];
      place = min(place, part_i[w]);
    }
    a.stats[at * a.chunks + chunk] = f32x4{m, s, __int_as_float(place), 0.0f};
  }
}

// Maximum, sum and the maximum's place of two parts of a row (a NaN is the largest).
MKV_DEV void join(float& m, float& s, int& place, float m2, float s2, int place2, float c) {
  const float top = maximum(m, m2);
  const bool first = m == top || m != m, second = m2 == top || m2 != m2;
  place = min(first ? place : 0x7fffffff, second ? place2 : 0x7fffffff);
  // (a sum without a finite maximum is not looked at)
  s = (m == top ? s : s * weight(m, top, c)) + (m2 == top ? s2 : s2 * weight(m2, top, c));
  m = top;
}

// A node in LDS.
struct Node {
  float m, s;      // of its row: maximum and sum
  float qm, qs;    // of its draft row
  int place;       // of the maximum, where greedy (or not finite): else -1
  int parent;
  int token;       // -1: outside the vocabulary
  float u;
  float ratio;     // p / q of its token in its parent's row
};

// The sum of what is left of p, by the whole workgroup.
template <int DT>
MKV_DEV double left_over(const VerifyArgs& a, int64_t row, float c, float pm, float pf, float qm, float qf, double* lds) {
  using P = Piece<DT>;
  const char* p = a.logits + row * a.row_stride * kSize<DT>;
  const char* q = a.draft + row * a.draft_stride * kSize<DT>;
  double sum = 0.0;
  for (int64_t i = (int64_t)threadIdx.x * P::kVec; i < a.vocab; i += kWalkThreads * P::kVec) {
    float x[P::kVec], y[P::kVec], part = 0.0f;
    P::load(p, i, a.vocab, x);
    P::load(q, i, a.vocab, y);
#pragma unroll
    for (int e = 0; e < P::kVec; ++e) part += fmaxf(pf * weight(x[e], pm, c) - qf * weight(y[e], qm, c), 0.0f);
    sum += part;
  }
  sum = wave_all(sum, [](double u, double v) { return u + v; });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < kWalkThreads / 64; ++w) sum += lds[w];
  return sum;
}

// The race p / E over what is left of p in a chunk (over p itself where rounding leaves
// nothing): the leader's value and place, by the whole workgroup.
// out: a bit a logit that is left out.
template <int DT, int THREADS>
MKV_DEV unsigned long long race(const VerifyArgs& a, const DrawState& st, int seq, int chunk, const uint32_t* out,
                                unsigned long long (*part)[THREADS / 64]) {
  using P = Piece<DT>;
  using N = Piece<MKV_DTYPE_F32>;
  const int tid = threadIdx.x;
  const char* prow = a.logits + st.row * a.row_stride * kSize<DT>;
  const char* qrow = a.draft + (a.draft ? st.row * a.draft_stride * kSize<DT> : 0);
  const char* nrow = reinterpret_cast<const char*>(a.noise + seq * a.noise_stride);
  auto run = [&](bool fallback) -> unsigned long long {
    float best = 0.0f;
    int at_best = 0;
#pragma unroll
    for (int j = 0; j < kChunk / THREADS / P::kVec; ++j) {
      const int at = (j * THREADS + tid) * P::kVec;
      const int64_t i = (int64_t)chunk * kChunk + at;
      if (i >= a.vocab) continue;
      float x[P::kVec], y[P::kVec], e[P::kVec];
      P::load(prow, i, a.vocab, x);
      if (st.q_mul > 0.0f) P::load(qrow, i, a.vocab, y);
#pragma unroll
      for (int v = 0; v < P::kVec; v += 4) N::load(nrow, i + v, a.vocab, e + v);
      const uint32_t gone = st.barred && !fallback ? out[at >> 5] >> (at & 31) : 0u;
#pragma unroll
      for (int v = 0; v < P::kVec; ++v) {
        float w = weight(x[v], st.p_max, st.c);
        if (!fallback) {
          w *= st.p_mul;
          if (st.q_mul > 0.0f) w -= st.q_mul * weight(y[v], st.q_max, st.c);
          w = gone >> v & 1 ? 0.0f : w;
        }
        // (past the row's end: x is -inf)
        const float value = w * __builtin_amdgcn_rcpf(e[v]);
        const bool ahead = w > 0.0f && value > best;
        best = ahead ? value : best;
        at_best = ahead ? at + v : at_best;
      }
    }
    // a lane's places rise, so that its first leader is the lowest
    unsigned long long key = best > 0.0f ? (unsigned long long)(fallback ? 0u : 1u) << 63 |
                                               (unsigned long long)__float_as_uint(best) << 32 |
                                               (uint32_t)~(uint32_t)((int64_t)chunk * kChunk + at_best)
                                         : 0ull;
    key = wave_all(key, [](unsigned long long u, unsigned long long v) { return u > v ? u : v; });
    if ((tid & 63) == 0) part[fallback][tid >> 6] = key;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) key = part[fallback][w] > key ? part[fallback][w] : key;
    return key;
  };
  const unsigned long long best = run(false);
  return best ? best : run(true);  // nothing is left in this chunk
}

template <int DT>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyArgs a) {
  extern __shared__ __align__(16) char lds[];
  Node* const nodes = reinterpret_cast<Node*>(lds);
  __shared__ double sums[kWalkThreads / 64];
  __shared__ uint32_t out_bits[kChunk / 32];
  __shared__ unsigned long long part[2][kWalkThreads / 64];
  const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Nodes rows = nodes_of(a, seq);
  const int n = rows.n;
  const float c = slope_of(a, seq);
  for (int i = tid; i < n; i += kWalkThreads) {
    const int64_t r = rows.first + i;
    const int64_t x = load_index(a.ids, r, a.ids_i64);
    nodes[i].token = x >= 0 && x < a.vocab ? (int)x : -1;
    const int64_t p = a.parents ? load_index(a.parents, r, a.parents_i64) : i - 1;
    nodes[i].parent = p >= 0 && p < i ? (int)p : -1;
    nodes[i].u = a.uniforms[r];
  }
  // ---- the rows' maxima and sums: as many lanes a row as it has chunks, up to 64 ----
  {
    const int group = min(a.group, 64), in = tid & (group - 1);
    for (int r0 = tid / group; r0 < (a.draft ? 2 : 1) * n; r0 += kWalkThreads / group) {
      const int which = r0 >= n ? 1 : 0, i = r0 - which * n;
      const f32x4* st = a.stats + (which * a.total + rows.first + i) * a.chunks;
      float m = kNegInf, s = 0.0f;
      int place = 0x7fffffff;
      for (int c0 = in; c0 < a.chunks; c0 += group) {
        const f32x4 v = st[c0];
        join(m, s, place, v[0], v[1], __float_as_int(v[2]), c);
      }
      for (int o = 1; o < group; o <<= 1)
        join(m, s, place, __shfl_xor(m, o), __shfl_xor(s, o), __shfl_xor(place, o), c);
      if (in == 0) {
        if (which == 0) {
          nodes[i].m = m;
          nodes[i].s = s;
          nodes[i].place = c == 0.0f || !finite(m) ? place : -1;
        } else {
          nodes[i].qm = m;
          nodes[i].qs = s;
        }
      }
    }
  }
  __syncthreads();
  for (int i = tid; i < n; i += kWalkThreads) {
    const int p = nodes[i].parent;
    const int x = nodes[i].token;
    float ratio = i == 0 ? 1.0f : 0.0f;
    if (p >= 0 && x >= 0) {
      if (nodes[p].place >= 0) {
        ratio = nodes[p].place == x ? 1.0f : 0.0f;
      } else {
        const float l = element<DT>(a.logits + (rows.first + p) * a.row_stride * kSize<DT>, x);
        float d = (l - nodes[p].m) * c, f = 1.0f / nodes[p].s;
        if (a.draft && finite(nodes[p].qm)) {
          d -= (element<DT>(a.draft + (rows.first + p) * a.draft_stride * kSize<DT>, x) - nodes[p].qm) * c;
          f *= nodes[p].qs;
        }
        ratio = l == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(d) * f;
      }
    }
    nodes[i].ratio = ratio;
    a.acceptance[rows.first + i] = fminf(ratio, 1.0f);
  }
  // (rows past the widest tree: never reached)
  for (int64_t i = rows.first + n + tid; i < min(max((int64_t)a.cu[seq + 1], rows.first), a.total); i += kWalkThreads)
    a.acceptance[i] = 0.0f;
  __syncthreads();
  // ---- the walk, every thread alike ----
  int64_t* const out = a.accepted + (int64_t)seq * a.max_nodes;
  int cur = 0, taken = n > 0 ? 1 : 0;
  if (tid == 0 && n > 0) out[0] = 0;
  float fa = 1.0f, fb = 0.0f;  // what is left: fa p - fb q (drafts without q: fa p, but for what was turned down)
  float rest = 1.0f;           // without q: p less what was turned down
  bool behind = false;         // a rejection whose sum is still to be taken
  // the first child of the node reached behind node `after`, n: none
  auto next_child = [&](int after) {
    for (int i0 = (after + 1) & ~63; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const uint64_t kids = __builtin_amdgcn_ballot_w64(i > after && i < n && nodes[min(i, n - 1)].parent == cur);
      if (kids) return i0 + __builtin_ctzll(kids);
    }
    return n;
  };
  for (int i = next_child(0); i < n; i = next_child(i)) {
    bool take;
    const bool with_q = a.draft && nodes[cur].place < 0 && finite(nodes[cur].qm);
    if (nodes[cur].place >= 0) {
      take = nodes[i].ratio > 0.0f;
    } else if (with_q) {
      if (behind) {
        const double left = left_over<DT>(a, rows.first + cur, c, nodes[cur].m, fa / nodes[cur].s, nodes[cur].qm,
                                          fb / nodes[cur].qs, sums);
        fa = left > 0.0 ? (float)(fa / left) : 0.0f;
        fb = left > 0.0 ? (float)(fb / left) : 0.0f;
        behind = false;
      }
      take = nodes[i].u < fa * nodes[i].ratio - fb;
      if (!take) {
        fb += 1.0f;
        behind = true;
      }
    } else {
      bool again = false;  // a token that was turned down is out
      for (int j = cur + 1; j < i; ++j) again |= nodes[j].parent == cur && nodes[j].token == nodes[i].token;
      take = !again && rest > 0.0f && nodes[i].u * rest < nodes[i].ratio;
      if (!take && !again) rest -= nodes[i].ratio;
    }
    if (take) {
      cur = i;
      if (tid == 0) out[taken] = i;
      ++taken;
      fa = 1.0f;
      fb = 0.0f;
      rest = 1.0f;
      behind = false;
    }
  }
  for (int i = taken + tid; i < a.max_nodes; i += kWalkThreads) out[i] = -1;
  if (tid == 0) a.num_accepted[seq] = taken;
  if (n == 0 || nodes[cur].place >= 0) {
    if (tid == 0) {
      a.next[seq] = n == 0 ? -1 : nodes[cur].place;
      a.state[seq] = DrawState{};
    }
    return;
  }
  DrawState st{};
  st.draws = 1;
  st.row = rows.first + cur;
  st.c = c;
  st.p_max = nodes[cur].m;
  st.p_mul = fa / nodes[cur].s;
  const bool with_q = a.draft && finite(nodes[cur].qm) && fb > 0.0f;
  if (with_q) {
    st.q_max = nodes[cur].qm;
    st.q_mul = fb / nodes[cur].qs;
  }
  if (a.chunks > 1) {
    if (tid != 0) return;
    for (int j = cur + 1; j < n; ++j)
      if (!with_q && nodes[j].parent == cur) a.barred[(int64_t)seq * a.max_nodes + st.barred++] = nodes[j].token;
    a.state[seq] = st;
    return;
  }
  // A vocabulary of one chunk: the draw is here, and its launch not made (64 sequences
  // of 3-24 nodes over 8000 logits: 32 us in three launches, 27 in two).
  for (int i = tid; i < kChunk / 32; i += kWalkThreads) out_bits[i] = 0;
  __syncthreads();
  st.barred = !with_q && cur + 1 < n;
  for (int j = cur + 1 + tid; j < n; j += kWalkThreads) {
    const int x = nodes[j].token;
    if (nodes[j].parent == cur && x >= 0) atomicOr(&out_bits[x >> 5], 1u << (x & 31));
  }
  __syncthreads();
  const unsigned long long won = race<DT, kWalkThreads>(a, st, seq, 0, out_bits, part);
  // (no key at all: E is infinite or not a number everywhere)
  if (tid == 0) a.next[seq] = won ? (int64_t)(uint32_t)~(uint32_t)won : 0;
}

// The next token where the walk ended, a workgroup a chunk; the sequence's last one to
// arrive writes the race's winner.
template <int DT>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
  const int chunk = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const DrawState st = a.state[seq];
  if (!st.draws) return;
  __shared__ uint32_t out[kChunk / 32];
  for (int i = tid; i < kChunk / 32; i += kThreads) out[i] = 0;
  __syncthreads();
  for (int i = tid; i < st.barred; i += kThreads) {
    const int64_t x = a.barred[(int64_t)seq * a.max_nodes + i] - (int64_t)chunk * kChunk;
    if (x >= 0 && x < kChunk) atomicOr(&out[x >> 5], 1u << (x & 31));
  }
  __syncthreads();
  __shared__ unsigned long long part[2][kThreads / 64];
  const unsigned long long best = race<DT, kThreads>(a, st, seq, chunk, out, part);
  if (tid != 0) return;
  // (a maximum: the order of the workgroups changes nothing.  Both counters are at the
  // memory's side; the first one's answer is here before the second one goes out)
  unsigned long long* const leader = &a.state[seq].best;
  unsigned long long was = __hip_atomic_fetch_max(leader, best, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  asm volatile("s_waitcnt vmcnt(0)" : "+v"(was) : : "memory");
  if (__hip_atomic_fetch_add(&a.state[seq].arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1 == (unsigned)a.chunks) {
    asm volatile("" ::: "memory");
    const unsigned long long won = __hip_atomic_load(leader, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // (no key at all: E is infinite or not a number everywhere)
    a.next[seq] = won ? (int64_t)(uint32_t)~(uint32_t)won : 0;
  }
}

int chunks_of(int vocab) { return (int)(((int64_t)vocab + kChunk - 1) / kChunk); }

template <int DT>
int launch_verify(const VerifyArgs& a, hipStream_t s) {
  const int64_t rows = a.total * (a.draft ? 2 : 1);
  if (rows) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(verify_stats_kernel<DT>),
                       dim3(a.chunks, (unsigned)(rows < 32768 ? rows : 32768), (unsigned)((rows + 32767) / 32768)),
                       dim3(kThreads), 0, s, a);
    if (hipError_t e = hipGetLastError()) return (int)e;
  }
  hipLaunchKernelGGL(HIP_KERNEL_NAME(verify_walk_kernel<DT>), dim3(a.num_seqs), dim3(kWalkThreads),
                     (size_t)a.max_nodes * sizeof(Node), s, a);
  if (hipError_t e = hipGetLastError()) return (int)e;
  if (a.chunks == 1) return MKV_OK;
  hipLaunchKernelGGL(HIP_KERNEL_NAME(verify_draw_kernel<DT>), dim3(a.chunks, a.num_seqs), dim3(kThreads), 0, s, a);
  return (int)hipGetLastError();
}

bool index_ok(int dt) { return dt == MKV_INDEX_I32 || dt == MKV_INDEX_I64; }

}  // namespace
}  // namespace mkv

using namespace mkv;

extern "C" size_t mkv_verify_drafts_workspace_size(int64_t total, int vocab, int num_seqs, int max_nodes, int has_draft) {
  if (total < 0 || vocab <= 0 || num_seqs < 0 || max_nodes < 0 || max_nodes > kMaxNodes) return 0;
  return (size_t)total * (has_draft ? 2 : 1) * chunks_of(vocab) * sizeof(f32x4) +
         (size_t)num_seqs * (sizeof(DrawState) + (size_t)max_nodes * sizeof(int32_t));
}

extern "C" int mkv_verify_drafts(int64_t* accepted, int64_t* num_accepted, int64_t* next_tokens, float* acceptance,
                                 const void* logits, int64_t row_stride, const void* draft_logits, int64_t draft_stride,
                                 int dtype, int64_t total, int vocab, const void* token_ids, int ids_dtype,
                                 const void* parents, int parents_dtype, const int32_t* cu_seqlens_q, int num_seqs,
                                 int max_nodes, const float* uniforms, const float* noise, int64_t noise_stride,
                                 const float* temperatures, void* workspace, size_t workspace_bytes, void* stream) {
  if (total < 0 || total > 0x1fffffff || vocab <= 0 || vocab > 0x7fff0000 || num_seqs < 0 || num_seqs > 65535 ||
      max_nodes < 1 || max_nodes > kMaxNodes)
    return MKV_ERR_BAD_SHAPE;
  if (!index_ok(ids_dtype) || (parents && !index_ok(parents_dtype))) return MKV_ERR_UNSUPPORTED_DTYPE;
  if (num_seqs == 0) return MKV_OK;
  if (!accepted || !num_accepted || !next_tokens || !cu_seqlens_q || !noise || !workspace ||
      (total && (!acceptance || !logits || !token_ids || !uniforms)))
    return MKV_ERR_NULL_POINTER;
  if (row_stride < vocab || noise_stride < vocab || (draft_logits && draft_stride < vocab)) return MKV_ERR_BAD_STRIDE;
  if (dtype != MKV_DTYPE_F32 && dtype != MKV_DTYPE_BF16 && dtype != MKV_DTYPE_F16) return MKV_ERR_UNSUPPORTED_DTYPE;
  const int size = dtype == MKV_DTYPE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(draft_logits)) % size ||
      reinterpret_cast<uintptr_t>(noise) % 4 || reinterpret_cast<uintptr_t>(workspace) & 15)
    return MKV_ERR_MISALIGNED;
  const int chunks = chunks_of(vocab);
  // (a grid's first two dimensions: below 2^32 threads)
  if ((int64_t)chunks * num_seqs > 0xffffff || (int64_t)chunks * (total < 16384 ? 2 * total : 32768) > 0xffffff)
    return MKV_ERR_BAD_SHAPE;
  if (workspace_bytes < mkv_verify_drafts_workspace_size(total, vocab, num_seqs, max_nodes, draft_logits != nullptr))
    return MKV_ERR_WORKSPACE_TOO_SMALL;
  VerifyArgs a;
  a.logits = reinterpret_cast<const char*>(logits);
  a.draft = reinterpret_cast<const char*>(draft_logits);
  a.row_stride = row_stride;
  a.draft_stride = draft_stride;
  a.total = total;
  a.vocab = vocab;
  a.chunks = chunks;
  a.group = 1;
  while (a.group < chunks && a.group < 64) a.group <<= 1;
  a.ids = token_ids;
  a.parents = parents;
  a.ids_i64 = ids_dtype == MKV_INDEX_I64;
  a.parents_i64 = parents_dtype == MKV_INDEX_I64;
  a.cu = cu_seqlens_q;
  a.num_seqs = num_seqs;
  a.uniforms = uniforms;
  a.noise = noise;
  a.noise_stride = noise_stride;
  a.temperatures = temperatures;
  a.max_nodes = max_nodes;
  a.accepted = accepted;
  a.num_accepted = num_accepted;
  a.next = next_tokens;
  a.acceptance = acceptance;
  a.stats = reinterpret_cast<f32x4*>(workspace);
  a.state = reinterpret_cast<DrawState*>(a.stats + (size_t)total * (draft_logits ? 2 : 1) * chunks);
  a.barred = reinterpret_cast<int32_t*>(a.state + num_seqs);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  switch (dtype) {
    case MKV_DTYPE_F32: return launch_verify<MKV_DTYPE_F32>(a, s);
    case MKV_DTYPE_BF16: return launch_verify<MKV_DTYPE_BF16>(a, s);
    default: return launch_verify<MKV_DTYPE_F16>(a, s);
  }
}
