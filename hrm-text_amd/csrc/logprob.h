// Log probabilities of given tokens, their entropy and the top alternatives, from logits, and the
// gradient of the logits: the language-model head's loss and scoring (models/lm_head.py:52, the
// cross entropy in fp32).
//
// For a row x of V logits and a target t:
//   m = max_j x_j, S = sum_j e^(x_j - m), W = sum_j e^(x_j - m) (x_j - m)
//   logprob = (x_t - m) - ln S,  entropy = ln S - W / S
// and for the gradients g of logprob and h of entropy, with ln p_j = (x_j - m) - ln S (m and ln S are
// kept apart: where |m| is large their sum would lose ln S):
//   dx_j = g ([j = t] - p_j) - h p_j (ln p_j + entropy).
// The top alternatives are the k largest logits, the lower index first among equal ones.
#pragma once
#include "common.h"

#include <type_traits>

namespace prefixlm {
namespace lp {

constexpr int NT = 512;           // threads of a forward workgroup
constexpr int kMaxTop = 64;
constexpr int kCand = 1024;       // candidates a workgroup sorts; more take the slow walk
constexpr int kUnroll = 4;        // 16-byte vectors a thread has in flight
constexpr int kMaxSplits = 64;
static_assert(kMaxTop <= NT && kMaxTop <= kCand, "a threshold has enough thread maxima");

struct Params {
  const void* x;
  const void* targets;            // int64 or int32 [rows], or null
  const float* g;                 // backward: gradient of logprob [rows], or null
  const float* h;                 // backward: gradient of entropy [rows], or null
  float* logprob;                 // [rows], or null
  float* entropy;                 // [rows], or null
  float* stats;                   // [rows, 2]: m (0 where it is -inf) and ln S
  float* top_val;                 // [rows, top]
  int64_t* top_id;                // [rows, top]
  void* dx;
  float* part;                    // [rows, nsplit, 4 floats]: m, S, W
  unsigned long long* part_top;   // [rows, nsplit, top]
  int64_t x_st, dx_st, rows, V;
  int64_t ignore;
  int top, wide_targets, nsplit;
};

// 8 consecutive elements, a row's vectors. The row's edges are what lies before the first vector and
// behind the last whole one, at most 14 elements, each of which one thread takes. A row may begin at
// any element. The forward's vectors begin with the row, so that a row's sums are added in one order
// wherever it lies (and cost a sixth more off 16 bytes: 1021 rows of 50257 logits 27.6 us, of 50256
// 24.0); the gradient's, which have no order, at its first 16-byte address.
typedef u32x4 u32x4_u __attribute__((aligned(2)));   // the target handles these at any alignment
typedef f32x4 f32x4_u __attribute__((aligned(4)));
template <class T>
struct Vec;
template <>
struct Vec<bf16> {
  u32x4 w;
  template <bool NT = false>
  __device__ __forceinline__ void load(const bf16* p) {
    const u32x4_u* q = reinterpret_cast<const u32x4_u*>(p);
    w = NT ? __builtin_nontemporal_load(q) : *q;
  }
  __device__ __forceinline__ float get(int e) const { return (e & 1) ? bf16hi(w[e >> 1]) : bf16lo(w[e >> 1]); }
};
template <>
struct Vec<float> {
  f32x4 w[2];
  template <bool NT = false>
  __device__ __forceinline__ void load(const float* p) {
    const f32x4_u* q = reinterpret_cast<const f32x4_u*>(p);
    w[0] = NT ? __builtin_nontemporal_load(q) : q[0];
    w[1] = NT ? __builtin_nontemporal_load(q + 1) : q[1];
  }
  __device__ __forceinline__ float get(int e) const { return w[e >> 2][e & 3]; }
};
struct Edges {
  int lead, rest;      // elements before the vectors, and behind
  int64_t nvec;
  __device__ __forceinline__ Edges(int lead_, int64_t V) {
    lead = (int)(lead_ < V ? lead_ : V);
    nvec = (V - lead) / 8;
    rest = (int)(V - lead - 8 * nvec);
  }
  __device__ __forceinline__ int count() const { return lead + rest; }
  __device__ __forceinline__ int64_t at(int i) const { return i < lead ? i : 8 * nvec + i; }
};
__device__ __forceinline__ float as_f32(bf16 x) { return (float)x; }
__device__ __forceinline__ float as_f32(float x) { return x; }

// The values' order as whole numbers, NaN above all; 0 is below every value
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);   // -0 as 0: they are equal
  return (b >> 31) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
  return __builtin_bit_cast(float, (k >> 31) ? k & 0x7fffffffu : ~k);
}
// larger value first, then lower index; never 0
__device__ __forceinline__ unsigned long long key_of(float x, int64_t j) {
  return ((unsigned long long)order_of(x) << 32) | (0xffffffffu - (uint32_t)j);
}

__device__ __forceinline__ float first_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}

// The running (m, S, W): S and W against ref(m), 0 where m is -inf
struct Stat {
  float m, s, w;
};
__device__ __forceinline__ Stat no_values() { return Stat{-INFINITY, 0.f, 0.f}; }
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }
// differences are kept above -1e30, so that 0 weight times them is 0
__device__ __forceinline__ float below(float d) { return fmaxf(d, -1e30f); }
template <bool ENT>
__device__ __forceinline__ void raise(Stat& a, float m) {
  const float r = ref_of(m), d = a.m - r;
  const float f = __builtin_amdgcn_exp2f(d * kLog2e);   // a.m = -inf: 0
  if (ENT) a.w = f * (a.w + a.s * below(d));
  a.s *= f;
  a.m = m;
}
template <bool ENT>
__device__ __forceinline__ void join(Stat& a, Stat b) {
  const float m = fmaxf(a.m, b.m);
  raise<ENT>(a, m);
  raise<ENT>(b, m);
  a.s += b.s;
  if (ENT) a.w += b.w;
}

// a takes the N values f, whose largest is returned
template <bool ENT, int N>
__device__ __forceinline__ float take(Stat& a, const float (&f)[N]) {
  float mx = f[0];
#pragma unroll
  for (int e = 1; e < N; ++e) mx = fmaxf(mx, f[e]);
  if (mx > a.m) raise<ENT>(a, mx);
  const float r = ref_of(a.m);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float d = f[e] - r, ex = __builtin_amdgcn_exp2f(d * kLog2e);
    a.s += ex;
    if (ENT) a.w += ex * below(d);
  }
  return mx;
}

__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const unsigned long long y = __shfl_xor(x, m);
    x = y > x ? y : x;
  }
  return x;
}
// What a workgroup holds while it picks the top elements
constexpr int kGroups = 8;        // of a thread's vectors, by their turn
struct TopShared {
  unsigned long long cand[kCand];
  float largest[kGroups][NT];     // of each thread's values in a group
  uint16_t list[kCand];           // groups to look at again: thread, and group << 9
  uint32_t keys[NT / 8];
  unsigned long long best[NT / 64];
  int n, groups;
};
static_assert(NT == 1 << 9 && kGroups << 9 <= 1 << 16, "a list's entry");

// The `top` largest keys of cand[0, n), in order, to put(rank, key)
template <class Put>
__device__ __forceinline__ void sorted_top(const unsigned long long* cand, int n, int top, Put put) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const unsigned long long c = cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > c;
    if (rank < top) put(rank, c);
  }
}

__device__ __forceinline__ int64_t target_of(const Params& P, int64_t row) {
  return P.wide_targets ? static_cast<const int64_t*>(P.targets)[row] : (int64_t) static_cast<const int32_t*>(P.targets)[row];
}
// A row's target and its logit
struct Target {
  bool counted, valid;
  float x;
};
template <class T>
__device__ __forceinline__ Target target_at(const Params& P, int64_t row) {
  Target r{false, false, 0.f};
  if (P.targets) {
    const int64_t t = target_of(P, row);
    r.counted = t != P.ignore;
    r.valid = t >= 0 && t < P.V;
    if (r.counted && r.valid) r.x = as_f32(static_cast<const T*>(P.x)[row * P.x_st + t]);
  }
  return r;
}

// What a row's result is, from its statistics
__device__ __forceinline__ void finish_row(const Params& P, int64_t row, const Stat& a, const Target& t) {
  const float ln_s = logf(a.s), r = ref_of(a.m);   // all logits -inf: ln 0
  P.stats[2 * row] = r;
  P.stats[2 * row + 1] = ln_s;
  if (P.logprob) P.logprob[row] = !t.counted ? 0.f : !t.valid ? __builtin_nanf("") : (t.x - r) - ln_s;
  if (P.entropy) P.entropy[row] = a.s == 0.f ? __builtin_nanf("") : ln_s - a.w / a.s;
}

// Workgroup = (row, split of its vectors); thread = every NT-th vector of 8 logits, with a running
// (m, S, W) of its own, joined at the end. One pass over the row, of which four vectors a thread are in
// registers and the next four on their way; four workgroups a CU. Bound by the loads where rows are
// many (6144 of 65536 bf16 logits, 805 MB, 135 to 158 us, 5.1 to 6.0 TB/s), by about ten operations a
// logit and the search behind the pass where all workgroups run at once (1021 rows of 50257 with
// entropy and eight alternatives 35 us, with neither 28), and by one CU's exponentials for
// few rows (4 rows of 65536 with five alternatives 10.1 us, without 6.4).
//
// TOP: after the pass the largest values of 64 sets of 8 threads are known. The k-th largest of those
// is reached by at least k elements, so only the groups of a thread's vectors whose largest reaches it
// are looked at again, one vector a thread (by the thread that holds the group, a round trip to memory
// for each: 4 x 65536 with 20 alternatives 14.8 us, now 11.0); the elements that reach it, mostly few
// more than k, are ranked against each other. Where they do not fit (rows of many equal values, or of fewer
// finite logits than alternatives), or a NaN is among them, which the maxima pass over, a walk finds the next
// largest k times (4 x 65536 with ten finite logits and 20 alternatives 164 us).
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(NT) void forward_kernel(Params P) {
  __shared__ Stat s_stat[NT / 64];
  __shared__ TopShared t;   // unused without TOP
  const int64_t row = blockIdx.x / P.nsplit;
  const int split = (int)(blockIdx.x % P.nsplit);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* x = static_cast<const T*>(P.x) + row * P.x_st;
  if (!ENT && !TOP && P.targets && target_of(P, row) == P.ignore) {   // nothing of the row is wanted
    if (P.nsplit == 1 && tid == 0) {
      P.logprob[row] = 0.f;
      P.stats[2 * row] = P.stats[2 * row + 1] = 0.f;
    }
    return;
  }
  const Edges edges(0, P.V);
  const int64_t per = (edges.nvec + P.nsplit - 1) / P.nsplit;
  const int64_t v0 = split * per < edges.nvec ? split * per : edges.nvec, v1 = v0 + per < edges.nvec ? v0 + per : edges.nvec;
  const int n_edge = split == 0 ? edges.count() : 0;

  Target target{false, false, 0.f};
  if (tid == 0 && P.nsplit == 1) target = target_at<T>(P, row);
  if (TOP)
#pragma unroll
    for (int i = 0; i < kGroups; ++i) t.largest[i][tid] = -INFINITY;
  // groups of kUnroll vectors a thread, the next one on its way while one is taken; vectors past the
  // last one are read as that one and count as -inf
  Stat a = no_values();
  const float edge = tid < n_edge ? as_f32(x[edges.at(tid)]) : -INFINITY;
  if (v0 < v1) {
    Vec<T> w[kUnroll];
    auto load = [&](int64_t g) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int64_t v = g + u * NT + tid;
        w[u].load(x + 8 * (v < v1 ? v : v1 - 1));
      }
    };
    load(v0);
    int turn = 0;
    for (int64_t g = v0; g < v1; g += kUnroll * NT) {
      float f[8 * kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
#pragma unroll
        for (int e = 0; e < 8; ++e) f[8 * u + e] = w[u].get(e);
      if (g + kUnroll * NT < v1) load(g + kUnroll * NT);
      if (g + kUnroll * NT > v1) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
#pragma unroll
          for (int e = 0; e < 8; ++e) f[8 * u + e] = g + u * NT + tid < v1 ? f[8 * u + e] : -INFINITY;
      }
      const float mx = take<ENT>(a, f);
      if (TOP) {
        float* l = &t.largest[turn & (kGroups - 1)][tid];
        *l = turn < kGroups ? mx : fmaxf(*l, mx);
        ++turn;
      }
    }
  }
  if (tid < n_edge) {
    const float f[1] = {edge};
    take<ENT>(a, f);
  }
  const float m_thread = a.m;
  const bool any = v0 + tid < v1 || tid < n_edge;
  auto join_lanes = [&](int m) {
    Stat b;
    b.m = __shfl_xor(a.m, m);
    b.s = __shfl_xor(a.s, m);
    b.w = ENT ? __shfl_xor(a.w, m) : 0.f;
    join<ENT>(a, b);
  };
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) join_lanes(m);
  if (lane == 0) s_stat[wave] = a;
  __syncthreads();
  a = s_stat[lane & (NT / 64 - 1)];
#pragma unroll
  for (int m = 1; m < NT / 64; m <<= 1) join_lanes(m);
  // the workgroup's: the first lane's, whose joins run in one order in every wave (the lanes' differ
  // in their last bit, and which of them holds an alternative is not fixed)
  a.m = first_lane(a.m);
  a.s = first_lane(a.s);
  a.w = first_lane(a.w);
  if (tid == 0) {
    if (P.nsplit == 1) {
      finish_row(P, row, a, target);
    } else {
      float* p = P.part + (row * P.nsplit + split) * 4;
      p[0] = a.m;
      p[1] = a.s;
      p[2] = a.w;
    }
  }
  if (!TOP) return;

  const int top = P.top;
  {
    uint32_t k = any ? order_of(m_thread) : 0;
    auto step = [&](auto ctrl) {   // over each 8 lanes
      const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)k, decltype(ctrl)::value, 0xF, 0xF, false);
      k = y > k ? y : k;
    };
    step(std::integral_constant<int, 0xB1>{});
    step(std::integral_constant<int, 0x4E>{});
    step(std::integral_constant<int, 0x141>{});
    if ((lane & 7) == 0) t.keys[tid >> 3] = k;
    if (tid == 0) t.n = t.groups = 0;
  }
  __syncthreads();
  static_assert(NT / 8 == 64 && kMaxTop <= 64, "one set a lane, and a top-th largest of them");
  uint32_t thr;
  {
    const uint32_t k = t.keys[lane];
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
      const uint32_t y = (uint32_t)__builtin_amdgcn_readlane((int)k, j);
      rank += y > k || (y == k && j < lane);
    }
    thr = (uint32_t)__builtin_amdgcn_readlane((int)k, (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(rank == top - 1)));
  }
  // fewer sets with elements than `top`: every element (none of them NaN, or the walk decides)
  const float least = thr ? value_of(thr) : -INFINITY;
  auto look = [&](float f, int64_t j) {
    if (f >= least) {
      const int at = atomicAdd(&t.n, 1);   // the order does not matter: they are ranked
      if (at < kCand) t.cand[at] = key_of(f, j);
    }
  };
  if (any && m_thread >= least) {
    for (int i = 0; i < kGroups; ++i)
      if (v0 + (int64_t)i * kUnroll * NT + tid < v1 && t.largest[i][tid] >= least) {
        const int at = atomicAdd(&t.groups, 1);
        if (at < kCand) t.list[at] = (uint16_t)(tid | i << 9);
      }
    if (tid < n_edge) look(edge, edges.at(tid));
  }
  __syncthreads();
  // a thread takes one vector of a listed group, so that all are on their way together (a group holds
  // one of the values that are looked for at least: more groups than fit are more candidates than fit)
  const int groups = t.groups;
  for (int k = tid; k < kUnroll * (groups < kCand ? groups : 0); k += NT) {
    const int of = t.list[k / kUnroll] & (NT - 1), i = t.list[k / kUnroll] >> 9;
    for (int64_t v = v0 + ((int64_t)i * kUnroll + k % kUnroll) * NT + of; v < v1; v += kGroups * kUnroll * NT) {
      Vec<T> w;
      w.load(x + 8 * v);
#pragma unroll
      for (int e = 0; e < 8; ++e) look(w.get(e), 8 * v + e);
    }
  }
  __syncthreads();
  const float ln_s = logf(a.s), ref = ref_of(a.m);
  // a split may hold fewer elements than `top`: the rest of its list is empty
  const int64_t held = 8 * (v1 - v0) + n_edge;
  const int want = held < top ? (int)held : top;
  auto put = [&](int r, unsigned long long c) {
    if (P.nsplit == 1) {
      P.top_val[row * top + r] = (value_of((uint32_t)(c >> 32)) - ref) - ln_s;
      P.top_id[row * top + r] = 0xffffffffu - (uint32_t)c;
    } else {
      P.part_top[(row * P.nsplit + split) * top + r] = c;
    }
  };
  if (P.nsplit > 1 && tid >= want && tid < top) P.part_top[(row * P.nsplit + split) * top + tid] = 0;
  const int n = t.n;
  if (n >= want && n <= kCand && groups < kCand && a.s == a.s) {
    sorted_top(t.cand, n, want, put);
    return;
  }
  unsigned long long last = ~0ull;
  for (int r = 0; r < want; ++r) {
    unsigned long long b = 0;
    auto look = [&](float f, int64_t j) {
      const unsigned long long c = key_of(f, j);
      if (c < last && c > b) b = c;
    };
    for (int64_t u = v0 + tid; u < v1; u += NT) {
      Vec<T> w;
      w.load(x + 8 * u);
#pragma unroll
      for (int e = 0; e < 8; ++e) look(w.get(e), 8 * u + e);
    }
    if (tid < n_edge) look(edge, edges.at(tid));
    b = wave_max_u64(b);
    if (lane == 0) t.best[wave] = b;
    __syncthreads();
    b = t.best[0];
    for (int g = 1; g < NT / 64; ++g) b = t.best[g] > b ? t.best[g] : b;
    if (tid == 0) put(r, b);
    last = b;
    __syncthreads();
  }
}

// Joins the splits of a row: one workgroup of 256 threads per row. Bound by its launch and the latency
// of its loads, which is what lp_nsplit's threshold weighs.
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(256) void combine_kernel(Params P) {
  __shared__ Stat s_row;
  __shared__ unsigned long long s_cand[kCand];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  if (!ENT && !TOP && P.targets && target_of(P, row) == P.ignore) {
    if (tid == 0) {
      P.logprob[row] = 0.f;
      P.stats[2 * row] = P.stats[2 * row + 1] = 0.f;
    }
    return;
  }
  const int n = P.nsplit * P.top;
  if (TOP)
    for (int i = tid; i < n; i += 256) s_cand[i] = P.part_top[row * n + i];
  if (tid < 64) {
    Stat a = no_values();
    if (tid < P.nsplit) {
      const float* p = P.part + (row * P.nsplit + tid) * 4;
      a.m = p[0];
      a.s = p[1];
      a.w = p[2];
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      Stat b;
      b.m = __shfl_xor(a.m, m);
      b.s = __shfl_xor(a.s, m);
      b.w = ENT ? __shfl_xor(a.w, m) : 0.f;
      join<ENT>(a, b);
    }
    if (tid == 0) {
      s_row = a;
      finish_row(P, row, a, target_at<T>(P, row));
    }
  }
  if (!TOP) return;
  __syncthreads();
  const float ln_s = logf(s_row.s), ref = ref_of(s_row.m);
  sorted_top(s_cand, n, P.top, [&](int r, unsigned long long c) {
    if (c == 0) return;   // an empty place (V >= top: the first `top` ranks hold elements)
    P.top_val[row * P.top + r] = (value_of((uint32_t)(c >> 32)) - ref) - ln_s;
    P.top_id[row * P.top + r] = 0xffffffffu - (uint32_t)c;
  });
}

template <bool NT, class V, class T>
__device__ __forceinline__ void store(T* p, V v) {
  if (NT)
    __builtin_nontemporal_store(v, reinterpret_cast<V*>(p));
  else
    *reinterpret_cast<V*>(p) = v;
}

// thread = vectors of 8 logits of one row; blockIdx.x = (row, block of 256 kUnroll vectors). The
// vectors begin where the gradient's row is aligned; the logits' row mostly is there too. The rows go
// from the last to the first: what the forward read last is read first, and partly still in the
// last-level cache. Bound by memory: 8192 x 65536 bf16, three quarters of them read, 1.88 GB in 292 to
// 298 us, 6.3 TB/s. NT: non-temporal accesses, for logits and gradients beyond kNtBytes together: the
// gradient is not in the caches when it is read anyway, and what it would push out are the logits
// (forward + backward with plain accesses and with these, 2048 x 32000 bf16, 262 MB, 80.6 and 69.2 us,
// 8192 x 65536 558 and 530, 1024 x 65536 fp32 157 and 132; 1024 x 32000 bf16, 131 MB, 37 either way).
constexpr int64_t kNtBytes = (int64_t)192 << 20;
template <class T, bool ENT, bool NT>
__global__ __launch_bounds__(256) void backward_kernel(Params P, int nblk) {
  const int64_t row = P.rows - 1 - blockIdx.x / nblk;
  const int64_t v0 = (int64_t)(blockIdx.x % nblk) * 256 * kUnroll + threadIdx.x;
  const T* x = static_cast<const T*>(P.x) + row * P.x_st;
  T* dx = static_cast<T*>(P.dx) + row * P.dx_st;
  const int64_t t = P.g ? target_of(P, row) : -1;   // without g there may be no targets
  const bool counted = P.g && t != P.ignore;
  float g = counted ? P.g[row] : 0.f;
  if (counted && (t < 0 || t >= P.V)) g = __builtin_nanf("");
  const float h = ENT && P.h ? P.h[row] : 0.f, H = ENT ? P.entropy[row] : 0.f;
  const float m = P.stats[2 * row], ln_s = P.stats[2 * row + 1];
  const bool zero = g == 0.f && h == 0.f;
  const Edges edges((int)((16 - ((uintptr_t)dx & 15)) % 16 / sizeof(T)), P.V);
  auto grad = [&](float f, int64_t j) {
    const float l = (f - m) - ln_s, p = __builtin_amdgcn_exp2f(l * kLog2e);
    float d = -g * p;
    if (ENT) d -= h * (p * (below(l) + H));
    return j == t ? d + g : d;
  };
  Vec<T> w[kUnroll];
  if (!zero) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (v0 + u * 256 < edges.nvec) w[u].template load<NT>(x + edges.lead + 8 * (v0 + u * 256));
  }
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    if (v0 + u * 256 >= edges.nvec) break;
    const int64_t j0 = edges.lead + 8 * (v0 + u * 256);
    float d[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e] = zero ? 0.f : grad(w[u].get(e), j0 + e);
    if constexpr (sizeof(T) == 2) {
      store<NT>(dx + j0, __builtin_bit_cast(u32x4, cvt8(d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7])));
    } else {
      store<NT>(dx + j0, f32x4{d[0], d[1], d[2], d[3]});
      store<NT>(dx + j0 + 4, f32x4{d[4], d[5], d[6], d[7]});
    }
  }
  if (blockIdx.x % nblk == 0 && (int)threadIdx.x < edges.count()) {
    const int64_t j = edges.at(threadIdx.x);
    dx[j] = (T)(zero ? 0.f : grad(as_f32(x[j]), j));
  }
}

}  // namespace lp
}  // namespace prefixlm
