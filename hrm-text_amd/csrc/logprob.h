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

// 8 consecutive elements, at any address that suits one element: the target handles 16-byte
// accesses at any alignment
typedef u32x4 u32x4_u __attribute__((aligned(2)));
typedef f32x4 f32x4_u __attribute__((aligned(4)));
template <class T>
struct Vec;
template <>
struct Vec<bf16> {
  u32x4 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const u32x4_u*>(p); }
  __device__ __forceinline__ float get(int e) const { return (e & 1) ? bf16hi(w[e >> 1]) : bf16lo(w[e >> 1]); }
};
template <>
struct Vec<float> {
  f32x4 w[2];
  __device__ __forceinline__ void load(const float* p) {
    w[0] = reinterpret_cast<const f32x4_u*>(p)[0];
    w[1] = reinterpret_cast<const f32x4_u*>(p)[1];
  }
  __device__ __forceinline__ float get(int e) const { return w[e >> 2][e & 3]; }
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

// a takes the N values f
template <bool ENT, int N>
__device__ __forceinline__ void take(Stat& a, const float (&f)[N]) {
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
}

__device__ __forceinline__ unsigned long long wave_max_u64(unsigned long long x) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const unsigned long long y = __shfl_xor(x, m);
    x = y > x ? y : x;
  }
  return x;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
  auto step = [&](auto ctrl) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, false);
    x = y > x ? y : x;
  };
  step(std::integral_constant<int, 0xB1>{});
  step(std::integral_constant<int, 0x4E>{});
  step(std::integral_constant<int, 0x141>{});
  step(std::integral_constant<int, 0x140>{});
  uint32_t r = 0;
#pragma unroll
  for (int l = 0; l < 64; l += 16) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_readlane((int)x, l);
    r = y > r ? y : r;
  }
  return r;
}

// What a workgroup holds while it picks the top elements
struct TopShared {
  unsigned long long cand[kCand];
  uint32_t keys[NT];
  unsigned long long best[NT / 64];
  uint32_t thr;
  int n;
};

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

// What a row's result is, from its statistics
__device__ __forceinline__ void finish_row(const Params& P, int64_t row, const Stat& a, float xt, bool counted, bool valid) {
  const float ln_s = logf(a.s), r = ref_of(a.m);   // all logits -inf: ln 0
  P.stats[2 * row] = r;
  P.stats[2 * row + 1] = ln_s;
  if (P.logprob) P.logprob[row] = !counted ? 0.f : !valid ? __builtin_nanf("") : (xt - r) - ln_s;
  if (P.entropy) P.entropy[row] = a.s == 0.f ? __builtin_nanf("") : ln_s - a.w / a.s;
}
__device__ __forceinline__ int64_t target_of(const Params& P, int64_t row) {
  return P.wide_targets ? static_cast<const int64_t*>(P.targets)[row] : (int64_t) static_cast<const int32_t*>(P.targets)[row];
}
template <class T>
__device__ __forceinline__ void finish(const Params& P, int64_t row, const Stat& a) {
  bool counted = false, valid = false;
  float xt = 0.f;
  if (P.targets) {
    const int64_t t = target_of(P, row);
    counted = t != P.ignore;
    valid = t >= 0 && t < P.V;
    if (counted && valid) xt = as_f32(static_cast<const T*>(P.x)[row * P.x_st + t]);
  }
  finish_row(P, row, a, xt, counted, valid);
}

// Workgroup = (row, split of its vectors); thread = every NT-th vector of 8 logits, with a running
// (m, S, W) of its own, joined at the end. One pass over the row.
//
// TOP: each thread's largest value is known after the pass. The k-th largest of those is reached by
// at least k elements, so only threads whose largest reaches it look at their elements again (about
// k of NT), and those elements, mostly little more than k, are ranked against each other. Where
// they do not fit (rows of many equal values), or a NaN is among them, which the maxima pass over, a
// walk finds the next largest k times.
template <class T, bool ENT, bool TOP>
__global__ __launch_bounds__(NT) void forward_kernel(Params P) {
  __shared__ Stat s_stat[NT / 64];
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
  const int64_t nv = (P.V + 7) / 8, full = P.V / 8;   // the last vector may be partial
  const int64_t per = (nv + P.nsplit - 1) / P.nsplit;
  const int64_t v0 = split * per, v1 = v0 + per < nv ? v0 + per : nv, vf = v1 < full ? v1 : full;

  Stat a = no_values();
  int64_t v = v0 + tid;
  for (; v + (kUnroll - 1) * NT < vf; v += kUnroll * NT) {
    Vec<T> w[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) w[u].load(x + 8 * (v + u * NT));
    float f[8 * kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int e = 0; e < 8; ++e) f[8 * u + e] = w[u].get(e);
    take<ENT>(a, f);
  }
  for (; v < v1; v += NT) {
    if (v < full) {
      Vec<T> w;
      w.load(x + 8 * v);
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = w.get(e);
      take<ENT>(a, f);
    } else {
      for (int64_t j = 8 * v; j < P.V; ++j) {
        const float f[1] = {as_f32(x[j])};
        take<ENT>(a, f);
      }
    }
  }
  const float m_thread = a.m;
  const bool any = v0 + tid < v1;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    Stat b;
    b.m = __shfl_xor(a.m, m);
    b.s = __shfl_xor(a.s, m);
    b.w = ENT ? __shfl_xor(a.w, m) : 0.f;
    join<ENT>(a, b);
  }
  if (lane == 0) s_stat[wave] = a;
  __syncthreads();
  if (tid == 0) {
    a = s_stat[0];
    for (int g = 1; g < NT / 64; ++g) join<ENT>(a, s_stat[g]);
    if (P.nsplit == 1) {
      finish<T>(P, row, a);
    } else {
      float* p = P.part + (row * P.nsplit + split) * 4;
      p[0] = a.m;
      p[1] = a.s;
      p[2] = a.w;
    }
    s_stat[0] = a;
  }
  if (!TOP) return;

  __shared__ TopShared t;
  const int top = P.top;
  t.keys[tid] = any ? order_of(m_thread) : 0;
  if (tid == 0) t.n = 0;
  __syncthreads();   // and s_stat[0] is the workgroup's
  if (wave == 0) {
    // the top-th largest of the threads' largest
    uint32_t mine[NT / 64];
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) mine[i] = t.keys[i * 64 + lane];
    uint32_t thr = 0;
    for (int r = 0; r < top; ++r) {
      uint32_t b = mine[0];
#pragma unroll
      for (int i = 1; i < NT / 64; ++i) b = mine[i] > b ? mine[i] : b;
      thr = wave_max_u32(b);
      // one of the threads that hold it is done
      const unsigned long long who = __builtin_amdgcn_ballot_w64(b == thr);
      if (lane == (int)__builtin_ctzll(who)) {
        bool gone = false;
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) {
          const bool hit = !gone && mine[i] == thr;
          gone |= hit;
          mine[i] = hit ? 0 : mine[i];
        }
      }
    }
    if (lane == 0) t.thr = thr;
  }
  __syncthreads();
  const uint32_t thr = t.thr;
  if (any && order_of(m_thread) >= thr) {
    for (int64_t u = v0 + tid; u < v1; u += NT)
      for (int64_t j = 8 * u; j < 8 * u + 8 && j < P.V; ++j) {
        const float f = as_f32(x[j]);
        if (order_of(f) >= thr) {
          const int at = atomicAdd(&t.n, 1);   // the order does not matter: they are ranked
          if (at < kCand) t.cand[at] = key_of(f, j);
        }
      }
  }
  __syncthreads();
  const float ln_s = logf(s_stat[0].s), ref = ref_of(s_stat[0].m);
  // a split may hold fewer elements than `top`: the rest of its list is empty
  const int64_t held = (8 * v1 < P.V ? 8 * v1 : P.V) - 8 * v0;
  const int want = held < top ? (held > 0 ? (int)held : 0) : top;
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
  if (n >= want && n <= kCand && s_stat[0].s == s_stat[0].s) {
    sorted_top(t.cand, n, want, put);
    return;
  }
  unsigned long long last = ~0ull;
  for (int r = 0; r < want; ++r) {
    unsigned long long b = 0;
    for (int64_t u = v0 + tid; u < v1; u += NT)
      for (int64_t j = 8 * u; j < 8 * u + 8 && j < P.V; ++j) {
        const unsigned long long c = key_of(as_f32(x[j]), j);
        if (c < last && c > b) b = c;
      }
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

// Joins the splits of a row: one workgroup of 256 threads per row
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
      finish<T>(P, row, a);
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

// thread = vectors of 8 logits of one row; blockIdx.x = (row, block of 256 kUnroll vectors)
template <class T, bool ENT>
__global__ __launch_bounds__(256) void backward_kernel(Params P, int nblk) {
  const int64_t row = blockIdx.x / nblk;
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
  auto grad = [&](float f, int64_t j) {
    const float l = (f - m) - ln_s, p = __builtin_amdgcn_exp2f(l * kLog2e);
    float d = -g * p;
    if (ENT) d -= h * (p * (below(l) + H));
    return j == t ? d + g : d;
  };
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int64_t j0 = 8 * (v0 + u * 256);
    if (j0 + 8 <= P.V) {
      float d[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = 0.f;
      if (!zero) {
        Vec<T> w;
        w.load(x + j0);
#pragma unroll
        for (int e = 0; e < 8; ++e) d[e] = grad(w.get(e), j0 + e);
      }
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<u32x4_u*>(dx + j0) =
            __builtin_bit_cast(u32x4, cvt8(d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7]));
      } else {
        reinterpret_cast<f32x4_u*>(dx + j0)[0] = f32x4{d[0], d[1], d[2], d[3]};
        reinterpret_cast<f32x4_u*>(dx + j0)[1] = f32x4{d[4], d[5], d[6], d[7]};
      }
    } else {
      for (int64_t j = j0; j < P.V; ++j) dx[j] = (T)(zero ? 0.f : grad(as_f32(x[j]), j));
    }
  }
}

}  // namespace lp
}  // namespace prefixlm
