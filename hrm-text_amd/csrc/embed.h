// Scaled embedding lookup and the gradient of its table (models/lm_head.py:34-43).
//
//   y_i = round(s * T[id_i]),   dT_v = round(s * sum over i with id_i = v of dy_i)
//
// The gradient needs the tokens grouped by id: a stable sort of (id, i), then one pass over the sorted
// tokens that adds the rows of each run in fp32, a chunk of 16 or 32 tokens by a wave, and a second one
// that adds the sums of a run over several chunks, in order. The sort is stable, so the sums have one order
// for the same ids and the result is bitwise deterministic; no atomics touch floating-point data. Where a
// run meets the chunks' borders, and so the order within it, depends on the tokens that sort before it.
#pragma once
#include "common.h"

namespace prefixlm {
namespace emb {

// 8 consecutive elements of a row, 16-byte aligned
template <class T>
struct Row8;
template <>
struct Row8<bf16> {
  u32x4 w;
  __device__ __forceinline__ void load(const bf16* p) { w = *reinterpret_cast<const u32x4*>(p); }
  __device__ __forceinline__ void arrive() { settle(w); }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = bf16lo(w[e]);
      f[2 * e + 1] = bf16hi(w[e]);
    }
  }
  __device__ static __forceinline__ void store(bf16* p, const float* f) {
    *reinterpret_cast<bf16x8*>(p) = cvt8(f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]);
  }
};
template <>
struct Row8<float> {
  f32x4 w[2];
  __device__ __forceinline__ void load(const float* p) {
    w[0] = reinterpret_cast<const f32x4*>(p)[0];
    w[1] = reinterpret_cast<const f32x4*>(p)[1];
  }
  __device__ __forceinline__ void arrive() {
    settle(__builtin_bit_cast(u32x4, w[0]));
    settle(__builtin_bit_cast(u32x4, w[1]));
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = w[e >> 2][e & 3];
  }
  __device__ static __forceinline__ void store(float* p, const float* f) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{f[0], f[1], f[2], f[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{f[4], f[5], f[6], f[7]};
  }
};

struct FwdParams {
  const void* table;
  const void* ids;
  void* y;
  int64_t table_st, y_st, T, V;
  int cols, wide_ids;
  float scale;
};
__device__ __forceinline__ int64_t id_of(const void* ids, int wide, int64_t i) {
  return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int32_t*>(ids)[i];
}

// thread = 8 columns of one token's row. Ids outside the table give NaN rows. Bound by memory: 16384
// rows of 2048 from a table in fp32 to bf16, 201 MB, 36 us, 5.6 TB/s; 64 rows 2.5 us, a launch's time.
template <class TT, class TY>
__global__ __launch_bounds__(256) void lookup_kernel(FwdParams P) {
  const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int c8 = P.cols >> 3;
  const int64_t i = idx / c8;
  if (i >= P.T) return;
  const int c = (int)(idx - i * c8) * 8;
  const int64_t id = id_of(P.ids, P.wide_ids, i);
  float f[8];
  if (id >= 0 && id < P.V) {
    Row8<TT> r;
    r.load(static_cast<const TT*>(P.table) + id * P.table_st + c);
    r.get(f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = __builtin_nanf("");
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] *= P.scale;
  Row8<TY>::store(static_cast<TY*>(P.y) + i * P.y_st + c, f);
}

// ---- the gradient ----------------------------------------------------------------------------
constexpr int kBits = 9, kBins = 1 << kBits;   // a digit; two cover 2^18 ids
constexpr int kSortThreads = 256, kSortWaves = kSortThreads / 64;
constexpr int kMaxTiles = 128;
constexpr int kMinRun = 16;                    // sorted tokens per wave of the sum: 16 or 32 (a lane has one)

struct SortParams {
  const void* ids;          // first pass: the caller's ids; else null
  const uint32_t* key_in;   // later passes
  const uint32_t* pos_in;
  uint32_t* key_out;
  uint32_t* pos_out;
  uint32_t* hist;           // [tiles, kBins]
  void* zero;               // rows to clear beside the sort, and this launch's share of them
  int64_t zero_begin, zero_end;   // in 16-byte units
  int64_t T, V, padding;
  int wide_ids, tile, tiles, shift;
};

// The id as a sort key; ids without a gradient (outside the table, or the padding id) come last
__device__ __forceinline__ uint32_t key_at(const SortParams& P, int64_t i) {
  if (!P.ids) return P.key_in[i];
  const int64_t id = id_of(P.ids, P.wide_ids, i);
  return id >= 0 && id < P.V && id != P.padding ? (uint32_t)id : (uint32_t)P.V;
}

// Workgroups past the sort's `sorting` clear the gradient: the sort is a chain of short steps that
// leaves the memory idle, and the clearing needs nothing from it.
template <int NTH>
__device__ __forceinline__ bool clears(const SortParams& P, int sorting) {
  const int b = (int)blockIdx.x - sorting;
  if (b < 0) return false;
  const int64_t n = (int64_t)(gridDim.x - sorting) * NTH * 4;
  const u32x4 z = {0u, 0u, 0u, 0u};
  u32x4* const to = static_cast<u32x4*>(P.zero);
  for (int64_t i = P.zero_begin + (int64_t)b * NTH * 4 + threadIdx.x; i < P.zero_end; i += n)
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u * NTH < P.zero_end) to[i + u * NTH] = z;
  return true;
}

// The lanes of this wave that are `in` and have this lane's digit: each sets its bit in the digit's
// word of `same` (the wave's own, all zero before and again after), in LDS. Nine ballots and 64-bit
// selects, the way without memory, take three times the instructions.
__device__ __forceinline__ unsigned long long lanes_with(unsigned long long* same, uint32_t digit, bool in, int lane) {
  if (in) atomicOr(&same[digit], 1ull << lane);
  __builtin_amdgcn_wave_barrier();
  const unsigned long long m = in ? same[digit] : 0;
  __builtin_amdgcn_wave_barrier();
  if (in && (m >> lane) == 1ull) same[digit] = 0;
  __builtin_amdgcn_wave_barrier();
  return m;
}

// How many of each digit a tile holds
__global__ __launch_bounds__(kSortThreads) void histogram_kernel(SortParams P) {
  if (clears<kSortThreads>(P, P.tiles)) return;
  __shared__ uint32_t n[kBins];
  for (int d = threadIdx.x; d < kBins; d += kSortThreads) n[d] = 0;
  __syncthreads();
  const int64_t i0 = (int64_t)blockIdx.x * P.tile, i1 = i0 + P.tile < P.T ? i0 + P.tile : P.T;
  for (int64_t i = i0 + threadIdx.x; i < i1; i += kSortThreads)
    atomicAdd(&n[(key_at(P, i) >> P.shift) & (kBins - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < kBins; d += kSortThreads) P.hist[(int64_t)blockIdx.x * kBins + d] = n[d];
}

// Moves a tile's tokens to their places by one digit, keeping their order: the place is the number
// of tokens with a lower digit, plus those of the same digit in earlier tiles, in earlier waves'
// parts of this tile, and before it in its wave's part. Bound by latency and LDS, one step of a wave
// after another.
__global__ __launch_bounds__(kSortThreads) void scatter_kernel(SortParams P) {
  if (clears<kSortThreads>(P, P.tiles)) return;
  static_assert(kBins == 2 * kSortThreads, "a thread has two digits");
  __shared__ uint32_t place[kSortWaves][kBins];
  __shared__ unsigned long long masks[kSortWaves][kBins];
  __shared__ uint32_t wave_sum[kSortWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t i0 = (int64_t)blockIdx.x * P.tile, i1 = i0 + P.tile < P.T ? i0 + P.tile : P.T;
  const int part = P.tile / kSortWaves;                     // a multiple of 64
  const int64_t w0 = i0 + (int64_t)wave * part, w1 = w0 + part < i1 ? w0 + part : i1;
  for (int d = tid; d < kSortWaves * kBins; d += kSortThreads) {
    (&place[0][0])[d] = 0;
    (&masks[0][0])[d] = 0;
  }
  __syncthreads();
  for (int64_t i = w0 + lane; i < w1; i += 64) atomicAdd(&place[wave][(key_at(P, i) >> P.shift) & (kBins - 1)], 1u);
  // digits 2 tid and 2 tid + 1: all tiles' tokens, and those of earlier tiles
  uint32_t all[2] = {0, 0}, before[2] = {0, 0};
  for (int b = 0; b < P.tiles; ++b) {
    const u32x2 h = reinterpret_cast<const u32x2*>(P.hist + (int64_t)b * kBins)[tid];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      all[e] += h[e];
      if (b < (int)blockIdx.x) before[e] += h[e];
    }
  }
  uint32_t sum = all[0] + all[1];
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint32_t y = __shfl_up(sum, m);
    if (lane >= m) sum += y;
  }
  if (lane == 63) wave_sum[wave] = sum;
  __syncthreads();   // the waves' counts too
  uint32_t low = sum - all[0] - all[1];
  for (int g = 0; g < wave; ++g) low += wave_sum[g];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t at = low + before[e];
    if (e) at += all[0];
#pragma unroll
    for (int g = 0; g < kSortWaves; ++g) {
      const uint32_t n = place[g][2 * tid + e];
      place[g][2 * tid + e] = at;
      at += n;
    }
  }
  __syncthreads();
  // each wave takes 64 tokens at a time, lanes with one digit share its place; kHeld of them loaded ahead
  constexpr int kHeld = 8;
  for (int64_t i0w = w0; i0w < w1; i0w += 64 * kHeld) {
    uint32_t key[kHeld], pos[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      const int64_t i = i0w + 64 * u + lane;
      key[u] = i < w1 ? key_at(P, i) : 0;
      pos[u] = i < w1 && !P.ids ? P.pos_in[i] : (uint32_t)i;
    }
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
      if (i0w + 64 * u >= w1) continue;
      const bool in = i0w + 64 * u + lane < w1;
      const uint32_t digit = (key[u] >> P.shift) & (kBins - 1);
      const uint32_t first = place[wave][digit];
      const unsigned long long same = lanes_with(masks[wave], digit, in, lane);
      if (in) {
        const uint32_t at = first + (uint32_t)__builtin_popcountll(same & ((1ull << lane) - 1));
        P.key_out[at] = key[u];
        P.pos_out[at] = pos[u];
        // the last lane of each digit moves its place on
        if ((same >> lane) == 1ull) place[wave][digit] = first + (uint32_t)__builtin_popcountll(same);
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// The whole sort in one launch, for up to 2^14 tokens and ids below 2^18: a token is one word, id <<
// 14 | i, and its place is the number of smaller words. Workgroup = `tile` tokens, 16 to 64 of them, so
// that there are up to one for each CU; its 16 waves hold 64 R of all words each, and one compare of a
// token's word (a scalar) with 64 of them, whose lanes are counted as scalars, is all that a token and
// 64 others take: bound by those compares and counts, T^2 / 64 (16384 tokens, with 32 MB cleared
// beside them, 32 us, 4999 11). A radix sort in one workgroup took 35 to 45 us for 16384, bound by
// LDS, one in four launches 28 without the clearing.
constexpr int kRankBits = 14, kRankThreads = 1024, kRankWaves = kRankThreads / 64;
constexpr int64_t kRankTokens = 1 << kRankBits, kRankIds = ((int64_t)1 << (32 - kRankBits)) - 1;

template <int R>
__global__ __launch_bounds__(kRankThreads) __attribute__((amdgpu_waves_per_eu(8, 8))) void rank_kernel(SortParams P) {
  if (clears<kRankThreads>(P, P.tiles)) return;
  __shared__ int count[kRankWaves][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int T = (int)P.T, per = P.tile, i = blockIdx.x * per + lane;
  const bool in = lane < per && i < T;
  uint32_t x[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int j = (wave * R + r) * 64 + lane;
    x[r] = j < T ? key_at(P, j) << kRankBits | (uint32_t)j : 0xffffffffu;   // above every token's
  }
  const uint32_t mine = in ? key_at(P, i) << kRankBits | (uint32_t)i : 0xffffffffu;
  int n = 0;
  for (int l0 = 0; l0 < per; l0 += 2) {
#pragma unroll
    for (int l = l0; l < l0 + 2; ++l) {
      const uint32_t w = (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
      int c = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(x[r] < w));
      n = lane == l ? c : n;
    }
  }
  count[wave][lane] = n;
  __syncthreads();
  if (wave == 0 && in) {
    int at = 0;
#pragma unroll
    for (int g = 0; g < kRankWaves; ++g) at += count[g][lane];
    P.key_out[at] = mine >> kRankBits;
    P.pos_out[at] = (uint32_t)i;
  }
}

struct SumParams {
  const uint32_t* key;
  const uint32_t* pos;
  const void* dy;
  void* grad;
  float* part;              // [chunks, 2, cols]: the runs that a chunk's first and last token belong to
  int64_t dy_st, T, V;
  int cols, chunks, run;
  float scale;
};

// Wave = (chunk of `run` sorted tokens, 512 columns). Runs that lie inside the chunk are written; a
// run that goes on in a neighbour leaves its sum in `part` (slot 0: the run the chunk begins with,
// if it began earlier; slot 1: the run that goes on behind it, if it began here). Bound by latency, a
// chain of keys, rows and stores, up to some 10000 tokens x 512 (8.4 us), and by memory then: 16384 x
// 2048 bf16 rows into a table in fp32 42 us, while the cleared table goes from the last-level cache
// to memory.
template <class TY, class TG>
__global__ __launch_bounds__(256) void sum_kernel(SumParams P) {
  const int cblk = (P.cols + 511) / 512, lane = threadIdx.x & 63;
  const int64_t w = __builtin_amdgcn_readfirstlane((int)((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int chunk = (int)(w / cblk);
  if (chunk >= P.chunks) return;
  const int c = (int)(w - (int64_t)chunk * cblk) * 512 + lane * 8;
  const bool on = c < P.cols;
  const int64_t t0 = (int64_t)chunk * P.run;
  const int n = (int)(P.T - t0 < P.run ? P.T - t0 : P.run);
  const uint32_t key = lane < n ? P.key[t0 + lane] : (uint32_t)P.V;
  const uint32_t pos = lane < n ? P.pos[t0 + lane] : 0;
  const uint32_t prev = t0 > 0 ? P.key[t0 - 1] : 0xffffffffu;
  const uint32_t next = t0 + P.run < P.T ? P.key[t0 + P.run] : 0xffffffffu;
  float acc[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] = 0.f;
  bool first = true;                 // still in the run that the chunk begins with
  const TY* dy = static_cast<const TY*>(P.dy) + c;
  constexpr int kAhead = 8;
  for (int t = 0; t < n; t += kAhead) {
    Row8<TY> r[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int64_t p = (uint32_t)__builtin_amdgcn_readlane((int)pos, t + u < n ? t + u : t);
      if (on) r[u].load(dy + p * P.dy_st);
    }
    // all at once here: a wait for the next token's row would be one for this token's stores too
#pragma unroll
    for (int u = 0; u < kAhead; ++u) r[u].arrive();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (t + u >= n) break;
      const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)key, t + u);
      if (k >= (uint32_t)P.V) return;   // the last ones have no gradient
      float f[8];
      if (on) r[u].get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f[e];
      const bool last = t + u == n - 1;
      const uint32_t k1 = last ? next : (uint32_t)__builtin_amdgcn_readlane((int)key, t + u + 1);
      if (k1 == k && !last) continue;
      const bool from_before = first && k == prev, goes_on = k1 == k;
      if (on) {
        if (from_before || goes_on) {
          float* p = P.part + ((int64_t)chunk * 2 + (from_before ? 0 : 1)) * P.cols + c;
          Row8<float>::store(p, acc);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[e] *= P.scale;
          Row8<TG>::store(static_cast<TG*>(P.grad) + (int64_t)k * P.cols + c, acc);
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      first = false;
    }
  }
}

// Wave = (chunk, 512 columns): the run that goes on behind the chunk, if it began there, is added up
// over the following chunks, in order; how many there are is searched with 64 lanes at a time. Bound by
// latency (3 to 7 us): the longest run is one wave's chain of its partials, eight in flight.
template <class TG>
__global__ __launch_bounds__(256) void join_kernel(SumParams P) {
  const int cblk = (P.cols + 511) / 512, lane = threadIdx.x & 63;
  const int64_t w = __builtin_amdgcn_readfirstlane((int)((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int chunk = (int)(w / cblk);
  if (chunk >= P.chunks - 1) return;
  const int c = (int)(w - (int64_t)chunk * cblk) * 512 + lane * 8;
  const int64_t t1 = (int64_t)(chunk + 1) * P.run;   // the next chunk's first token
  const uint32_t k = P.key[t1 - 1];
  if (k >= (uint32_t)P.V || P.key[t1] != k) return;
  if (chunk > 0 && P.key[t1 - P.run] == k && P.key[t1 - P.run - 1] == k) return;   // it began earlier
  // the chunks after this one that it reaches: those whose first token is k's
  int end = chunk + 2;
  for (;;) {
    const bool more = end + lane < P.chunks && P.key[(int64_t)(end + lane) * P.run] == k;
    const unsigned long long not_k = ~__builtin_amdgcn_ballot_w64(more);
    if (not_k) {
      end += (int)__builtin_ctzll(not_k);
      break;
    }
    end += 64;
  }
  if (c >= P.cols) return;
  float acc[8];
  Row8<float> r;
  r.load(P.part + ((int64_t)chunk * 2 + 1) * P.cols + c);
  r.get(acc);
  constexpr int kAhead = 8;
  for (int g = chunk + 1; g < end; g += kAhead) {
    Row8<float> ahead[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) ahead[u].load(P.part + (int64_t)(g + u < end ? g + u : end - 1) * 2 * P.cols + c);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float f[8];
      ahead[u].get(f);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = g + u < end ? acc[e] + f[e] : acc[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= P.scale;
  Row8<TG>::store(static_cast<TG*>(P.grad) + (int64_t)k * P.cols + c, acc);
}

}  // namespace emb
}  // namespace prefixlm
