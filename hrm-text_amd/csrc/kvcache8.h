// KV-cache attention over a cache held in 8 bits, with one scale for each 64 rows and head.
//
// The cache of one (batch row, head), head-major so that a head's rows are contiguous:
//   codes   [Smax, 128]     e4m3 or int8: row j of a complete block (64 rows) is scale * code
//   scale   [Smax / 64]     fp32: largest magnitude of the block times fp32(1/448) (e4m3) or
//                           fp32(1/127) (int8), at least 2^-126; a block that holds an infinity
//                           or NaN gets such a scale
//   recent  [128, 128]      bf16: row j of the last 64 to 127 rows in slot j % 128, as given
// A row is rounded to 8 bits once, from its bf16 value, when its block is complete, so the cache's
// content does not depend on how many rows each call brought. The ring also lets a caller take rows
// back, to one block before the incomplete one of the furthest length that the cache has had: the rows of
// the block that is incomplete again are still there. A multiple of 64 reads no ring rows.
//
// A call with len rows in the cache attends: rows below len / 64 * 64 from the codes, the rest
// below len from the ring, and the call's new rows as given, so nothing reads what the call writes.
//
// Kernels:
//   decode  : one query per row; as kvcache.h's, with half the bytes per key: 8 lanes hold a key's
//             128 codes, 16 bytes each. The workgroup of the last split also takes the bf16 rows
//             and the new one, puts that one into the ring and rounds a block it completes;
//   extend  : several queries per row, on the matrix cores: codes become bf16 on their way into
//             LDS, exactly; the scales go to the scores and, for V, to the probabilities;
//   append  : new rows of an extend or prefill into ring, codes and scales: beside the attention of up
//             to 64 rows, behind that of more.
// The splits' partials and their combine are kvcache.h's.
#pragma once
#include "common.h"
#include "kvcache.h"

namespace prefixlm {
namespace kv8 {

using kvc::D;
using kvc::ExtGeo;
using kvc::kPart;
using kvc::max_mag;
using kvc::max_ref;
using kvc::row_inv;
constexpr int NT = kvc::NT;
constexpr int kBlock = 64;     // rows that share a scale
constexpr int kRing = 128;     // rows kept in bf16

struct Params {
  const bf16* q;
  const bf16* k;          // new rows (may be null)
  const bf16* v;
  uint8_t* kc;
  uint8_t* vc;
  float* ks;
  float* vs;
  bf16* kr;
  bf16* vr;
  bf16* out;
  float* part;            // [B, S, H, nsplit, kPart]
  const int32_t* seqlens; // device [B]; null: every row has seqlen_const
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh;
  int B, S, H, Smax, nsplit, causal, seqlen_const;
  int s_new;              // rows appended by this call: S, or 0 without new k, v
  int nqb;                // extend: query blocks of 32 QW rows
  int n_main, touched;    // extend: workgroups from n_main on append, `touched` blocks per (b, h)
  float scale_log2;
};

__device__ __forceinline__ int cache_len(const Params& P, int b) {
  return min(max(P.seqlens ? P.seqlens[b] : P.seqlen_const, 0), P.Smax);
}
// The keys that query i sees of a cache row of length len: [0, n)
__device__ __forceinline__ int keys_seen(const Params& P, int len, int i) {
  const int lk = min(P.Smax, len + P.s_new);
  return P.causal ? min(lk, len + P.s_new - P.S + i + 1) : lk;
}

// ---- the two code types ------------------------------------------------------------------
struct E4M3 {
  static constexpr float kInvMax = 1.f / 448.f;
  // 4 codes as fp32
  __device__ static __forceinline__ void get(uint32_t w, float* f) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    f[0] = a[0], f[1] = a[1], f[2] = b[0], f[3] = b[1];
  }
  // round to nearest, ties to even; |f| <= 448
  __device__ static __forceinline__ uint32_t put(const float* f) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], w, true);
  }
};
struct Int8 {
  static constexpr float kInvMax = 1.f / 127.f;
  __device__ static __forceinline__ void get(uint32_t w, float* f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = (float)lo_byte(w, e);
  }
  // NaN and infinities (of blocks whose scale says so already) become 0
  __device__ static __forceinline__ uint32_t put(const float* f) {
    uint32_t w = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float r = __builtin_rintf(f[e]);
      const int c = __builtin_fabsf(r) <= 127.f ? (int)r : 0;
      w |= ((uint32_t)c & 0xffu) << (8 * e);
    }
    return w;
  }
};
// 8 codes as 8 bf16, exactly
template <class C>
__device__ __forceinline__ u32x4 codes_bf16(const u32x2& w) {
  float f[8];
  C::get(w[0], f);
  C::get(w[1], f + 4);
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = pack_hi(__builtin_bit_cast(uint32_t, f[2 * i]), __builtin_bit_cast(uint32_t, f[2 * i + 1]));
  return r;
}
// The scale of a block whose largest magnitude, as bf16 bits, is mag (NaN above infinity above all)
template <class C>
__device__ __forceinline__ float block_scale(uint32_t mag) {
  const float s = __builtin_bit_cast(float, mag << 16) * C::kInvMax;
  return s < 0x1p-126f ? 0x1p-126f : s;   // NaN stays
}

// x / s for many x, correctly rounded, with a few operations each where the compiler's division takes
// a dozen (the rounding of 2 x 16 x 1021 rows 11.2 -> 9.4 us): y = 1 / s rounded
// (one Newton step from the 1-ulp reciprocal), q = x y, and q + (x - q s) y rounds to x / s as long as
// the residual x - q s is exact, which a scale below 2^-60 is multiplied up for. Scales and rows come
// from bf16, so there are 128 mantissas of each: the tests take them all. By an infinite scale, whose
// steps would end in 0 * inf, finite x give 0 and others NaN: s = y = 0.
struct Divisor {
  float s, y, up;
  __device__ __forceinline__ explicit Divisor(float scale) {
    up = scale < 0x1p-60f ? 0x1p64f : 1.f;
    s = scale * up;
    const float y0 = __builtin_amdgcn_rcpf(s);
    y = __builtin_fmaf(__builtin_fmaf(-s, y0, 1.f), y0, y0);
    if (scale == INFINITY) s = y = 0.f;
  }
  __device__ __forceinline__ float divides(float x) const {
    x *= up;
    const float q = x * y;
    return __builtin_copysignf(__builtin_fmaf(__builtin_fmaf(-q, s, x), y, q), x);   // -0 stays
  }
};

// ---- taking rows into the cache ------------------------------------------------------------
// The workgroup rounds the complete block `blk` of (b, h), whose row j is row(j) (256 bytes of
// bf16), into 8 bits: threads of 16 columns, NTH / 8 rows at a time.
template <class C, int NTH, class Row>
__device__ __forceinline__ void round_block(uint8_t* codes, float* scale, int blk, uint32_t* s_mag, Row row) {
  constexpr int R = kBlock / (NTH / 8);
  const int tid = threadIdx.x, g = tid >> 3, c = 16 * (tid & 7);
  u32x4 x[R][2];
  u16x2 m = {0, 0};
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const u32x4* p = reinterpret_cast<const u32x4*>(row(blk * kBlock + r * (NTH / 8) + g) + c);
    x[r][0] = p[0];
    x[r][1] = p[1];
    m = max_mag(max_mag(m, x[r][0]), x[r][1]);
  }
  uint32_t mag = max((uint32_t)m[0], (uint32_t)m[1]);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) mag = max(mag, (uint32_t)__shfl_xor((int)mag, s));
  __syncthreads();   // s_mag may be in use by the block before
  if ((tid & 63) == 0) s_mag[tid >> 6] = mag;
  __syncthreads();
  mag = s_mag[0];
#pragma unroll
  for (int g2 = 1; g2 < NTH / 64; ++g2) mag = max(mag, s_mag[g2]);
  const float s = block_scale<C>(mag);
  if (tid == 0) scale[blk] = s;
  const Divisor by(s);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t y = x[r][i >> 1][2 * (i & 1) + e];
        f[2 * e] = by.divides(bf16lo(y));
        f[2 * e + 1] = by.divides(bf16hi(y));
      }
      w[i] = C::put(f);
    }
    *reinterpret_cast<u32x4*>(codes + ((int64_t)blk * kBlock + r * (NTH / 8) + g) * D + c) = w;
  }
}

// Workgroup `wg` = (b, h, touched block, keys or values): rounds its block if it is complete now; the
// first touched block's also puts the last rows into the ring, after it has read the ring's old rows.
template <class C, int NTH = NT>
__device__ __forceinline__ void append(const Params& P, int wg, int nblk, uint32_t* s_mag) {
  const int n = wg & 1, bh = (wg >> 1) / nblk, i = (wg >> 1) - bh * nblk;
  const int b = bh / P.H, h = bh - b * P.H;
  const int len = cache_len(P, b), end = min(P.Smax, len + P.s_new);
  const int blk = len / kBlock + i;
  bf16* const ring = (n ? P.vr : P.kr) + (int64_t)bh * kRing * D;
  const bf16* const fresh = n ? P.v + b * P.v_sb + h * P.v_sh : P.k + b * P.k_sb + h * P.k_sh;
  const int64_t st = n ? P.v_ss : P.k_ss;
  if (blk < end / kBlock)
    round_block<C, NTH>((n ? P.vc : P.kc) + (int64_t)bh * P.Smax * D, (n ? P.vs : P.ks) + (int64_t)bh * (P.Smax / kBlock),
                        blk, s_mag, [&](int j) { return j < len ? ring + (j & (kRing - 1)) * D : fresh + (j - len) * st; });
  if (i) return;
  __syncthreads();   // every thread has read the ring
  const int j0 = max(len, end / kBlock * kBlock - kBlock), c = 8 * (threadIdx.x & 15);
  for (int j = j0 + (threadIdx.x >> 4); j < end; j += NTH / 16)
    *reinterpret_cast<u32x4*>(ring + (j & (kRing - 1)) * D + c) =
        *reinterpret_cast<const u32x4*>(fresh + (j - len) * st + c);
}
// A thread has 16 columns of one row: bound by its chain of loads, maximum, barrier and stores (2 x 16
// heads x 1021 rows, 25 MB: 8.9 us, 9.8 with two rows a thread, 12.2 with four; as workgroups of the
// prefill's launch, whose LDS and registers let few of them run at once, 3 us more than so).
constexpr int kAppendThreads = 512;
template <class C>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(Params P, int nblk) {
  __shared__ uint32_t s_mag[kAppendThreads / 64];
  append<C, kAppendThreads>(P, blockIdx.x, nblk, s_mag);
}

// ---- one query per row ------------------------------------------------------------------------
__device__ __forceinline__ float row8_sum(float x) {   // over each 8 lanes
  x += dpp_f<0xB1>(x);
  x += dpp_f<0x4E>(x);
  x += dpp_f<0x141>(x);
  return x;
}

// blockIdx.x = (b * H + h) * nsplit + split. The splits share the complete blocks evenly; the last
// one has the fewest and takes the bf16 rows too. kSlots keys in flight per 8 lanes. Bound by memory
// where pairs are many (64 x 16 pairs on 3003 rows, 799 MB, 129 us, 6.2 TB/s, which is above what a
// copy reaches), by latency where they are few (16 pairs on 783 rows 8.0 us).
template <class C, int NTH>
__global__ __launch_bounds__(NTH) void decode_kernel(Params P) {
  constexpr int NWAVE = NTH / 64, G = NTH / 8, kSlots = 4, kStep = G * kSlots;
  static_assert(kStep % kBlock == 0, "steps of whole blocks");
  __shared__ float s_m[NWAVE], s_l[NWAVE];
  __shared__ f32x4 s_o[NWAVE][D / 4];
  __shared__ uint32_t s_mag[NWAVE];
  const int split = blockIdx.x % P.nsplit, bh = blockIdx.x / P.nsplit;
  const int h = bh % P.H, b = bh / P.H;
  const int tid = threadIdx.x, grp = tid >> 3, g8 = tid & 7;
  const int len = cache_len(P, b), nb = len / kBlock, nfull = nb * kBlock;
  const int per = (nb + P.nsplit - 1) / P.nsplit * kBlock;
  const int k0 = min(nfull, split * per), k1 = min(nfull, k0 + per);
  const uint8_t* kbase = P.kc + (int64_t)bh * P.Smax * D + 16 * g8;
  const uint8_t* vbase = P.vc + (int64_t)bh * P.Smax * D + 16 * g8;
  const float* ksc = P.ks + (int64_t)bh * (P.Smax / kBlock);
  const float* vsc = P.vs + (int64_t)bh * (P.Smax / kBlock);
  u32x4 kw[kSlots], vw[kSlots];
  float kf[kSlots], vf[kSlots];
  auto load = [&](int j0) {   // j0: the group's first key of the step
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
      const int j = min(j0 + u * G, k1 - 1);   // clamped rows are masked below
      kw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(kbase + (int64_t)j * D));
      vw[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(vbase + (int64_t)j * D));
      kf[u] = ksc[j / kBlock];
      vf[u] = vsc[j / kBlock];
    }
  };
  if (k0 + grp < k1) load(k0 + grp);
  float q[16];
  {
    const u32x4* p = reinterpret_cast<const u32x4*>(P.q + b * P.q_sb + h * P.q_sh + 16 * g8);
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const u32x4 w = p[n];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        q[8 * n + 2 * e] = bf16lo(w[e]) * P.scale_log2;
        q[8 * n + 2 * e + 1] = bf16hi(w[e]) * P.scale_log2;
      }
    }
  }
  float m = -INFINITY, l = 0.f, o[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] = 0.f;
  for (int j0 = k0 + grp; j0 < k1; j0 += kStep) {
    float s[kSlots], mx = m;
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[4];
        C::get(kw[u][i], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) d += q[4 * i + e] * f[e];
      }
      d = row8_sum(d) * kf[u];
      s[u] = j0 + u * G < k1 ? d : -INFINITY;
      mx = fmaxf(mx, s[u]);
    }
    const float ref = max_ref(mx), alpha = __builtin_amdgcn_exp2f(m - ref);   // m = -inf at first: 0
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] *= alpha;
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
      const float p = __builtin_amdgcn_exp2f(s[u] - ref);
      l += p;
      // a clamped row weighs nothing, whatever its scale
      const float pv = j0 + u * G < k1 ? p * vf[u] : 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float f[4];
        C::get(vw[u][i], f);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * i + e] += pv * f[e];
      }
    }
    m = mx;
    if (j0 + kStep < k1) load(j0 + kStep);
  }
  const bool fresh = P.s_new && len < P.Smax;
  bf16* const kr = P.kr + (int64_t)bh * kRing * D;
  bf16* const vr = P.vr + (int64_t)bh * kRing * D;
  const bf16* const kn = P.k + b * P.k_sb + h * P.k_sh;
  const bf16* const vn = P.v + b * P.v_sb + h * P.v_sh;
  const bool tail = split == P.nsplit - 1;
  if (tail) {
    // the bf16 rows behind the blocks, and the new one
    for (int j = nfull + grp; j < len + (fresh ? 1 : 0); j += G) {
      const u32x4* kp = reinterpret_cast<const u32x4*>((j < len ? kr + (j & (kRing - 1)) * D : kn) + 16 * g8);
      const u32x4* vp = reinterpret_cast<const u32x4*>((j < len ? vr + (j & (kRing - 1)) * D : vn) + 16 * g8);
      const u32x4 k2[2] = {kp[0], kp[1]}, v2[2] = {vp[0], vp[1]};
      float d = 0.f;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          d += q[8 * n + 2 * e] * bf16lo(k2[n][e]) + q[8 * n + 2 * e + 1] * bf16hi(k2[n][e]);
      d = row8_sum(d);
      const float mx = fmaxf(m, d), ref = max_ref(mx);
      const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(d - ref);
      m = mx;
      l = l * alpha + p;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[8 * n + 2 * e] = o[8 * n + 2 * e] * alpha + p * bf16lo(v2[n][e]);
          o[8 * n + 2 * e + 1] = o[8 * n + 2 * e + 1] * alpha + p * bf16hi(v2[n][e]);
        }
    }
  }
  // merge the wave's eight groups, then the waves
  float M = m;
#pragma unroll
  for (int x = 8; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
  const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
  l *= a;
#pragma unroll
  for (int e = 0; e < 16; ++e) o[e] *= a;
#pragma unroll
  for (int x = 8; x < 64; x <<= 1) {
    l += __shfl_xor(l, x);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] += __shfl_xor(o[e], x);
  }
  const int w = tid >> 6;
  if ((tid & 63) < 8) {
    if (g8 == 0) {
      s_m[w] = M;
      s_l[w] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s_o[w][4 * g8 + i] = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
  }
  __syncthreads();
  if (tid < D / 4) {
    M = s_m[0];
#pragma unroll
    for (int g = 1; g < NWAVE; ++g) M = fmaxf(M, s_m[g]);
    float L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NWAVE; ++g) {
      const float wgt = s_m[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[g] - M);
      L += wgt * s_l[g];
      acc += wgt * s_o[g][tid];
    }
    if (P.nsplit == 1) {
      const float inv = row_inv(keys_seen(P, len, 0), L);
      *reinterpret_cast<bf16x4*>(P.out + b * P.o_sb + h * P.o_sh + 4 * tid) =
          cvt4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    } else {
      float* dst = P.part + (((int64_t)b * P.H + h) * P.nsplit + split) * kPart;
      if (tid == 0) {
        dst[0] = M;
        dst[1] = L;
      }
      *reinterpret_cast<f32x4*>(dst + 4 + 4 * tid) = acc;
    }
  }
  if (!(tail && fresh)) return;
  // the cache takes the new row
  if ((len & (kBlock - 1)) == kBlock - 1) {
#pragma unroll 1
    for (int n = 0; n < 2; ++n) {
      const bf16 *const ring = n ? vr : kr, *const now = n ? vn : kn;
      round_block<C, NTH>((n ? P.vc : P.kc) + (int64_t)bh * P.Smax * D, (n ? P.vs : P.ks) + (int64_t)bh * (P.Smax / kBlock),
                          nb, s_mag, [&](int j) { return j < len ? ring + (j & (kRing - 1)) * D : now; });
    }
  }
  if (tid < 32) {
    const int c = 8 * (tid & 15);
    *reinterpret_cast<u32x4*>((tid & 16 ? vr : kr) + (len & (kRing - 1)) * D + c) =
        *reinterpret_cast<const u32x4*>((tid & 16 ? vn : kn) + c);
  }
}

// ---- several queries per row --------------------------------------------------------------------
// Queries [q0, q1) over keys [k0, k1) without the matrix cores: a 16-lane group per query, key by
// key, for blocks whose values, scales or scores are not finite or whose scores could pass fp32's
// range before they are scaled: on the matrix cores 0 * inf would reach queries that must not see
// the key. row(j, n, f, &unit): this lane's 8 columns of key (n = 0) or value (n = 1) j are unit * f.
template <class KMax, class Row>
__device__ __forceinline__ void extend_block_valu(const Params& P, int b, int h, int split, int q0, int q1, int k0,
                                                  int k1, KMax kmax, Row row) {
  constexpr int GROUPS = NT / 16;
  const int g16 = threadIdx.x & 15;
#pragma unroll 1
  for (int i = q0 + (threadIdx.x >> 4); i < q1; i += GROUPS) {
    float q[8], o[8];
    const u32x4 qv = *reinterpret_cast<const u32x4*>(P.q + b * P.q_sb + i * P.q_ss + h * P.q_sh + 8 * g16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      q[2 * e] = bf16lo(qv[e]) * P.scale_log2;
      q[2 * e + 1] = bf16hi(qv[e]) * P.scale_log2;
      o[2 * e] = o[2 * e + 1] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int j = k0; j < min(k1, kmax(i)); ++j) {
      float k[8], v[8], ku, vu, s = 0.f;
      row(j, 0, k, &ku);
      row(j, 1, v, &vu);
#pragma unroll
      for (int e = 0; e < 8; ++e) s += q[e] * k[e];
      s = row16_sum(s) * ku;
      const float mx = fmaxf(m, s), ref = max_ref(mx);
      const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(s - ref);
      m = mx;
      l = l * alpha + p;
      const float pv = p * vu;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = o[e] * alpha + pv * v[e];
    }
    if (P.nsplit == 1) {
      const float inv = row_inv(kmax(i), l);
      *reinterpret_cast<bf16x8*>(P.out + b * P.o_sb + i * P.o_ss + h * P.o_sh + 8 * g16) =
          cvt8(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv, o[4] * inv, o[5] * inv, o[6] * inv, o[7] * inv);
    } else {
      float* dst = P.part + ((((int64_t)b * P.S + i) * P.H + h) * P.nsplit + split) * kPart;
      if (g16 == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{m, l, 0.f, 0.f};
      *reinterpret_cast<f32x4*>(dst + 4 + 8 * g16) = f32x4{o[0], o[1], o[2], o[3]};
      *reinterpret_cast<f32x4*>(dst + 8 + 8 * g16) = f32x4{o[4], o[5], o[6], o[7]};
    }
  }
}

// Workgroup = (b, h, 32 QW queries, split of the keys), waves and tiles as in kvcache.h. A strip of
// 16 staged rows is either codes or bf16 rows, and the 32 keys that a wave multiplies at a time
// have one scale, as blocks begin at multiples of 64.
//
// The probabilities, times the values' scale, go into P V as three bf16 terms, which add up to the 24 bits
// of the fp32 value, as in kvcache.h. Two, each cut, take less (4 x 16 heads x 45 queries on 2000 rows 24.2
// us, with three 25.5; 2 x 12 x 256 on 10500 84.3 and 94.2) but leave up to 2^-15 of each probability, all
// towards zero, which sums that cancel show.
// Bound by each wave's chain of LDS, products and exponentials, and for few tiles by what a split costs
// once: its first loads, the join of the key groups, its partials. 64 pairs x 45 queries, ten splits: on 2000
// rows 21.8 us, on 4000 33.4, so 11.6 for each 2000 rows and 10 besides, and the combine 4.6; 24 x 100, 21
// splits: on 5250 rows 29.7, on 10500 46.1, 16.4 for each 5250 and 13 besides, combine 6.9, append 4.9; 24 x
// 256, ten splits: 52.9 and 86.8, 34 and 19, 8.7, 5.1. Fewer address operations change nothing.
constexpr int kTerms = 3;
template <class C, int QW>
__global__ __launch_bounds__(NT, 2) void extend_kernel(Params P) {
  using G = ExtGeo<QW>;
  constexpr int KW = G::KW, TK = G::TK, TILE = G::TILE, NS = D / 16, NP = TK / 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int bad;   // some value, scale or score is not finite, or a score could not be formed
  __shared__ uint32_t s_mag[NT / 64];
  // Up to 64 new rows go into the cache beside the attention, which reads none of what this writes: the
  // blocks they complete begin at or behind the first one it takes in bf16, and the ring rows that
  // it reads, from that block's first on, are less than 128 before the last new one.
  if ((int)blockIdx.x >= P.n_main) {
    append<C>(P, (int)blockIdx.x - P.n_main, P.touched, s_mag);
    return;
  }
  // unit u = (b, h, split); its query blocks sit 8 grid indices apart, on one XCD
  const int qb = (blockIdx.x >> 3) % P.nqb;
  const int u = (int)((blockIdx.x >> 3) / P.nqb) * 8 + (blockIdx.x & 7);
  if (u >= P.B * P.H * P.nsplit) return;
  const int split = u % P.nsplit, bh = u / P.nsplit;
  const int h = bh % P.H, b = bh / P.H;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = w % QW, kw = w / QW;
  const int len = cache_len(P, b);
  const int lk = min(P.Smax, len + P.s_new);      // keys in the cache after the append
  const int q0 = qb * 32 * QW;
  // query i sees keys [0, kmax(i))
  auto kmax = [&](int i) { return keys_seen(P, len, i); };
  const int per = ((lk + P.nsplit - 1) / P.nsplit + TK - 1) / TK * TK;   // keys per split, whole tiles
  const int k0 = split * per;
  const int k1 = min(kmax(min(P.S, q0 + 32 * QW) - 1), k0 + per);
  const int kall = kmax(q0);                      // keys below are seen by every query of the block
  const int qrow = q0 + 32 * qw + l32;            // this lane's query
  const bool active = q0 + 32 * qw < P.S;
  const int kq = min(k1, kmax(min(qrow, P.S - 1)));
  const int kend_w = active ? min(k1, kmax(min(P.S, q0 + 32 * qw + 32) - 1)) : 0;

  const int nfull = len / kBlock * kBlock;        // rows held as codes
  const uint8_t* const kc = P.kc + (int64_t)bh * P.Smax * D;
  const uint8_t* const vc = P.vc + (int64_t)bh * P.Smax * D;
  const float* const ksc = P.ks + (int64_t)bh * (P.Smax / kBlock);
  const float* const vsc = P.vs + (int64_t)bh * (P.Smax / kBlock);
  const bf16* const kr = P.kr + (int64_t)bh * kRing * D;
  const bf16* const vr = P.vr + (int64_t)bh * kRing * D;
  const bf16* const kn = P.k + b * P.k_sb + h * P.k_sh;
  const bf16* const vn = P.v + b * P.v_sb + h * P.v_sh;
  // row j >= nfull of the keys or the values
  auto k_row = [&](int j) { return j < len ? kr + (j & (kRing - 1)) * D : kn + (j - len) * P.k_ss; };
  auto v_row = [&](int j) { return j < len ? vr + (j & (kRing - 1)) * D : vn + (j - len) * P.v_ss; };

  // staging: thread = 16-byte chunk sch of rows srow + 16 r; V rows in permuted order
  const int srow = tid >> 4, sch = tid & 15, vrow = perm_row(srow);
  // Rows past k1 are loaded as the last one below it and masked; a row has its first 8 bytes loaded, all
  // of a code row's, and a bf16 row the others. So no register is written on two paths, and all loads
  // of a tile are on their way together until the tile is stored (as 16 bytes on two paths, with
  // zeroed registers past k1, every 16 rows waited for those before them: 4 x 16 heads x 45 queries on
  // 2000 rows 28.0 us, so 24.3; 16 x 16 x 32 on 2157 92.8 and 61.8; both with two terms of P).
  // pointers that meet from two paths have to say that they are of global memory, or the loads do not know
  typedef const __attribute__((address_space(1))) char* gbytes;
  typedef const __attribute__((address_space(1))) u32x2* gu32x2;
  u32x2 klo[NP], khi[NP], vlo[NP], vhi[NP];
  float next_k, next_v;   // the scales of this wave's 32 keys of the tile
  auto load_kv = [&](int t0) {
    gbytes pk[NP], pv[NP];
    const bool coded = t0 + TK <= nfull;
    if (coded) {
#pragma unroll
      for (int r = 0; r < NP; ++r) {
        pk[r] = (gbytes)(kc + (int64_t)min(t0 + 16 * r + srow, k1 - 1) * D + 8 * sch);
        pv[r] = (gbytes)(vc + (int64_t)min(t0 + 16 * r + vrow, k1 - 1) * D + 8 * sch);
      }
    } else {
#pragma unroll
      for (int r = 0; r < NP; ++r) {
        const int jk = min(t0 + 16 * r + srow, k1 - 1), jv = min(t0 + 16 * r + vrow, k1 - 1);
        pk[r] = jk < nfull ? (gbytes)(kc + (int64_t)jk * D + 8 * sch)
                           : (gbytes)(k_row(jk) + 8 * sch);
        pv[r] = jv < nfull ? (gbytes)(vc + (int64_t)jv * D + 8 * sch)
                           : (gbytes)(v_row(jv) + 8 * sch);
      }
    }
#pragma unroll
    for (int r = 0; r < NP; ++r) {
      klo[r] = *(gu32x2)(pk[r]);
      vlo[r] = *(gu32x2)(pv[r]);
    }
    if (!coded) {
#pragma unroll
      for (int r = 0; r < NP; ++r) {   // a code row's bytes again, unused
        khi[r] = *(gu32x2)(pk[r] + (min(t0 + 16 * r, k1 - 1) < nfull ? 0 : 8));
        vhi[r] = *(gu32x2)(pv[r] + (min(t0 + 16 * r, k1 - 1) < nfull ? 0 : 8));
      }
    }
    const int blk = max(min(t0 + 32 * kw, nfull - 1), 0) / kBlock;
    next_k = ksc[blk];
    next_v = vsc[blk];
  };
  auto store_kv = [&](int buf, int t0) {
    char* base = smem + buf * G::BUF + srow * RS + sch * 16;
    u32x4 vs[NP];
#pragma unroll
    for (int r = 0; r < NP; ++r) {
      // a strip whose first row is clamped is one whose rows all are: its codes or rows are the last one's
      u32x4 k;
      if (min(t0 + 16 * r, k1 - 1) < nfull) {
        k = codes_bf16<C>(klo[r]);
        vs[r] = codes_bf16<C>(vlo[r]);
      } else {
        k = u32x4{klo[r][0], klo[r][1], khi[r][0], khi[r][1]};
        vs[r] = u32x4{vlo[r][0], vlo[r][1], vhi[r][0], vhi[r][1]};
      }
      *reinterpret_cast<u32x4*>(base + 16 * r * RS) = k;
      *reinterpret_cast<u32x4*>(base + TILE + 16 * r * RS) = vs[r];
    }
    u16x2 m = {0, 0};
#pragma unroll
    for (int r = 0; r < NP; ++r) m = max_mag(m, vs[r]);
    if (m[0] >= 0x7f80 || m[1] >= 0x7f80) bad = 1;
  };

  float m_run = -INFINITY, l_run = 0.f;
  f32x16 oacc[4];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[t][r] = 0.f;

  if (k0 < k1) {
    const int nt = (k1 - k0 + TK - 1) / TK;
    load_kv(k0);
    // Q^T fragments: lane holds query qrow, d = 16 s + 8 hh + 0..7 (rows past S: the last one, not stored)
    bf16x8 qf[NS];
    {
      const bf16* qp = P.q + b * P.q_sb + h * P.q_sh + min(qrow, P.S - 1) * P.q_ss + 8 * hh;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
    }
    if (tid == 0) bad = 0;
    __syncthreads();
    store_kv(0, k0);
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(__builtin_bit_cast(u32x4, qf[s]));
    __syncthreads();
    // |q| below 2^100: products with codes (up to 448) and sums of 128 of them stay finite
    u16x2 qm = {0, 0};
#pragma unroll
    for (int s = 0; s < NS; ++s) qm = max_mag(qm, __builtin_bit_cast(u32x4, qf[s]));
    if (qm[0] >= 0x7180 || qm[1] >= 0x7180) bad = 1;
    for (int t = 0; t < nt; ++t) {
      const int buf = G::NBUF == 2 ? t & 1 : 0;
      const float this_k = next_k, this_v = next_v;
      load_kv(k0 + (t + 1) * TK);
      const int kk = k0 + t * TK + 32 * kw;   // first key of this wave's 32
      if (kk < kend_w) {
        const char* kt = smem + buf * G::BUF + (32 * kw + l32) * RS + hh * 16;
        const char* vt = smem + buf * G::BUF + TILE + 32 * kw * RS + xt_lane_off(lane);
        f32x16 sacc;
#pragma unroll
        for (int r = 0; r < 16; ++r) sacc[r] = 0.f;
        bf16x8 ka[NS];
        ka[0] = *reinterpret_cast<const bf16x8*>(kt);
        ka[1] = *reinterpret_cast<const bf16x8*>(kt + 32);
#pragma unroll
        for (int s = 0; s < NS; ++s) {   // operands two steps ahead
          if (s + 2 < NS) ka[s + 2] = *reinterpret_cast<const bf16x8*>(kt + 32 * (s + 2));
          sched_fence();
          sacc = mfma32x32x16(ka[s], qf[s], sacc);
          sched_fence();
        }
        // key kk + 8 (r / 4) + 4 hh + r % 4 is seen iff it is below kq
        const int tk = kq - kk - 4 * hh;
        const bool coded = kk < nfull;
        const float unit_k = coded ? this_k : 1.f, unit_v = coded ? this_v : 1.f;
        if (!(unit_k < INFINITY && unit_v < INFINITY)) bad = 1;
        const float c = P.scale_log2 * unit_k;
#pragma unroll
        for (int r = 0; r < 16; ++r) sacc[r] *= c;   // before the mask: the scale may have any sign
        if (kk + 32 > min(kall, k1)) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[r] = (8 * (r >> 2) + (r & 3) < tk) ? sacc[r] : -INFINITY;
        }
        float mx = sacc[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, sacc[r]);
        mx = halves_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_run) != 0) {
          const float m_new = fmaxf(m_run, mx);
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
        }
        const float m_use = max_ref(m_run);
        u32x4 xt[8];
        xt[0] = lds_read_xt(vt, 0, 0);
        xt[1] = lds_read_xt(vt, 0, 1);
        // 16 keys at a time: P's terms (n = 0 first), times V
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float e[8], ps = 0.f;
          bf16x8 pt[kTerms];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            e[i] = __builtin_amdgcn_exp2f(sacc[8 * half + i] - m_use);
            ps += e[i];
          }
          l_run += ps;
#pragma unroll
          for (int i = 0; i < 8; ++i) e[i] *= unit_v;
#pragma unroll
          for (int n = 0; n < kTerms; ++n) {
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, e[2 * i + 1]),
                                           __builtin_bit_cast(uint32_t, e[2 * i]), 0x07060302u);
            pt[n] = __builtin_bit_cast(bf16x8, w);
#pragma unroll
            for (int i = 0; i < 8; ++i)   // exact
              e[i] -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, e[i]) & 0xffff0000u);
          }
#pragma unroll
          for (int dt = 0; dt < 4; ++dt) {
            const int x = 4 * half + dt;
            if (x + 2 < 8) xt[x + 2] = lds_read_xt(vt, (x + 2) / 4, (x + 2) % 4);
#pragma unroll
            for (int n = 0; n < kTerms; ++n) oacc[dt] = mfma32x32x16(__builtin_bit_cast(bf16x8, xt[x]), pt[n], oacc[dt]);
          }
        }
      }
      if (G::NBUF == 1) __syncthreads();
      if (t + 1 < nt) store_kv(G::NBUF == 2 ? buf ^ 1 : 0, k0 + (t + 1) * TK);
      __syncthreads();
    }
    l_run = halves_sum(l_run);
    // the KW waves of one query block: waves kw > 0 hand theirs to wave kw = 0
    if (KW > 1) {
      if (kw > 0) {
        float* area = reinterpret_cast<float*>(smem + (w - QW) * G::MERGE);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
#pragma unroll
          for (int m = 0; m < 4; ++m)
            *reinterpret_cast<f32x4*>(area + ((4 * dt + m) * 64 + lane) * 4) =
                f32x4{oacc[dt][4 * m], oacc[dt][4 * m + 1], oacc[dt][4 * m + 2], oacc[dt][4 * m + 3]};
        area[64 * 64 + lane] = m_run;
        area[65 * 64 + lane] = l_run;
      }
      __syncthreads();
      if (kw == 0) {
        float mo[KW], M = m_run;
#pragma unroll
        for (int g = 1; g < KW; ++g) {
          mo[g] = reinterpret_cast<const float*>(smem + (g * QW + qw - QW) * G::MERGE)[64 * 64 + lane];
          M = fmaxf(M, mo[g]);
        }
        mo[0] = m_run;
        m_run = M;
        float L = 0.f;
#pragma unroll
        for (int g = 0; g < KW; ++g) {
          const float* area = reinterpret_cast<const float*>(smem + (g * QW + qw - QW) * G::MERGE);
          const float wgt = mo[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mo[g] - M);
          L += wgt * (g == 0 ? l_run : area[65 * 64 + lane]);
#pragma unroll
          for (int dt = 0; dt < 4; ++dt)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
              if (g == 0) {
#pragma unroll
                for (int e = 0; e < 4; ++e) oacc[dt][4 * m + e] *= wgt;
              } else {
                const f32x4 x = *reinterpret_cast<const f32x4*>(area + ((4 * dt + m) * 64 + lane) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) oacc[dt][4 * m + e] += wgt * x[e];
              }
            }
        }
        l_run = L;
      }
    }
    // a score past the range upwards leaves NaN; one past it downwards (raw below -3.4e38) only
    // counts where every key that the query sees here scores about as low
    if (kw == 0 && active && min(k1, kmax(min(qrow, P.S - 1))) > k0 &&
        (l_run != l_run || m_run < 200.f - 3e38f * fabsf(P.scale_log2)))
      bad = 1;
    __syncthreads();
    if (bad) {
      extend_block_valu(P, b, h, split, q0, min(P.S, q0 + 32 * QW), k0, k1, kmax,
                        [&](int j, int n, float* f, float* unit) {
                          if (j < nfull) {
                            const u32x2 w = *reinterpret_cast<const u32x2*>((n ? vc : kc) + (int64_t)j * D + 8 * sch);
                            C::get(w[0], f);
                            C::get(w[1], f + 4);
                            *unit = (n ? vsc : ksc)[j / kBlock];
                          } else {
                            const u32x4 w = *reinterpret_cast<const u32x4*>((n ? v_row(j) : k_row(j)) + 8 * sch);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                              f[2 * e] = bf16lo(w[e]);
                              f[2 * e + 1] = bf16hi(w[e]);
                            }
                            *unit = 1.f;
                          }
                        });
      return;
    }
  }
  if (kw == 0 && active) {
    if (P.nsplit == 1) {
      // whole rows through LDS
      const float inv = row_inv(kmax(min(qrow, P.S - 1)), l_run);
      char* wl = smem + qw * OUT_WAVE_BYTES;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          *reinterpret_cast<bf16x4*>(wl + l32 * OUT_RS + (32 * dt + 8 * m + 4 * hh) * 2) =
              cvt4(oacc[dt][4 * m] * inv, oacc[dt][4 * m + 1] * inv, oacc[dt][4 * m + 2] * inv,
                   oacc[dt][4 * m + 3] * inv);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int row = (lane >> 4) + 4 * r, i = q0 + 32 * qw + row;
        const u32x4 v = *reinterpret_cast<const u32x4*>(wl + row * OUT_RS + (lane & 15) * 16);
        if (i < P.S) *reinterpret_cast<u32x4*>(P.out + b * P.o_sb + i * P.o_ss + h * P.o_sh + 8 * (lane & 15)) = v;
      }
    } else if (qrow < P.S) {
      float* dst = P.part + ((((int64_t)b * P.S + qrow) * P.H + h) * P.nsplit + split) * kPart;
      if (hh == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{m_run, l_run, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          *reinterpret_cast<f32x4*>(dst + 4 + 32 * dt + 8 * m + 4 * hh) =
              f32x4{oacc[dt][4 * m], oacc[dt][4 * m + 1], oacc[dt][4 * m + 2], oacc[dt][4 * m + 3]};
    }
  }
}

}  // namespace kv8
}  // namespace prefixlm
