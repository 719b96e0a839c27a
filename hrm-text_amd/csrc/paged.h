// Attention over a key-value cache in pages.
//
// One layer's pool is [P, Hkv, ps, D] for the keys and the same for the values: P pages of ps rows (a
// power of two from 16 to 1024), a page's rows of one head contiguous. A table [N, M] gives column c of
// sequence n the page of its rows c ps .. c ps + ps - 1; an entry outside [0, P) is no page. refs[p] is how
// many entries hold page p. Query head h belongs to key-value head h / G, G = Hq / Hkv.
//
// A call with len rows in sequence b and S new ones attends, for query i, keys j < n_i: with
// lk = min(M ps, len + s_new), n_i = lk, or with `causal` min(lk, len + s_new - S + i + 1). Keys below
// len come from the pages, and rows without a page are not seen; keys from len on are the call's own rows,
// as given, so nothing reads what the call writes. New rows are stored in pages that the sequence holds
// alone (refs 1); others are not stored.
//
// The G query heads of a key-value head and the S queries are the R = S G rows that share its keys: row
// r is query r / G of head h G + r % G. Kernels:
//   decode  : up to four rows, split over the keys, without the matrix cores;
//   stream  : up to 16 RT rows. Each wave walks 32 keys at a time by itself, through LDS of its own into the
//             matrix cores;
//   tile    : more rows: 64 or 128 a workgroup, which share tiles of the keys in LDS;
//   combine : joins the splits.
#pragma once
#include "common.h"
#include "kvcache.h"

namespace prefixlm {
namespace pkv {

using kvc::max_mag;
using kvc::max_ref;

constexpr int NT = 256;
constexpr int NWAVE = NT / 64;
constexpr int kKeys = 32;          // keys of a wave's step
constexpr int kMaxSplits = 64;
// floats per partial: max (log2 units), sum, whether a key was seen, unused, o[D]
template <int D>
constexpr int kPart = D + 4;

struct Params {
  const bf16* q;
  const bf16* k;           // new rows (may be null)
  const bf16* v;
  bf16* kp;                // the layer's pages
  bf16* vp;
  const int32_t* refs;     // [P]
  const int32_t* table;    // [B, M]
  bf16* out;
  float* part;             // [B, Hkv, R, nsplit, kPart]
  const int32_t* seqlens;  // device [B]; null: every sequence has seqlen_const
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh, table_sb;
  int B, S, Hkv, G, P, cap, ps_log2, nsplit, causal, seqlen_const;
  int s_new;               // rows appended by this call: S, or 0 without new k, v
  int nrb;                 // row blocks
  float scale_log2;
};

// Read-only data at addresses that are the same for a whole wave: through the scalar cache
typedef const __attribute__((address_space(4))) int32_t uniform_i32;
__device__ __forceinline__ uniform_i32* uniform(const int32_t* p) { return (uniform_i32*)(uintptr_t)p; }

__device__ __forceinline__ int cache_len(const Params& P, int b) {
  return min(max(P.seqlens ? P.seqlens[b] : P.seqlen_const, 0), P.cap);
}
// The keys that query i sees of a sequence of length len: [0, n)
__device__ __forceinline__ int keys_seen(const Params& P, int len, int i) {
  const int lk = min(P.cap, len + P.s_new);
  return P.causal ? min(lk, len + P.s_new - P.S + i + 1) : lk;
}
// 1 / (sum of the weights): a row that sees no key is 0, one whose scores are all -inf NaN
__device__ __forceinline__ float row_inv(bool seen, float sum) { return seen ? 1.f / sum : 0.f; }

// D(16x16 f32) += A(16x32 bf16) B(32x16 bf16). Lane l holds A[l%16][8 (l/16) + 0..7] and
// B[8 (l/16) + 0..7][l%16]; register r of the result is D[4 (l/16) + r][l%16].
__device__ __forceinline__ f32x4 mfma16x16x32(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// max / sum over lanes l, l ^ 16, l ^ 32 and l ^ 48
__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, __shfl_xor(x, 16));
  return halves_max(x);
}
__device__ __forceinline__ float rows_sum(float x) {
  x += __shfl_xor(x, 16);
  return halves_sum(x);
}

// This workgroup's share of the new rows of (b, h), part `part` of `parts`, into their pages
template <int D, int NTH = NT>
__device__ __forceinline__ void append_share(const Params& P, int b, int h, int len, int part, int parts) {
  constexpr int CH = D / 8;   // 16-byte chunks of a row
  const int c = 8 * (threadIdx.x % CH), is_v = (threadIdx.x / CH) & 1;
  for (int i = part + parts * (threadIdx.x / (2 * CH)); i < P.s_new; i += parts * (NTH / (2 * CH))) {
    const int j = len + i;
    if (j >= P.cap) break;
    const int page = P.table[b * P.table_sb + (j >> P.ps_log2)];
    if ((unsigned)page >= (unsigned)P.P || P.refs[page] != 1) continue;
    const int64_t at = ((((int64_t)page * P.Hkv + h) << P.ps_log2) + (j & ((1 << P.ps_log2) - 1))) * D + c;
    if (is_v)
      *reinterpret_cast<u32x4*>(P.vp + at) = *reinterpret_cast<const u32x4*>(P.v + b * P.v_sb + i * P.v_ss + h * P.v_sh + c);
    else
      *reinterpret_cast<u32x4*>(P.kp + at) = *reinterpret_cast<const u32x4*>(P.k + b * P.k_sb + i * P.k_ss + h * P.k_sh + c);
  }
}

// Rows [r0, r1) over keys [k0, k1) without the matrix cores: 16 lanes a row, key by key. For splits
// whose values hold an infinity or NaN (0 * inf in P V would reach rows that must not see the key), and
// for scores that pass fp32's range before the softmax scale, or whose largest is about -3e38: here the
// scale comes first.
template <int D>
__device__ __forceinline__ void walk_rows(const Params& P, int b, int h, int split, int r0, int r1, int k0, int k1, int len) {
  constexpr int E = D / 16;
  const int g16 = threadIdx.x & 15;
  const int R = P.S * P.G;
  auto get = [&](const bf16* p, float* f) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = (float)p[E * g16 + e];
  };
#pragma unroll 1
  for (int r = r0 + (threadIdx.x >> 4); r < r1; r += NT / 16) {
    const int i = r / P.G, hq = h * P.G + r % P.G;
    float q[E], o[E], x[E];
    get(P.q + b * P.q_sb + i * P.q_ss + hq * P.q_sh, q);
#pragma unroll
    for (int e = 0; e < E; ++e) q[e] *= P.scale_log2, o[e] = 0.f;
    float m = -INFINITY, l = 0.f, seen = 0.f;
#pragma unroll 1
    for (int j = k0; j < min(k1, keys_seen(P, len, i)); ++j) {
      const bf16 *kr, *vr;
      if (j < len) {
        const int page = P.table[b * P.table_sb + (j >> P.ps_log2)];
        if ((unsigned)page >= (unsigned)P.P) continue;
        const int64_t at = ((((int64_t)page * P.Hkv + h) << P.ps_log2) + (j & ((1 << P.ps_log2) - 1))) * D;
        kr = P.kp + at;
        vr = P.vp + at;
      } else {
        kr = P.k + b * P.k_sb + (j - len) * P.k_ss + h * P.k_sh;
        vr = P.v + b * P.v_sb + (j - len) * P.v_ss + h * P.v_sh;
      }
      seen = 1.f;
      get(kr, x);
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) s += q[e] * x[e];
      s = row16_sum(s);
      const float mx = fmaxf(m, s), ref = max_ref(mx);
      const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(s - ref);
      m = mx;
      l = l * alpha + p;
      get(vr, x);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + p * x[e];
    }
    if (P.nsplit == 1) {
      const float inv = row_inv(seen != 0.f, l);
      bf16* dst = P.out + b * P.o_sb + i * P.o_ss + hq * P.o_sh + E * g16;
#pragma unroll
      for (int e = 0; e < E; ++e) dst[e] = (bf16)(o[e] * inv);
    } else {
      float* dst = P.part + ((((int64_t)b * P.Hkv + h) * R + r) * P.nsplit + split) * kPart<D>;
      if (g16 == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{m, l, seen, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) dst[4 + E * g16 + e] = o[e];
    }
  }
}

// ---- few rows ---------------------------------------------------------------------------------
// Sum over the D / 8 lanes that hold a key row
template <int D>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp_f<0xB1>(x);                 // quad_perm [1,0,3,2]
  x += dpp_f<0x4E>(x);                 // quad_perm [2,3,0,1]
  x += dpp_f<0x141>(x);                // row_half_mirror
  if (D == 128) x += dpp_f<0x140>(x);  // row_mirror
  return x;
}

// NR rows (R of them real) of one (b, h, split): blockIdx.x = (b Hkv + h) nsplit + split. Each wave walks 16
// NH keys at a time by itself; D / 8 lanes hold a key row, 16 bytes each, and take its products with all
// rows.
template <int D, int NR, int NTH>
__global__ __launch_bounds__(NTH) void decode_kernel(Params P) {
  constexpr int NWAVE = NTH / 64, CH = D / 8, RPL = 64 / CH, NH = D == 128 ? 1 : 2, U = 16 / RPL;
  constexpr int kStep = 16 * NH * NWAVE;     // keys of a workgroup's step
  __shared__ float s_m[NWAVE][NR], s_l[NWAVE][NR], s_seen[NWAVE][NR];
  __shared__ f32x4 s_o[NWAVE][NR][D / 4];
  const int split = blockIdx.x % P.nsplit, bh = blockIdx.x / P.nsplit;
  const int h = bh % P.Hkv, b = bh / P.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, c8 = 8 * (lane % CH), grp = lane / CH;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = P.S * P.G;
  const int len = __builtin_amdgcn_readfirstlane(cache_len(P, b));
  const int lk = min(P.cap, len + P.s_new);
  const int per = ((lk + P.nsplit - 1) / P.nsplit + kStep - 1) / kStep * kStep;
  const int k0 = split * per;
  const int k1 = min(k0 + per, keys_seen(P, len, P.S - 1));     // the last row sees the most
  const int kall = min(min(k1, len), keys_seen(P, len, 0));     // cached keys below are seen by every row

  uniform_i32* const tab = uniform(P.table + b * P.table_sb);
  const int psm = (1 << P.ps_log2) - 1;
  const bf16* const kn = P.s_new ? P.k + b * P.k_sb + h * P.k_sh + c8 : nullptr;
  const bf16* const vn = P.s_new ? P.v + b * P.v_sb + h * P.v_sh + c8 : nullptr;
  const u32x4 zero = {0u, 0u, 0u, 0u};
  u32x4 kw[NH][U], vw[NH][U];
  int page[NH];                 // of the 16 keys to load next
  bool ok[NH];                  // the cached ones among the 16 keys have a page
  auto look = [&](int j0) {
#pragma unroll
    for (int hf = 0; hf < NH; ++hf) page[hf] = j0 + 16 * hf < len ? tab[(j0 + 16 * hf) >> P.ps_log2] : -1;
  };
  const uint32_t off = (uint32_t)(grp * D + c8) * 2;
  auto load = [&](int j0) {
#pragma unroll
    for (int hf = 0; hf < NH; ++hf) {
      const int j = j0 + 16 * hf;
      ok[hf] = (unsigned)page[hf] < (unsigned)P.P;
      const int64_t at = ((((int64_t)(ok[hf] ? page[hf] : 0) * P.Hkv + h) << P.ps_log2) + (j & psm)) * D;
      const char *kb = reinterpret_cast<const char*>(P.kp + at), *vb = reinterpret_cast<const char*>(P.vp + at);
      if (ok[hf] && j + 16 <= len) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          kw[hf][u] = kvc::load_once(reinterpret_cast<const bf16*>(kb + off + u * (RPL * D * 2)));
          vw[hf][u] = kvc::load_once(reinterpret_cast<const bf16*>(vb + off + u * (RPL * D * 2)));
        }
      } else {
        // the last cached rows, the new ones, none: row by row
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int jr = j + u * RPL + grp;
          kw[hf][u] = vw[hf][u] = zero;
          if (jr < len ? ok[hf] : jr < lk) {
            kw[hf][u] = *reinterpret_cast<const u32x4*>(jr < len ? kb + off + u * (RPL * D * 2) : reinterpret_cast<const char*>(kn + (jr - len) * P.k_ss));
            vw[hf][u] = *reinterpret_cast<const u32x4*>(jr < len ? vb + off + u * (RPL * D * 2) : reinterpret_cast<const char*>(vn + (jr - len) * P.v_ss));
          }
        }
      }
    }
  };
  int j0 = k0 + 16 * NH * w;
  if (j0 < k1) {
    look(j0);
    load(j0);
    look(j0 + kStep);
  }
  float q[NR][8], o[NR][8], m[NR], l[NR], seen[NR];
  int nlim[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int rr = min(r, R - 1);
    const u32x4 x = *reinterpret_cast<const u32x4*>(P.q + b * P.q_sb + (rr / P.G) * P.q_ss + (h * P.G + rr % P.G) * P.q_sh + c8);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[r][2 * e] = bf16lo(x[e]) * P.scale_log2, q[r][2 * e + 1] = bf16hi(x[e]) * P.scale_log2;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[r][e] = 0.f;
    m[r] = -INFINITY, l[r] = 0.f, seen[r] = 0.f;
    nlim[r] = min(k1, keys_seen(P, len, rr / P.G));
  }
  for (; j0 < k1; j0 += kStep) {
    float s[NR][NH][U];
#pragma unroll
    for (int hf = 0; hf < NH; ++hf)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = bf16lo(kw[hf][u][e]), x[2 * e + 1] = bf16hi(kw[hf][u][e]);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          float d = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) d += q[r][e] * x[e];
          s[r][hf][u] = lanes_sum<D>(d);
        }
      }
    bool full = j0 + 16 * NH <= kall;
#pragma unroll
    for (int hf = 0; hf < NH; ++hf) full = full && ok[hf];
    uint32_t hides = 0;          // bit (r, hf, u): the row does not see this lane's key
    if (!full) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int hf = 0; hf < NH; ++hf)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int j = j0 + 16 * hf + u * RPL + grp;
            const bool sees = j < nlim[r] && (ok[hf] || j >= len);
            seen[r] = sees ? 1.f : seen[r];
            s[r][hf][u] = sees ? s[r][hf][u] : -INFINITY;
            hides |= (sees ? 0u : 1u) << ((r * NH + hf) * U + u);
          }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (full) seen[r] = 1.f;
      float mx = m[r];
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[r][hf][u]);
      const float ref = max_ref(mx), alpha = __builtin_amdgcn_exp2f(m[r] - ref);   // m = -inf at first: 0
      m[r] = mx;
      l[r] *= alpha;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[r][e] *= alpha;
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[r][hf][u] = __builtin_amdgcn_exp2f(s[r][hf][u] - ref);
          l[r] += s[r][hf][u];
        }
    }
#pragma unroll
    for (int hf = 0; hf < NH; ++hf)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[2 * e] = bf16lo(vw[hf][u][e]), x[2 * e + 1] = bf16hi(vw[hf][u][e]);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          // a value that the row does not see may be infinite
          if (!full && (hides >> ((r * NH + hf) * U + u) & 1)) continue;
#pragma unroll
          for (int e = 0; e < 8; ++e) o[r][e] += s[r][hf][u] * x[e];
        }
      }
    if (j0 + kStep < k1) {
      load(j0 + kStep);
      look(j0 + 2 * kStep);
    }
  }
  // the wave's groups, then the waves
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float M = m[r];
#pragma unroll
    for (int x = CH; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
    const float a = m[r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[r] - M);
    l[r] *= a;
#pragma unroll
    for (int x = CH; x < 64; x <<= 1) {
      l[r] += __shfl_xor(l[r], x);
      seen[r] = fmaxf(seen[r], __shfl_xor(seen[r], x));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      o[r][e] *= a;
#pragma unroll
      for (int x = CH; x < 64; x <<= 1) o[r][e] += __shfl_xor(o[r][e], x);
    }
    if (lane < CH) {
      if (lane == 0) s_m[w][r] = M, s_l[w][r] = l[r], s_seen[w][r] = seen[r];
      s_o[w][r][2 * lane] = f32x4{o[r][0], o[r][1], o[r][2], o[r][3]};
      s_o[w][r][2 * lane + 1] = f32x4{o[r][4], o[r][5], o[r][6], o[r][7]};
    }
  }
  __syncthreads();
  if (tid < NR * (D / 4)) {
    const int r = tid / (D / 4), c = tid % (D / 4);
    if (r < R) {
      float M = s_m[0][r], L = 0.f, any = 0.f;
#pragma unroll
      for (int g = 1; g < NWAVE; ++g) M = fmaxf(M, s_m[g][r]);
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int g = 0; g < NWAVE; ++g) {
        const float wgt = s_m[g][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[g][r] - M);
        L += wgt * s_l[g][r];
        any = fmaxf(any, s_seen[g][r]);
        acc += wgt * s_o[g][r][c];
      }
      if (P.nsplit == 1) {
        const float inv = row_inv(any != 0.f, L);
        *reinterpret_cast<bf16x4*>(P.out + b * P.o_sb + (r / P.G) * P.o_ss + (h * P.G + r % P.G) * P.o_sh + 4 * c) =
            cvt4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
      } else {
        float* dst = P.part + (((int64_t)bh * R + r) * P.nsplit + split) * kPart<D>;
        if (c == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{M, L, any, 0.f};
        *reinterpret_cast<f32x4*>(dst + 4 + 4 * c) = acc;
      }
    }
  }
  append_share<D, NTH>(P, b, h, len, split, P.nsplit);
}

// ---- more of them -------------------------------------------------------------------------------
template <int D>
struct Geo {
  static constexpr int NS = D / 32;              // steps of the contraction over d
  static constexpr int ND = D / 16;              // 16-column tiles of o; 16-byte loads a lane of 32 keys
  static constexpr int CH = D / 8;               // 16-byte chunks of a row
  static constexpr int RPL = 64 / CH;            // rows a load
  // V rows in LDS: 8 rows apart by 8 banks each, so that the 32 lanes of a transposing read's cycle, 8
  // rows of 32 bytes, take all 64 banks
  static constexpr int VS = 2 * D + 32;
  // K rows in LDS: 4 banks apart, so that 16 rows' 16 bytes at one column take all 64
  static constexpr int KS = 2 * D + 16;
  static constexpr int OS = D + 4;               // floats of a row of o where the waves meet
  static constexpr int AREA = kKeys * (VS + KS); // bytes a wave
  static_assert(AREA >= 16 * OS * 4, "16 rows of o fit");
};

// blockIdx.x: row blocks of one (b, h, split) eight indices apart, on one XCD.
template <int D, int RT>
__global__ __launch_bounds__(NT, RT == 1 ? 3 : 2) void stream_kernel(Params P) {
  using G = Geo<D>;
  constexpr int NS = G::NS, ND = G::ND, CH = G::CH, HL = ND / 2;   // HL: V loads of 16 keys
  __shared__ __attribute__((aligned(16))) char smem[NWAVE][G::AREA];
  __shared__ float s_m[NWAVE][16], s_l[NWAVE][16], s_seen[NWAVE][16];
  __shared__ int s_bad;
  const int rb = (blockIdx.x >> 3) % P.nrb;
  const int unit = (int)((blockIdx.x >> 3) / P.nrb) * 8 + (blockIdx.x & 7);
  if (unit >= P.B * P.Hkv * P.nsplit) return;
  const int split = unit % P.nsplit, bh = unit / P.nsplit;
  const int h = bh % P.Hkv, b = bh / P.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int R = P.S * P.G, r0 = rb * 16 * RT, r1 = min(R, r0 + 16 * RT);
  const int len = __builtin_amdgcn_readfirstlane(cache_len(P, b));
  const int lk = min(P.cap, len + P.s_new);
  // the splits share a sequence's own keys, in whole steps
  const int per = ((lk + P.nsplit - 1) / P.nsplit + kKeys - 1) / kKeys * kKeys;
  const int k0 = split * per;
  const int k1 = min(k0 + per, keys_seen(P, len, (r1 - 1) / P.G));   // the last row sees the most
  const int kall = keys_seen(P, len, r0 / P.G);                      // every row sees the keys below
  if (tid == 0) s_bad = 0;

  uniform_i32* const tab = uniform(P.table + b * P.table_sb);
  const int psm = (1 << P.ps_log2) - 1;
  const bf16* const kn = P.s_new ? P.k + b * P.k_sb + h * P.k_sh + 8 * (lane % CH) : nullptr;
  const bf16* const vn = P.s_new ? P.v + b * P.v_sb + h * P.v_sh + 8 * (lane % CH) : nullptr;
  char* const area = smem[w];

  u32x4 kw[ND], vw[ND];
  bool ok[2];              // the 16 keys have a page, or are new rows
  const u32x4 zero = {0u, 0u, 0u, 0u};
  const uint32_t off = (uint32_t)(lane / CH * D + 8 * (lane % CH)) * 2;
  auto load = [&](int j0) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int j = j0 + 16 * hf;
      const int page = j < len ? tab[j >> P.ps_log2] : -1;
      const bool held = (unsigned)page < (unsigned)P.P;
      const int64_t at = ((((int64_t)(held ? page : 0) * P.Hkv + h) << P.ps_log2) + (j & psm)) * D;
      const char *kb = reinterpret_cast<const char*>(P.kp + at), *vb = reinterpret_cast<const char*>(P.vp + at);
      ok[hf] = held;
      if (held && j + 16 <= len) {
#pragma unroll
        for (int u = 0; u < HL; ++u) {
          kw[hf * HL + u] = kvc::load_once(reinterpret_cast<const bf16*>(kb + off + u * (G::RPL * D * 2)));
          vw[hf * HL + u] = kvc::load_once(reinterpret_cast<const bf16*>(vb + off + u * (G::RPL * D * 2)));
        }
      } else {
        // the last cached rows, the new ones, none: row by row
#pragma unroll
        for (int u = 0; u < HL; ++u) {
          const int jr = j + u * G::RPL + lane / CH;
          kw[hf * HL + u] = vw[hf * HL + u] = zero;
          if (jr < len ? held : jr < lk) {
            kw[hf * HL + u] = *reinterpret_cast<const u32x4*>(
                jr < len ? kb + off + u * (G::RPL * D * 2) : reinterpret_cast<const char*>(kn + (jr - len) * P.k_ss));
            vw[hf * HL + u] = *reinterpret_cast<const u32x4*>(
                jr < len ? vb + off + u * (G::RPL * D * 2) : reinterpret_cast<const char*>(vn + (jr - len) * P.v_ss));
          }
        }
      }
    }
  };

  float m_run[RT], l_run[RT], seen[RT];
  f32x4 oacc[RT][ND];
  int nlim[RT];            // this lane's row sees keys below, of this split
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    m_run[t] = -INFINITY, l_run[t] = 0.f, seen[t] = 0.f;
    nlim[t] = min(k1, keys_seen(P, len, min(r0 + 16 * t + l16, R - 1) / P.G));
#pragma unroll
    for (int d = 0; d < ND; ++d) oacc[t][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  u16x2 vmag = {0, 0};

  int j0 = k0 + kKeys * w;
  if (j0 < k1) {
    load(j0);
    // Q^T: lane holds row l16, columns 32 s + 8 g4 + 0..7 (rows past the last: that one, not stored)
    bf16x8 qf[RT][NS];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int r = min(r0 + 16 * t + l16, R - 1);
      const bf16* qp = P.q + b * P.q_sb + (r / P.G) * P.q_ss + (h * P.G + r % P.G) * P.q_sh + 8 * g4;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[t][s] = *reinterpret_cast<const bf16x8*>(qp + 32 * s);
    }
    char* const karea = area + kKeys * G::VS;
    const char *const vt = area + (4 * g4 + (l16 >> 2)) * G::VS + 8 * (l16 & 3), *const kt = karea + l16 * G::KS + 16 * g4;
    const int row = lane / CH, c16 = 16 * (lane % CH);
    for (; j0 < k1; j0 += kKeys * NWAVE) {
#pragma unroll
      for (int u = 0; u < ND; ++u) *reinterpret_cast<u32x4*>(karea + (u * G::RPL + row) * G::KS + c16) = kw[u];
#pragma unroll
      for (int u = 0; u < ND; ++u) {
        vmag = max_mag(vmag, vw[u]);
        *reinterpret_cast<u32x4*>(area + (u * G::RPL + row) * G::VS + c16) = vw[u];
      }
      // a page that is missing hides cached keys only
      const bool ok0 = ok[0], ok1 = ok[1];
      if (j0 + kKeys * NWAVE < k1) load(j0 + kKeys * NWAVE);
      // K: lane holds key l16 of 16, columns 32 n + 8 g4 + 0..7
      f32x4 s[RT][2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          const bf16x8 kf = *reinterpret_cast<const bf16x8*>(kt + 16 * hf * G::KS + 64 * n);
#pragma unroll
          for (int t = 0; t < RT; ++t) s[t][hf] = mfma16x16x32(kf, qf[t][n], n ? s[t][hf] : f32x4{0.f, 0.f, 0.f, 0.f});
        }
      bf16x8 pt[RT][3];
#pragma unroll
      for (int t = 0; t < RT; ++t) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[t][hf][r] *= P.scale_log2;   // before the mask: the scale may have any sign
        if (j0 + kKeys > min(kall, k1) || !ok0 || !ok1) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int j = j0 + 16 * hf + 4 * g4 + r;
              const bool sees = j < nlim[t] && ((hf ? ok1 : ok0) || j >= len);
              seen[t] = sees ? 1.f : seen[t];
              s[t][hf][r] = sees ? s[t][hf][r] : -INFINITY;
            }
        } else {
          seen[t] = 1.f;
        }
        float mx = s[t][0][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[t][e >> 2][e & 3]);
        mx = rows_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_run[t]) != 0) {
          const float m_new = fmaxf(m_run[t], mx);
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[t] - m_new);
          m_run[t] = m_new;
          l_run[t] *= alpha;
#pragma unroll
          for (int d = 0; d < ND; ++d) oacc[t][d] *= alpha;
        }
        const float m_use = max_ref(m_run[t]);
        float e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          e[i] = __builtin_amdgcn_exp2f(s[t][i >> 2][i & 3] - m_use);
          l_run[t] += e[i];
        }
        // the probabilities go into P V as three bf16 terms, which add up to their fp32 bits
#pragma unroll
        for (int n = 0; n < 3; ++n) {
          u32x4 x;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            x[i] = pack_hi(__builtin_bit_cast(uint32_t, e[2 * i]), __builtin_bit_cast(uint32_t, e[2 * i + 1]));
          pt[t][n] = __builtin_bit_cast(bf16x8, x);
#pragma unroll
          for (int i = 0; i < 8; ++i)   // exact
            e[i] -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, e[i]) & 0xffff0000u);
        }
      }
      // V^T: lane holds column 16 d + l16 of keys 4 g4 + 0..3 and 16 + 4 g4 + 0..3, as s has them
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x2 x0 = lds_read_tr(vt, 32 * d), x1 = lds_read_tr(vt, 16 * G::VS + 32 * d);
        const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{x0[0], x0[1], x1[0], x1[1]});
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int n = 0; n < 3; ++n) oacc[t][d] = mfma16x16x32(vf, pt[t][n], oacc[t][d]);
      }
    }
  }

  __syncthreads();   // s_bad is cleared
  bool bad = vmag[0] >= 0x7f80 || vmag[1] >= 0x7f80;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    l_run[t] = rows_sum(l_run[t]);
    // a score past the range upwards leaves NaN; one past it downwards (raw below -3.4e38) only counts
    // where every key that the row sees here scores about as low
    bad |= seen[t] != 0.f && (l_run[t] != l_run[t] || m_run[t] < 200.f - 3e38f * fabsf(P.scale_log2));
    seen[t] = rows_max(seen[t]);
  }
  if (bad) s_bad = 1;
  // the waves' results meet, 16 rows at a time
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    if (t) __syncthreads();
    float* o = reinterpret_cast<float*>(area) + l16 * G::OS + 4 * g4;
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(o + 16 * d) = oacc[t][d];
    if (g4 == 0) s_m[w][l16] = m_run[t], s_l[w][l16] = l_run[t], s_seen[w][l16] = seen[t];
    __syncthreads();
    if (s_bad) break;
    constexpr int E = D / 16;
    const int row = tid >> 4, r = r0 + 16 * t + row;
    if (r >= r1) continue;
    float M = s_m[0][row], L = 0.f, any = 0.f, x[E];
#pragma unroll
    for (int g = 1; g < NWAVE; ++g) M = fmaxf(M, s_m[g][row]);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll
    for (int g = 0; g < NWAVE; ++g) {
      const float wgt = s_m[g][row] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[g][row] - M);
      L += wgt * s_l[g][row];
      any = fmaxf(any, s_seen[g][row]);
      const float* src = reinterpret_cast<const float*>(smem[g]) + row * G::OS + E * l16;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(src + e);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[e + c] += wgt * y[c];
      }
    }
    if (P.nsplit == 1) {
      const float inv = row_inv(any != 0.f, L);
      bf16* dst = P.out + b * P.o_sb + (r / P.G) * P.o_ss + (h * P.G + r % P.G) * P.o_sh + E * l16;
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<bf16x4*>(dst + e) = cvt4(x[e] * inv, x[e + 1] * inv, x[e + 2] * inv, x[e + 3] * inv);
    } else {
      float* dst = P.part + ((((int64_t)b * P.Hkv + h) * R + r) * P.nsplit + split) * kPart<D>;
      if (l16 == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{M, L, any, 0.f};
#pragma unroll
      for (int e = 0; e < E; e += 4) *reinterpret_cast<f32x4*>(dst + 4 + E * l16 + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
    }
  }
  if (s_bad) walk_rows<D>(P, b, h, split, r0, r1, k0, k1, len);
  append_share<D>(P, b, h, len, rb * P.nsplit + split, P.nrb * P.nsplit);
}

// ---- many rows -----------------------------------------------------------------------------------
// Workgroup = 32 QW rows of (b, h, split): QW waves along the rows and KW = 4 / QW along the keys, as the
// contiguous cache's extend kernel: a staged tile of 32 KW keys serves all of them, S^T = K Q^T with the
// row as the lane column, V^T from transposing reads.
template <int D, int QW>
struct TileGeo {
  static constexpr int KW = 4 / QW;
  static constexpr int TK = 32 * KW;                     // keys a tile
  static constexpr int CH = D / 8, RPP = NT / CH;        // 16-byte chunks of a row; rows that all threads load at once
  static constexpr int NP = TK / RPP;
  static constexpr int NDT = D / 32;
  // rows 12 banks apart modulo 64 times an odd number, four rows 48: see RS in common.h
  static constexpr int RSD = 2 * D + 48;
  static constexpr int TILE = TK * RSD, BUF = 2 * TILE;  // K tile, V tile; two of them
  static constexpr int OUT = 32 * (2 * D + 16);          // a wave's output rows
  static constexpr int MERGE = 64 * 16 * NDT * 4 + 3 * 64 * 4;   // a wave's O, max, sum, seen
  static constexpr int LDS_BYTES = 2 * BUF;
  static_assert((4 - QW) * MERGE <= LDS_BYTES && QW * OUT <= LDS_BYTES, "epilogue areas fit");
};

template <int D, int QW>
__global__ __launch_bounds__(NT, 2) void tile_kernel(Params P) {
  using G = TileGeo<D, QW>;
  constexpr int KW = G::KW, TK = G::TK, NP = G::NP, NDT = G::NDT, NS = D / 16, CH = G::CH, RSD = G::RSD;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_bad, s_hole;   // a value row or score is not finite; a tile had rows without a page
  const int rb = (blockIdx.x >> 3) % P.nrb;
  const int unit = (int)((blockIdx.x >> 3) / P.nrb) * 8 + (blockIdx.x & 7);
  if (unit >= P.B * P.Hkv * P.nsplit) return;
  const int split = unit % P.nsplit, bh = unit / P.nsplit;
  const int h = bh % P.Hkv, b = bh / P.Hkv;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = w % QW, kw = w / QW;
  const int R = P.S * P.G, r0 = rb * 32 * QW, r1 = min(R, r0 + 32 * QW);
  const int len = __builtin_amdgcn_readfirstlane(cache_len(P, b));
  const int lk = min(P.cap, len + P.s_new);
  const int per = ((lk + P.nsplit - 1) / P.nsplit + TK - 1) / TK * TK;
  const int k0 = split * per;
  const int k1 = min(k0 + per, keys_seen(P, len, (r1 - 1) / P.G));
  const int kall = keys_seen(P, len, r0 / P.G);                  // every row of the block sees the keys below
  const int row = min(r0 + 32 * qw + l32, R - 1);                // this lane's (past the last: that one, not stored)
  const int ri = row / P.G, rh = h * P.G + row % P.G;
  const bool active = r0 + 32 * qw < R;
  const int kq = min(k1, keys_seen(P, len, ri));
  const int kend_w = active ? min(k1, keys_seen(P, len, (min(R, r0 + 32 * qw + 32) - 1) / P.G)) : 0;

  uniform_i32* const tab = uniform(P.table + b * P.table_sb);
  const int psm = (1 << P.ps_log2) - 1;
  // staging: thread = chunk sch of rows srow + RPP n; V rows in permuted order
  const int srow = tid / CH, sch = tid % CH, vrow = perm_row(srow);
  const int g16 = __builtin_amdgcn_readfirstlane(srow & ~15);    // this wave's 16 keys of a pass
  const bf16* const kn = P.s_new ? P.k + b * P.k_sb + h * P.k_sh + 8 * sch : nullptr;
  const bf16* const vn = P.s_new ? P.v + b * P.v_sb + h * P.v_sh + 8 * sch : nullptr;
  const uint32_t koff = (uint32_t)((srow & 15) * D + 8 * sch) * 2, voff = (uint32_t)((vrow & 15) * D + 8 * sch) * 2;
  u32x4 ks[NP], vs[NP];
  const u32x4 zero = {0u, 0u, 0u, 0u};
  int page[NP];                 // of this wave's keys of the tile to load next
  auto look = [&](int t0) {
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int j = t0 + G::RPP * n + g16;
      page[n] = j < len ? tab[j >> P.ps_log2] : -1;
    }
  };
  auto load = [&](int t0) {
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int j = t0 + G::RPP * n + g16;
      const bool held = (unsigned)page[n] < (unsigned)P.P;
      const int64_t at = ((((int64_t)(held ? page[n] : 0) * P.Hkv + h) << P.ps_log2) + (j & psm)) * D;
      const char *kb = reinterpret_cast<const char*>(P.kp + at), *vb = reinterpret_cast<const char*>(P.vp + at);
      if (held && j + 16 <= len) {
        ks[n] = *reinterpret_cast<const u32x4*>(kb + koff);
        vs[n] = *reinterpret_cast<const u32x4*>(vb + voff);
      } else {
        // the last cached rows, the new ones, none: row by row
        if (j < min(len, k1) && !held) s_hole = 1;
        const int jk = j + (srow & 15), jv = j + (vrow & 15);
        ks[n] = vs[n] = zero;
        if (jk < len ? held : jk < k1)
          ks[n] = *reinterpret_cast<const u32x4*>(jk < len ? kb + koff : reinterpret_cast<const char*>(kn + (jk - len) * P.k_ss));
        if (jv < len ? held : jv < k1)
          vs[n] = *reinterpret_cast<const u32x4*>(jv < len ? vb + voff : reinterpret_cast<const char*>(vn + (jv - len) * P.v_ss));
      }
    }
  };
  u16x2 vmag = {0, 0};
  auto store = [&](int buf) {
    char* base = smem + buf * G::BUF + srow * RSD + sch * 16;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      *reinterpret_cast<u32x4*>(base + G::RPP * n * RSD) = ks[n];
      *reinterpret_cast<u32x4*>(base + G::TILE + G::RPP * n * RSD) = vs[n];
      vmag = max_mag(vmag, vs[n]);
    }
  };

  float m_run = -INFINITY, l_run = 0.f, seen = 0.f;
  f32x16 oacc[NDT];
#pragma unroll
  for (int t = 0; t < NDT; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) oacc[t][r] = 0.f;
  if (tid == 0) s_bad = 0, s_hole = 0;
  __syncthreads();

  if (k0 < k1) {
    const int nt = (k1 - k0 + TK - 1) / TK;
    look(k0);
    load(k0);
    look(k0 + TK);
    // Q^T fragments: lane holds its row, columns 16 s + 8 hh + 0..7
    bf16x8 qf[NS];
    {
      const bf16* qp = P.q + b * P.q_sb + ri * P.q_ss + rh * P.q_sh + 8 * hh;
#pragma unroll
      for (int s = 0; s < NS; ++s) qf[s] = *reinterpret_cast<const bf16x8*>(qp + 16 * s);
    }
    store(0);
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(__builtin_bit_cast(u32x4, qf[s]));
    __syncthreads();
    const float c = P.scale_log2;
    for (int t = 0; t < nt; ++t) {
      const int buf = t & 1;
      if (t + 1 < nt) {
        load(k0 + (t + 1) * TK);
        look(k0 + (t + 2) * TK);
      }
      const int kk = k0 + t * TK + 32 * kw;   // first key of this wave's 32
      if (kk < kend_w) {
        const char* kt = smem + buf * G::BUF + (32 * kw + l32) * RSD + hh * 16;
        const char* vt = smem + buf * G::BUF + G::TILE + 32 * kw * RSD + xt_lane_off<RSD>(lane);
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
#pragma unroll
        for (int r = 0; r < 16; ++r) sacc[r] *= c;   // before the mask: the scale may have any sign
        const bool hole = s_hole != 0;
        if (kk + 32 > min(kall, k1) || hole) {
          // key kk + 8 (r / 4) + 4 hh + r % 4 is seen iff it is below kq, and cached ones have a page
          bool ok[2];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int j = kk + 16 * g;
            ok[g] = !hole || j >= len || (unsigned)tab[j >> P.ps_log2] < (unsigned)P.P;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = kk + 8 * (r >> 2) + 4 * hh + (r & 3);
            const bool sees = j < kq && (ok[r >> 3] || j >= len);
            seen = sees ? 1.f : seen;
            sacc[r] = sees ? sacc[r] : -INFINITY;
          }
        } else {
          seen = 1.f;
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
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
        }
        const float m_use = max_ref(m_run);
        u32x4 xt[2 * NDT];
        xt[0] = lds_read_xt<RSD>(vt, 0, 0);
        xt[1] = lds_read_xt<RSD>(vt, 0, 1);
        // 16 keys at a time: P's three bf16 terms, which add up to its fp32 bits, times V
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float e[8], ps = 0.f;
          bf16x8 pt[3];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            e[i] = __builtin_amdgcn_exp2f(sacc[8 * half + i] - m_use);
            ps += e[i];
          }
          l_run += ps;
#pragma unroll
          for (int n = 0; n < 3; ++n) {
            u32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = pack_hi(__builtin_bit_cast(uint32_t, e[2 * i]), __builtin_bit_cast(uint32_t, e[2 * i + 1]));
            pt[n] = __builtin_bit_cast(bf16x8, x);
#pragma unroll
            for (int i = 0; i < 8; ++i)   // exact
              e[i] -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, e[i]) & 0xffff0000u);
          }
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) {
            const int x = NDT * half + dt;
            if (x + 2 < 2 * NDT) xt[x + 2] = lds_read_xt<RSD>(vt, (x + 2) / NDT, (x + 2) % NDT);
#pragma unroll
            for (int n = 0; n < 3; ++n) oacc[dt] = mfma32x32x16(__builtin_bit_cast(bf16x8, xt[x]), pt[n], oacc[dt]);
          }
        }
      }
      if (t + 1 < nt) store(buf ^ 1);
      __syncthreads();
    }
  }
  l_run = halves_sum(l_run);
  // a score past the range upwards leaves NaN; one past it downwards (raw below -3.4e38) only counts
  // where every key that the row sees here scores about as low
  if (vmag[0] >= 0x7f80 || vmag[1] >= 0x7f80 || (seen != 0.f && (l_run != l_run || m_run < 200.f - 3e38f * fabsf(P.scale_log2))))
    s_bad = 1;
  seen = halves_max(seen);
  // the KW waves of 32 rows: waves kw > 0 hand theirs to wave kw = 0
  if (KW > 1) {
    if (kw > 0) {
      float* area = reinterpret_cast<float*>(smem + (w - QW) * G::MERGE);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          *reinterpret_cast<f32x4*>(area + ((4 * dt + m) * 64 + lane) * 4) =
              f32x4{oacc[dt][4 * m], oacc[dt][4 * m + 1], oacc[dt][4 * m + 2], oacc[dt][4 * m + 3]};
      area += 64 * 16 * NDT;
      area[lane] = m_run;
      area[64 + lane] = l_run;
      area[128 + lane] = seen;
    }
    __syncthreads();
    if (kw == 0) {
      float mo[KW], M = m_run;
#pragma unroll
      for (int g = 1; g < KW; ++g) {
        mo[g] = reinterpret_cast<const float*>(smem + (g * QW + qw - QW) * G::MERGE)[64 * 16 * NDT + lane];
        M = fmaxf(M, mo[g]);
      }
      mo[0] = m_run;
      m_run = M;
      float L = 0.f;
#pragma unroll
      for (int g = 0; g < KW; ++g) {
        const float* area = reinterpret_cast<const float*>(smem + (g * QW + qw - QW) * G::MERGE);
        const float wgt = mo[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mo[g] - M);
        L += wgt * (g == 0 ? l_run : area[64 * 16 * NDT + 64 + lane]);
        if (g) seen = fmaxf(seen, area[64 * 16 * NDT + 128 + lane]);
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
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
  __syncthreads();
  if (s_bad) {
    walk_rows<D>(P, b, h, split, r0, r1, k0, k1, len);
  } else if (kw == 0 && active) {
    if (P.nsplit == 1) {
      // whole rows through LDS
      constexpr int ORS = 2 * D + 16;
      const float inv = row_inv(seen != 0.f, l_run);
      char* wl = smem + qw * G::OUT;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          *reinterpret_cast<bf16x4*>(wl + l32 * ORS + (32 * dt + 8 * m + 4 * hh) * 2) =
              cvt4(oacc[dt][4 * m] * inv, oacc[dt][4 * m + 1] * inv, oacc[dt][4 * m + 2] * inv,
                   oacc[dt][4 * m + 3] * inv);
#pragma unroll
      for (int n = 0; n < 32 / (64 / CH); ++n) {
        const int rr = lane / CH + (64 / CH) * n, r = r0 + 32 * qw + rr;
        const u32x4 v = *reinterpret_cast<const u32x4*>(wl + rr * ORS + (lane % CH) * 16);
        if (r < R)
          *reinterpret_cast<u32x4*>(P.out + b * P.o_sb + (r / P.G) * P.o_ss + (h * P.G + r % P.G) * P.o_sh + 8 * (lane % CH)) = v;
      }
    } else if (r0 + 32 * qw + l32 < R) {
      float* dst = P.part + (((int64_t)bh * R + row) * P.nsplit + split) * kPart<D>;
      if (hh == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{m_run, l_run, seen, 0.f};
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          *reinterpret_cast<f32x4*>(dst + 4 + 32 * dt + 8 * m + 4 * hh) =
              f32x4{oacc[dt][4 * m], oacc[dt][4 * m + 1], oacc[dt][4 * m + 2], oacc[dt][4 * m + 3]};
    }
  }
  append_share<D>(P, b, h, len, rb * P.nsplit + split, P.nrb * P.nsplit);
}

// One wave per (b, h, r): lane s weighs split s, then D / 4 lanes a split add their four columns.
template <int D>
__global__ __launch_bounds__(256) void combine_kernel(Params P) {
  constexpr int L4 = D / 4, NG = 64 / L4;
  const int R = P.S * P.G;
  const int64_t u = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 6;
  const int lane = threadIdx.x & 63, col = lane % L4, grp = lane / L4;
  if (u >= (int64_t)P.B * P.Hkv * R) return;
  const float* src = P.part + u * P.nsplit * kPart<D>;
  const int n = P.nsplit;   // at most 64
  f32x4 head = {-INFINITY, 0.f, 0.f, 0.f};
  if (lane < n) head = *reinterpret_cast<const f32x4*>(src + lane * kPart<D>);
  const float M = wave_max(head[0]);
  const float wgt = head[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(head[0] - M);
  float L = wgt * head[1];
  const bool seen = __builtin_amdgcn_ballot_w64(head[2] != 0.f) != 0;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = grp; s0 < n + grp; s0 += 8 * NG) {
    // eight loads in flight; past the last split its partial again, not added (it may be inf)
    f32x4 o[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] = *reinterpret_cast<const f32x4*>(src + min(s0 + NG * x, n - 1) * kPart<D> + 4 + 4 * col);
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const int at = s0 + NG * x;
      const f32x4 y = acc + __shfl(wgt, at & 63) * o[x];
      acc = at < n ? y : acc;
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) L += __shfl_xor(L, m);
#pragma unroll
  for (int m = L4; m < 64; m <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], m);
  const float inv = row_inv(seen, L);
  const int r = (int)(u % R), bh = (int)(u / R), h = bh % P.Hkv, b = bh / P.Hkv;
  if (grp == 0)
    *reinterpret_cast<bf16x4*>(P.out + b * P.o_sb + (r / P.G) * P.o_ss + (h * P.G + r % P.G) * P.o_sh + 4 * col) =
        cvt4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}

}  // namespace pkv
}  // namespace prefixlm
