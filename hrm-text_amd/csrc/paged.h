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
//   decode  : one row, without the matrix cores;
//   stream  : up to 16 rows. Each wave walks 32 keys at a time by itself, through LDS of its own into the
//             matrix cores;
//   tile    : more rows: 64 or 128 a workgroup, which share tiles of the keys in LDS;
//   combine : joins the pieces of a unit.
//
// A unit is a block of rows of one (sequence, key-value head); its keys are tiles. Where units are few (up to 384 for one
// row, 256 for more, of up to 256 sequences), each is cut into pieces, as many as its sequence's tiles are worth, so that
// sequences of any lengths end together (Sched). Where they are many, each is one workgroup, whatever its length: a batch
// of short sequences and a very long one then ends with the long one's units alone.
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
constexpr int kMaxShared = 256;    // sequences of a call whose units are cut
constexpr float kAbove = 8.f;      // log2 of how far a weight may pass the largest one so far (tile)
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
  float* part;             // [workgroups, rows of a block, kPart]: a piece's result, where it is not the whole unit's
  int32_t* pre;            // [B + 1]: workgroups before each sequence, from the first one for the combine
  const int32_t* seqlens;  // device [B]; null: every sequence has seqlen_const
  int64_t q_sb, q_ss, q_sh, k_sb, k_ss, k_sh, v_sb, v_ss, v_sh, o_sb, o_ss, o_sh, table_sb;
  int B, S, Hkv, G, P, cap, ps_log2, causal, seqlen_const;
  int s_new;               // rows appended by this call: S, or 0 without new k, v
  int nrb;                 // row blocks
  int nwg;                 // workgroups that the units share; 0: one for each unit
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
// Weights are taken 2^spread below the largest score's, so that the n of a row add up to at most 1/2 and what they weigh
// stays within fp32's range wherever the values do
__device__ __forceinline__ float spread(int n) { return (float)(33 - __builtin_clz(max(n, 1))); }
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

// ---- which workgroup takes what --------------------------------------------------------------------
// Workgroup = tiles [first, first + count) of TS keys, piece `piece` of the `pieces` of unit (b, h, rb). With
// P.nwg the units of a sequence of t tiles are cut into n(t) = ceil(t / c) pieces each, c the smallest length, of
// those that a few bisections try, at which all pieces together are at most P.nwg: the pieces are then of nearly
// the same length, whatever the sequences' are, and all in flight at once. Each wave finds c by itself, lane i
// holding sequences i, i + 64, ... It costs 1 us of a call and saves what the longest sequence took more than the
// others with as many pieces for each (48 x 2 heads of eight on 7284-12554 rows 92 us with eight, now 84). Dealing the
// tiles out evenly, wherever units begin and end, was as fast for one row and slower for several (24 x 4 heads of 20 rows 48
// us where pieces took 40): a workgroup then begins and ends two units.
template <int RB, int TS>
struct Sched {
  int b, h, rb, len, first, count, piece, pieces, wg;

  __device__ __forceinline__ static int tiles(const Params& P, int len, int rb) {
    const int n = keys_seen(P, len, (min(P.S * P.G, (rb + 1) * RB) - 1) / P.G);   // the last row sees the most
    return max(1, (max(n, 0) + TS - 1) / TS);
  }
  __device__ __forceinline__ bool begin(const Params& P) {
    const int lane = threadIdx.x & 63;
    piece = first = 0;
    pieces = 1;
    if (P.nwg == 0) {
      // Row blocks of one (b, h) eight indices apart, on one XCD. The longest sequences first (16 x 16 x 512 rows on
      // 1109-6998 645 us in their own order, 534 so), and of an XCD's 64 workgroups that start at once, two a CU, the later
      // 32 the other way round, so that a long one shares its CU with a short one (4 x 16 x 509 on 1454-2353 93 us, 89 so)
      int j = (int)(blockIdx.x >> 3);
      const int most = min((int)(gridDim.x >> 3), 64);
      if (RB >= 64 && j >= 32 && j < most) j = 31 + most - j;
      rb = P.nrb - 1 - j % P.nrb;
      const int u = j / P.nrb * 8 + (int)(blockIdx.x & 7);
      if (u >= P.B * P.Hkv) return false;
      wg = 0;
      h = u % P.Hkv;
      b = u / P.Hkv;
      if (RB >= 64 && P.seqlens && P.B > 1 && P.B <= 64) {
        const int mine = lane < P.B ? cache_len(P, lane) : -1;
        int at = 0;
        for (int i = 0; i < P.B; ++i) {
          const int other = __builtin_amdgcn_readlane(mine, i);
          at += other > mine || (other == mine && i < lane);
        }
        b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < P.B && at == b));
        len = __builtin_amdgcn_readlane(mine, b);
      } else {
        len = __builtin_amdgcn_readfirstlane(cache_len(P, b));
      }
      count = tiles(P, len, rb);
      return true;
    }
    constexpr int NB = kMaxShared / 64;
    int lens[NB], t[NB], sum = 0;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      const int i = lane + 64 * k;
      lens[k] = i < P.B ? cache_len(P, i) : 0;
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      t[k] = lane + 64 * k < P.B ? tiles(P, lens[k], P.nrb - 1) : 0;
      sum += t[k];
    }
    const int units = P.Hkv * P.nrb, most = P.nwg / units;      // pieces of all sequences' units of one head and block
    const float total = (float)__builtin_amdgcn_readlane(wave_scan(sum), 63);
    auto cut = [&](float inv, int (&n)[NB]) {                   // the pieces of each sequence; their sum
      int s = 0;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        n[k] = (int)__builtin_ceilf((float)t[k] * inv);         // 0 for no sequence
        s += n[k];
      }
      return __builtin_amdgcn_readlane(wave_scan(s), 63);
    };
    // a sequence has at most t / c + 1 pieces: a length that is long enough, and one that none below could be
    int n[NB], lower[NB];
    float c1 = fmaxf(1.f, 1.001f * total / (float)max(1, most - P.B)), c0 = fmaxf(1.f, total / (float)most);
    if (most <= P.B || cut(1.f / c1, n) > most) {
      // rounding, or hardly more workgroups than units: one piece each
#pragma unroll
      for (int k = 0; k < NB; ++k) n[k] = t[k] ? 1 : 0;
    } else {
#pragma unroll 1
      for (int i = 0; i < 5; ++i) {
        const float c = i ? 0.5f * (c0 + c1) : c0;
        if (cut(1.f / c, lower) > most) {
          c0 = c;
        } else {
          c1 = c;
#pragma unroll
          for (int k = 0; k < NB; ++k) n[k] = lower[k];
          if (i == 0) break;
        }
      }
    }
    // the workgroups before each sequence
    wg = (int)blockIdx.x;
    int base = 0;
    b = -1;
#pragma unroll
    for (int k = 0; k < NB; ++k) {
      if (64 * k >= P.B) break;
      const int upto = base + units * wave_scan(n[k]);
      if (wg == 0 && threadIdx.x < 64 && lane + 64 * k < P.B) P.pre[lane + 64 * k + 1] = upto;
      const int end = __builtin_amdgcn_readlane(upto, 63);
      if (b < 0 && wg < end) {
        const int at = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= wg));
        b = 64 * k + at;
        len = __builtin_amdgcn_readlane(lens[k], at);
        pieces = __builtin_amdgcn_readlane(n[k], at);
        piece = wg - (__builtin_amdgcn_readlane(upto, at) - units * pieces);
      }
      base = end;
    }
    if (wg == 0 && threadIdx.x == 0) P.pre[0] = 0;
    if (b < 0) return false;
    const int u = piece / pieces;
    piece -= u * pieces;
    h = u / P.nrb;
    rb = u - h * P.nrb;
    // the pieces that there are no tiles for are empty
    const int all = tiles(P, len, rb), per = (all + pieces - 1) / pieces;
    first = min(all, piece * per);
    count = min(all - first, per);
    return true;
  }
  // The compiler does not see that all of it is the same for a whole wave
  __device__ __forceinline__ void settle() {
    for (int* x : {&b, &h, &rb, &len, &first, &count, &piece, &pieces, &wg}) *x = __builtin_amdgcn_readfirstlane(*x);
  }
  // where row r0 of the piece's result goes, if it is not the unit's
  template <int D>
  __device__ __forceinline__ float* partial(const Params& P) const {
    return pieces == 1 ? nullptr : P.part + (int64_t)wg * RB * kPart<D>;
  }
};

// 16 bytes a lane of 16 rows of a page, off a uniform base; ONCE: kept out of the caches
template <int D>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_rows(const bf16* p) { return make_rsrc(p, 16 * D * 2); }
template <bool ONCE>
__device__ __forceinline__ u32x4 page_chunk(__amdgpu_buffer_rsrc_t rows, uint32_t off) {
  return __builtin_amdgcn_raw_buffer_load_b128(rows, (int)off, 0, ONCE ? 2 : 0);
}
// 16 bytes of a row of a sequence: `cached`, or `at` elements into the new rows `fresh`; of zeros if it is not there, so
// that nothing waits for what is read
__device__ const u32x4 kNoRow = {0, 0, 0, 0};
__device__ __forceinline__ u32x4 row_chunk(bool there, bool old, const char* cached, const bf16* fresh, int64_t at) {
  const char* p = old ? cached : reinterpret_cast<const char*>(fresh + at);
  return *reinterpret_cast<const u32x4*>(there ? p : reinterpret_cast<const char*>(&kNoRow));
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

// Rows [r0, r1) over keys [k0, k1) without the matrix cores: 16 lanes a row, key by key. For pieces
// whose values hold an infinity or NaN (0 * inf in P V would reach rows that must not see the key), and
// for scores that pass fp32's range before the softmax scale, or whose largest is about -3e38: here the
// scale comes first. A scale of 0, which hides whether they did, brings every row here: right, and slow.
// down: what the unit's other pieces take the weights below.
template <int D>
__device__ __forceinline__ void walk_rows(const Params& P, int b, int h, int r0, int r1, int k0, int k1, int len, float down, float* part) {
  constexpr int E = D / 16;
  const int g16 = threadIdx.x & 15;
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
      const float alpha = __builtin_amdgcn_exp2f(m - ref), p = __builtin_amdgcn_exp2f(s - (ref + down));
      m = mx;
      l = l * alpha + p;
      get(vr, x);
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = o[e] * alpha + p * x[e];
    }
    if (!part) {
      const float inv = row_inv(seen != 0.f, l);
      bf16* dst = P.out + b * P.o_sb + i * P.o_ss + hq * P.o_sh + E * g16;
#pragma unroll
      for (int e = 0; e < E; ++e) dst[e] = (bf16)(o[e] * inv);
    } else {
      float* dst = part + (r - r0) * kPart<D>;
      if (g16 == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{m, l, seen, 0.f};
#pragma unroll
      for (int e = 0; e < E; ++e) dst[4 + E * g16 + e] = o[e];
    }
  }
}

// ---- one row ----------------------------------------------------------------------------------
// Sum over the D / 8 lanes that hold a key row
template <int D>
__device__ __forceinline__ float lanes_sum(float x) {
  x += dpp_f<0xB1>(x);                 // quad_perm [1,0,3,2]
  x += dpp_f<0x4E>(x);                 // quad_perm [2,3,0,1]
  x += dpp_f<0x141>(x);                // row_half_mirror
  if (D == 128) x += dpp_f<0x140>(x);  // row_mirror
  return x;
}

// R = 1. Each wave walks 16 NH keys at a time by itself; D / 8 lanes hold a key row, 16 bytes each. Bound by memory
// where there is much to read (64 x 16 heads on 2163-3972 rows, 1.58 GB: 250 us, 6.3 TB/s; 3 x 12 on 20735-25651, 428 MB,
// 69 us, 6.2), by the chain of length, page, keys, joining where there is little (16 heads on 783 rows 6.0 us, and 3.8
// the combine). The matrix cores (stream) are as fast on the former and 0.6 to 1.2 us slower on the latter.
template <int D, int NTH>
__global__ __launch_bounds__(NTH) void decode_kernel(Params P) {
  constexpr int NWAVE = NTH / 64, CH = D / 8, RPL = 64 / CH, NH = D == 128 ? 1 : 2, U = 16 / RPL;
  constexpr int kStep = 16 * NH * NWAVE;     // keys of a workgroup's step, a tile
  __shared__ float s_m[NWAVE], s_l[NWAVE], s_seen[NWAVE];
  __shared__ f32x4 s_o[NWAVE][D / 4];
  Sched<1, kStep> sc;
  if (!sc.begin(P)) return;
  sc.settle();
  const int b = sc.b, h = sc.h, len = sc.len;
  const int tid = threadIdx.x, lane = tid & 63, c8 = 8 * (lane % CH), grp = lane / CH;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lk = min(P.cap, len + P.s_new);
  const int k0 = sc.first * kStep;
  const int k1 = min(k0 + sc.count * kStep, lk);
  const int kold = min(k1, len);               // keys below are cached

  uniform_i32* const tab = uniform(P.table + b * P.table_sb);
  const int psm = (1 << P.ps_log2) - 1;
  const bf16 *const kn = P.k + b * P.k_sb + h * P.k_sh, *const vn = P.v + b * P.v_sb + h * P.v_sh;
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
      if (ok[hf] && j + 16 <= len) {
        const __amdgpu_buffer_rsrc_t kr = page_rows<D>(P.kp + at), vr = page_rows<D>(P.vp + at);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          kw[hf][u] = page_chunk<true>(kr, off + u * (RPL * D * 2));
          vw[hf][u] = page_chunk<true>(vr, off + u * (RPL * D * 2));
        }
      } else {
        // the last cached rows, the new one, none: row by row
        const char *kb = reinterpret_cast<const char*>(P.kp + at), *vb = reinterpret_cast<const char*>(P.vp + at);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int jr = j + u * RPL + grp;
          const bool old = jr < len, there = old ? ok[hf] : jr < lk;
          kw[hf][u] = row_chunk(there, old, kb + off + u * (RPL * D * 2), kn, (jr - len) * P.k_ss + c8);
          vw[hf][u] = row_chunk(there, old, vb + off + u * (RPL * D * 2), vn, (jr - len) * P.v_ss + c8);
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
  const float down = spread(lk);
  float q[8], o[8], m = -INFINITY, l = 0.f, seen = 0.f;
  {
    const u32x4 x = *reinterpret_cast<const u32x4*>(P.q + b * P.q_sb + h * P.q_sh + c8);
#pragma unroll
    for (int e = 0; e < 4; ++e) q[2 * e] = bf16lo(x[e]) * P.scale_log2, q[2 * e + 1] = bf16hi(x[e]) * P.scale_log2;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  for (; j0 < k1; j0 += kStep) {
    float s[NH][U];
    bool full = j0 + 16 * NH <= kold;
#pragma unroll
    for (int hf = 0; hf < NH; ++hf) {
      full = full && ok[hf];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) d += q[2 * e] * bf16lo(kw[hf][u][e]) + q[2 * e + 1] * bf16hi(kw[hf][u][e]);
        s[hf][u] = lanes_sum<D>(d);
      }
    }
    if (full) {
      seen = 1.f;
    } else {
      // what is not there weighs nothing; its values were read as 0
#pragma unroll
      for (int hf = 0; hf < NH; ++hf)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int j = j0 + 16 * hf + u * RPL + grp;
          const bool sees = j < k1 && (ok[hf] || j >= len);
          seen = sees ? 1.f : seen;
          s[hf][u] = sees ? s[hf][u] : -INFINITY;
        }
    }
    float mx = m;
#pragma unroll
    for (int hf = 0; hf < NH; ++hf)
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[hf][u]);
    const float ref = max_ref(mx), alpha = __builtin_amdgcn_exp2f(m - ref);   // m = -inf at first: 0
    m = mx;
    l *= alpha;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] *= alpha;
#pragma unroll
    for (int hf = 0; hf < NH; ++hf)
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = __builtin_amdgcn_exp2f(s[hf][u] - (ref + down));
        l += p;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          o[2 * e] += p * bf16lo(vw[hf][u][e]);
          o[2 * e + 1] += p * bf16hi(vw[hf][u][e]);
        }
      }
    if (j0 + kStep < k1) {
      load(j0 + kStep);
      look(j0 + 2 * kStep);
    }
  }
  // the wave's groups, then the waves
  float M = m;
#pragma unroll
  for (int x = CH; x < 64; x <<= 1) M = fmaxf(M, __shfl_xor(M, x));
  const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
  l *= a;
#pragma unroll
  for (int x = CH; x < 64; x <<= 1) {
    l += __shfl_xor(l, x);
    seen = fmaxf(seen, __shfl_xor(seen, x));
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    o[e] *= a;
#pragma unroll
    for (int x = CH; x < 64; x <<= 1) o[e] += __shfl_xor(o[e], x);
  }
  if (lane < CH) {
    if (lane == 0) s_m[w] = M, s_l[w] = l, s_seen[w] = seen;
    s_o[w][2 * lane] = f32x4{o[0], o[1], o[2], o[3]};
    s_o[w][2 * lane + 1] = f32x4{o[4], o[5], o[6], o[7]};
  }
  __syncthreads();
  if (tid < D / 4) {
    float L = 0.f, any = 0.f;
    M = s_m[0];
#pragma unroll
    for (int g = 1; g < NWAVE; ++g) M = fmaxf(M, s_m[g]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NWAVE; ++g) {
      const float wgt = s_m[g] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[g] - M);
      L += wgt * s_l[g];
      any = fmaxf(any, s_seen[g]);
      acc += wgt * s_o[g][tid];
    }
    if (float* part = sc.template partial<D>(P)) {
      if (tid == 0) *reinterpret_cast<f32x4*>(part) = f32x4{M, L, any, 0.f};
      *reinterpret_cast<f32x4*>(part + 4 + 4 * tid) = acc;
    } else {
      const float inv = row_inv(any != 0.f, L);
      *reinterpret_cast<bf16x4*>(P.out + b * P.o_sb + h * P.o_sh + 4 * tid) =
          cvt4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    }
  }
  append_share<D, NTH>(P, b, h, len, sc.piece, sc.pieces);
}

// ---- up to 16 rows -------------------------------------------------------------------------------
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

// R <= 16. Each wave walks 32 keys at a time by itself: S^T = K Q^T by 16 keys, then O^T += V^T P^T, K and V through LDS
// of its own, so that both are read from memory in whole rows (K straight into the matrix cores, 64 bytes of 16 rows a
// load, took 105 us where this took 92 then). Bound by memory: 48 x 2 key-value heads of eight query heads on 7284-12554
// rows, 479 MB, 81 us, 5.9 TB/s, and 5 the combine. Two workgroups a CU (72 KB of LDS, 212 registers).
template <int D>
__global__ __launch_bounds__(NT, 2) void stream_kernel(Params P) {
  using G = Geo<D>;
  constexpr int NS = G::NS, ND = G::ND, CH = G::CH, HL = ND / 2;   // HL: loads of 16 rows
  __shared__ __attribute__((aligned(16))) char smem[NWAVE][G::AREA];
  __shared__ float s_m[NWAVE][16], s_l[NWAVE][16], s_seen[NWAVE][16];
  __shared__ int s_bad;
  const int tid = threadIdx.x, lane = tid & 63, l16 = lane & 15, g4 = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  constexpr int kStep = kKeys * NWAVE;       // keys of a workgroup's step, a tile
  Sched<16, kStep> sc;
  if (!sc.begin(P)) return;
  sc.settle();
  const int b = sc.b, h = sc.h, len = sc.len, R = P.S * P.G;
  const int lk = min(P.cap, len + P.s_new);
  const int k0 = sc.first * kStep;
  const int k1 = min(k0 + sc.count * kStep, keys_seen(P, len, P.S - 1));   // the last row sees the most
  const int kall = keys_seen(P, len, 0);                             // every row sees the keys below
  if (tid == 0) s_bad = 0;

  uniform_i32* const tab = uniform(P.table + b * P.table_sb);
  const int psm = (1 << P.ps_log2) - 1;
  const bf16 *const kn = P.k + b * P.k_sb + h * P.k_sh, *const vn = P.v + b * P.v_sb + h * P.v_sh;
  char* const area = smem[w];

  u32x4 kw[ND], vw[ND];
  bool ok[2];              // the 16 keys have a page, or are new rows
  const uint32_t off = (uint32_t)(lane / CH * D + 8 * (lane % CH)) * 2;
  auto load = [&](int j0) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const int j = j0 + 16 * hf;
      const int page = j < len ? tab[j >> P.ps_log2] : -1;
      const bool held = (unsigned)page < (unsigned)P.P;
      const int64_t at = ((((int64_t)(held ? page : 0) * P.Hkv + h) << P.ps_log2) + (j & psm)) * D;
      ok[hf] = held;
      if (held && j + 16 <= len) {
        const __amdgpu_buffer_rsrc_t kr = page_rows<D>(P.kp + at), vr = page_rows<D>(P.vp + at);
#pragma unroll
        for (int u = 0; u < HL; ++u) {
          kw[hf * HL + u] = page_chunk<true>(kr, off + u * (G::RPL * D * 2));
          vw[hf * HL + u] = page_chunk<true>(vr, off + u * (G::RPL * D * 2));
        }
      } else {
        // the last cached rows, the new ones, none: row by row
        const char *kb = reinterpret_cast<const char*>(P.kp + at), *vb = reinterpret_cast<const char*>(P.vp + at);
#pragma unroll
        for (int u = 0; u < HL; ++u) {
          const int jr = j + u * G::RPL + lane / CH;
          const bool old = jr < len, there = old ? held : jr < lk;
          kw[hf * HL + u] = row_chunk(there, old, kb + off + u * (G::RPL * D * 2), kn, (jr - len) * P.k_ss + 8 * (lane % CH));
          vw[hf * HL + u] = row_chunk(there, old, vb + off + u * (G::RPL * D * 2), vn, (jr - len) * P.v_ss + 8 * (lane % CH));
        }
      }
    }
  };

  const float down = spread(lk);
  float m_run = -INFINITY, l_run = 0.f, seen = 0.f;
  f32x4 oacc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) oacc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int row = min(l16, R - 1), ri = row / P.G;         // this lane's row (past the last: that one, not stored)
  const int nlim = min(k1, keys_seen(P, len, ri));
  u16x2 vmag = {0, 0};

  int j0 = k0 + kKeys * w;
  if (j0 < k1) {
    load(j0);
    // Q^T: lane holds its row, columns 32 s + 8 g4 + 0..7
    bf16x8 qf[NS];
    const bf16* qp = P.q + b * P.q_sb + ri * P.q_ss + (h * P.G + row - ri * P.G) * P.q_sh + 8 * g4;
#pragma unroll
    for (int n = 0; n < NS; ++n) qf[n] = *reinterpret_cast<const bf16x8*>(qp + 32 * n);
    char* const karea = area + kKeys * G::VS;
    const char *const vt = area + (4 * g4 + (l16 >> 2)) * G::VS + 8 * (l16 & 3), *const kt = karea + l16 * G::KS + 16 * g4;
    const int lrow = lane / CH, c16 = 16 * (lane % CH);
    for (; j0 < k1; j0 += kStep) {
#pragma unroll
      for (int u = 0; u < ND; ++u) *reinterpret_cast<u32x4*>(karea + (u * G::RPL + lrow) * G::KS + c16) = kw[u];
#pragma unroll
      for (int u = 0; u < ND; ++u) {
        vmag = max_mag(vmag, vw[u]);
        *reinterpret_cast<u32x4*>(area + (u * G::RPL + lrow) * G::VS + c16) = vw[u];
      }
      // a page that is missing hides cached keys only
      const bool ok0 = ok[0], ok1 = ok[1];
      if (j0 + kStep < k1) load(j0 + kStep);
      // K: lane holds key l16 of 16, columns 32 n + 8 g4 + 0..7
      f32x4 s[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        s[hf] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NS; ++n)
          s[hf] = mfma16x16x32(*reinterpret_cast<const bf16x8*>(kt + 16 * hf * G::KS + 64 * n), qf[n], s[hf]);
        s[hf] *= P.scale_log2;   // before the mask: the scale may have any sign
      }
      if (j0 + kKeys > min(kall, k1) || !ok0 || !ok1) {
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = j0 + 16 * hf + 4 * g4 + r;
            const bool sees = j < nlim && ((hf ? ok1 : ok0) || j >= len);
            seen = sees ? 1.f : seen;
            s[hf][r] = sees ? s[hf][r] : -INFINITY;
          }
      } else {
        seen = 1.f;
      }
      float mx = s[0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx = fmaxf(mx, s[e >> 2][e & 3]);
      mx = rows_max(mx);
      if (__builtin_amdgcn_ballot_w64(mx > m_run) != 0) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
        m_run = m_new;
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < ND; ++d) oacc[d] *= alpha;
      }
      const float m_use = max_ref(m_run) + down;
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = __builtin_amdgcn_exp2f(s[i >> 2][i & 3] - m_use);
        l_run += e[i];
      }
      // the probabilities go into P V as three bf16 terms, which add up to their fp32 bits
      bf16x8 pt[3];
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
      // V^T: lane holds column 16 d + l16 of keys 4 g4 + 0..3 and 16 + 4 g4 + 0..3, as s has them
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const u32x2 x0 = lds_read_tr(vt, 32 * d), x1 = lds_read_tr(vt, 16 * G::VS + 32 * d);
        const bf16x8 vf = __builtin_bit_cast(bf16x8, u32x4{x0[0], x0[1], x1[0], x1[1]});
#pragma unroll
        for (int n = 0; n < 3; ++n) oacc[d] = mfma16x16x32(vf, pt[n], oacc[d]);
      }
    }
  }

  __syncthreads();   // s_bad is cleared
  l_run = rows_sum(l_run);
  // a score past the range upwards leaves NaN; one past it downwards (raw below -3.4e38) only counts
  // where every key that the row sees here scores about as low
  if (vmag[0] >= 0x7f80 || vmag[1] >= 0x7f80 ||
      (seen != 0.f && (l_run != l_run || m_run < 200.f - 3e38f * fabsf(P.scale_log2))))
    s_bad = 1;
  seen = rows_max(seen);
  // the waves' results meet
  float* const part = sc.template partial<D>(P);
  {
    float* o = reinterpret_cast<float*>(area) + l16 * G::OS + 4 * g4;
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(o + 16 * d) = oacc[d];
    if (g4 == 0) s_m[w][l16] = m_run, s_l[w][l16] = l_run, s_seen[w][l16] = seen;
  }
  __syncthreads();
  if (s_bad) {
    walk_rows<D>(P, b, h, 0, R, k0, k1, len, down, part);
  } else if (const int r = tid >> 4; r < R) {
    constexpr int E = D / 16;
    float M = s_m[0][r], L = 0.f, any = 0.f, x[E];
#pragma unroll
    for (int g = 1; g < NWAVE; ++g) M = fmaxf(M, s_m[g][r]);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = 0.f;
#pragma unroll
    for (int g = 0; g < NWAVE; ++g) {
      const float wgt = s_m[g][r] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s_m[g][r] - M);
      L += wgt * s_l[g][r];
      any = fmaxf(any, s_seen[g][r]);
      const float* src = reinterpret_cast<const float*>(smem[g]) + r * G::OS + E * l16;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(src + e);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[e + c] += wgt * y[c];
      }
    }
    if (!part) {
      const float inv = row_inv(any != 0.f, L);
      bf16* dst = P.out + b * P.o_sb + (r / P.G) * P.o_ss + (h * P.G + r % P.G) * P.o_sh + E * l16;
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<bf16x4*>(dst + e) = cvt4(x[e] * inv, x[e + 1] * inv, x[e + 2] * inv, x[e + 3] * inv);
    } else {
      float* dst = part + r * kPart<D>;
      if (l16 == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{M, L, any, 0.f};
#pragma unroll
      for (int e = 0; e < E; e += 4) *reinterpret_cast<f32x4*>(dst + 4 + E * l16 + e) = f32x4{x[e], x[e + 1], x[e + 2], x[e + 3]};
    }
  }
  append_share<D>(P, b, h, len, sc.piece, sc.pieces);
}

// ---- more rows ------------------------------------------------------------------------------------
// Workgroup = 32 QW rows of (b, h) over a unit's or a piece's keys: QW waves along the rows and KW = 4 / QW along the
// keys; a staged tile of 64 keys serves all of them. S^T = K Q^T with the row as the lane column, V^T from transposing
// reads. 4 x 16 heads x 509 rows on 1454-2353 take 89 us (402 TFLOP/s; first 124), on 1582-2028 84, 16 x 16 x 512 on
// 6053-6782 808 (557 TFLOP/s; first 890):
//  - the weights go into P V as three bf16 terms, the upper 8 bits of what the terms before leave, which hold the fp32
//    value as in the other kernels. Two, each rounded to nearest, took 75 and 706 us of the latter two, but left up to 90
//    2^-24 of sums that cancel and three times as many results off their nearest bf16 as a softmax in fp32 leaves;
//  - what a row's weights are relative to (m_run) is raised only once one passes it by 2^kAbove: any reference does;
//  - the scale is applied with that reference in one fma: to |scale|, a negative one having turned q's signs;
//  - tiles in one page or of new rows alone are loaded off one base, with the bounds that the buffer checks.
// Bound by the waves' own chains (two a SIMD): of an iteration's 4700 cycles for two tiles the matrix cores take 2050, the
// vector instructions 2200, loads and stores alone 2600. Loads that reach further ahead (one word of each line, two to five
// tiles before) made it 6 to 8% slower.
template <int D, int QW>
struct TileGeo {
  static constexpr int KW = 4 / QW, NK = QW == 4 ? 2 : 1;  // waves along the keys; times 32 keys a wave has of a tile
  static constexpr int TK = 32 * KW * NK;                // keys a tile
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

template <int D, int QW, bool WIDE>
__global__ __launch_bounds__(NT, 2) void tile_kernel(Params P) {
  using G = TileGeo<D, QW>;
  constexpr int KW = G::KW, NK = G::NK, TK = G::TK, NP = G::NP, NDT = G::NDT, NS = D / 16, CH = G::CH, RSD = G::RSD;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ int s_bad, s_hole;   // a value row or score is not finite; a tile had rows without a page
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hh = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int qw = w % QW, kw = w / QW;
  Sched<32 * QW, TK> sc;
  if (!sc.begin(P)) return;
  sc.settle();
  const int b = sc.b, h = sc.h, len = sc.len;
  const int R = P.S * P.G, r0 = sc.rb * 32 * QW, r1 = min(R, r0 + 32 * QW);
  const int k0 = sc.first * TK;
  const int k1 = min(k0 + sc.count * TK, keys_seen(P, len, (r1 - 1) / P.G));
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
  const bf16 *const kn = P.k + b * P.k_sb + h * P.k_sh, *const vn = P.v + b * P.v_sb + h * P.v_sh;
  const uint32_t koff = (uint32_t)((srow & 15) * D + 8 * sch) * 2, voff = (uint32_t)((vrow & 15) * D + 8 * sch) * 2;
  // and of new rows, which 31 bits reach over a tile unless they are very far apart
  const bool near = P.k_ss < (1 << 23) && P.v_ss < (1 << 23);
  static_assert(TK == 64, "WIDE: a tile lies in one page");
  const uint32_t kfar = (uint32_t)((srow & 15) * (int)P.k_ss + 8 * sch) * 2, vfar = (uint32_t)((vrow & 15) * (int)P.v_ss + 8 * sch) * 2;
  u32x4 ks[NP], vs[NP];
  int page[NP];                 // of this wave's keys of the tile to load next
  auto look = [&](int t0) {
    if (WIDE) {
      page[0] = t0 < len ? tab[t0 >> P.ps_log2] : -1;
      return;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int j = t0 + G::RPP * n + g16;
      page[n] = j < len ? tab[j >> P.ps_log2] : -1;
    }
  };
  auto load = [&](int t0) {
    if (WIDE && t0 + TK <= len && (unsigned)page[0] < (unsigned)P.P) {
      const int64_t at = ((((int64_t)page[0] * P.Hkv + h) << P.ps_log2) + (t0 & psm)) * D;
      const __amdgpu_buffer_rsrc_t kr = make_rsrc(P.kp + at, TK * D * 2), vr = make_rsrc(P.vp + at, TK * D * 2);
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        const int s = (G::RPP * n + g16) * D * 2;
        ks[n] = __builtin_amdgcn_raw_buffer_load_b128(kr, (int)koff, s, 0);
        vs[n] = __builtin_amdgcn_raw_buffer_load_b128(vr, (int)voff, s, 0);
      }
      return;
    }
    if (t0 >= len && near) {
      // new rows; 0 past the last
      const int rows = min(TK, k1 - t0);
      const __amdgpu_buffer_rsrc_t kr = make_rsrc(kn + (t0 - len) * P.k_ss, rows > 0 ? (uint32_t)((rows - 1) * (int)P.k_ss + D) * 2 : 0);
      const __amdgpu_buffer_rsrc_t vr = make_rsrc(vn + (t0 - len) * P.v_ss, rows > 0 ? (uint32_t)((rows - 1) * (int)P.v_ss + D) * 2 : 0);
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        ks[n] = __builtin_amdgcn_raw_buffer_load_b128(kr, (int)(kfar + (G::RPP * n + g16) * (int)P.k_ss * 2), 0, 0);
        vs[n] = __builtin_amdgcn_raw_buffer_load_b128(vr, (int)(vfar + (G::RPP * n + g16) * (int)P.v_ss * 2), 0, 0);
      }
      return;
    }
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      const int j = t0 + G::RPP * n + g16;
      const int pg = page[WIDE ? 0 : n];
      const bool held = j < len && (unsigned)pg < (unsigned)P.P;
      const int64_t at = ((((int64_t)(held ? pg : 0) * P.Hkv + h) << P.ps_log2) + (j & psm)) * D;
      if (held && j + 16 <= len) {
        ks[n] = page_chunk<false>(page_rows<D>(P.kp + at), koff);
        vs[n] = page_chunk<false>(page_rows<D>(P.vp + at), voff);
      } else {
        // the last cached rows and the first new ones, rows without a page: row by row
        if (j < min(len, k1) && !held) s_hole = 1;
        const char *kb = reinterpret_cast<const char*>(P.kp + at), *vb = reinterpret_cast<const char*>(P.vp + at);
        const int jk = j + (srow & 15), jv = j + (vrow & 15);
        ks[n] = row_chunk(jk < len ? held : jk < k1, jk < len, kb + koff, kn, (jk - len) * P.k_ss + 8 * sch);
        vs[n] = row_chunk(jv < len ? held : jv < k1, jv < len, vb + voff, vn, (jv - len) * P.v_ss + 8 * sch);
      }
    }
  };
  auto store = [&](int buf) {
    char* base = smem + buf * G::BUF + srow * RSD + sch * 16;
#pragma unroll
    for (int n = 0; n < NP; ++n) {
      *reinterpret_cast<u32x4*>(base + G::RPP * n * RSD) = ks[n];
      *reinterpret_cast<u32x4*>(base + G::TILE + G::RPP * n * RSD) = vs[n];
    }
  };

  const float down = spread(min(P.cap, len + P.s_new)) + kAbove;
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
      for (int s = 0; s < NS; ++s) {
        // -q for a negative scale
        u32x4 x = *reinterpret_cast<const u32x4*>(qp + 16 * s);
        const uint32_t flip = P.scale_log2 < 0.f ? 0x80008000u : 0u;
        for (int e = 0; e < 4; ++e) x[e] ^= flip;
        qf[s] = __builtin_bit_cast(bf16x8, x);
      }
    }
    store(0);
#pragma unroll
    for (int s = 0; s < NS; ++s) settle(__builtin_bit_cast(u32x4, qf[s]));
    __syncthreads();
    const float c = fabsf(P.scale_log2);
    for (int t = 0; t < nt; ++t) {
      const int buf = t & 1;
      if (t + 1 < nt) {
        load(k0 + (t + 1) * TK);
        look(k0 + (t + 2) * TK);
      }
      const int kk = k0 + t * TK + 32 * NK * kw;   // first key of this wave's
      if (kk < kend_w) {
        const char* kt = smem + buf * G::BUF + (32 * NK * kw + l32) * RSD + hh * 16;
        const char* vt = smem + buf * G::BUF + G::TILE + 32 * NK * kw * RSD + xt_lane_off<RSD>(lane);
        f32x16 sacc[NK];
#pragma unroll
        for (int x = 0; x < NK; ++x) {
#pragma unroll
          for (int r = 0; r < 16; ++r) sacc[x][r] = 0.f;
          bf16x8 ka[NS];
          ka[0] = *reinterpret_cast<const bf16x8*>(kt + 32 * x * RSD);
          ka[1] = *reinterpret_cast<const bf16x8*>(kt + 32 * x * RSD + 32);
#pragma unroll
          for (int s = 0; s < NS; ++s) {   // operands two steps ahead
            if (s + 2 < NS) ka[s + 2] = *reinterpret_cast<const bf16x8*>(kt + 32 * x * RSD + 32 * (s + 2));
            sched_fence();
            sacc[x] = mfma32x32x16(ka[s], qf[s], sacc[x]);
            sched_fence();
          }
        }
        const bool hole = s_hole != 0;
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < NK; ++x) {
          const int kx = kk + 32 * x;
          if (kx + 32 > min(kall, k1) || hole) {
            // key kx + 8 (r / 4) + 4 hh + r % 4 is seen iff it is below kq, and cached ones have a page
            bool ok[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              const int j = kx + 16 * g;
              ok[g] = !hole || j >= len || (unsigned)tab[j >> P.ps_log2] < (unsigned)P.P;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const int j = kx + 8 * (r >> 2) + 4 * hh + (r & 3);
              const bool sees = j < kq && (ok[r >> 3] || j >= len);
              seen = sees ? 1.f : seen;
              sacc[x][r] = sees ? sacc[x][r] : -INFINITY;
            }
          } else {
            seen = 1.f;
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sacc[x][r]);
        }
        mx = c * halves_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_run + kAbove) != 0) {
          const float m_new = fmaxf(m_run, mx);
          const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
          m_run = m_new;
          l_run *= alpha;
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[dt][r] *= alpha;
        }
        const float m_use = max_ref(m_run) + down;
#pragma unroll
        for (int x = 0; x < NK; ++x) {
          const char* vx = vt + 32 * x * RSD;
          u32x4 xt[2 * NDT];
          xt[0] = lds_read_xt<RSD>(vx, 0, 0);
          xt[1] = lds_read_xt<RSD>(vx, 0, 1);
          // 16 keys at a time: the weights' three bf16 terms, which add up to their fp32 bits, times V
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            float e[8], ps = 0.f;
            bf16x8 pt[3];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              e[i] = __builtin_amdgcn_exp2f(c * sacc[x][8 * half + i] - m_use);
              ps += e[i];
            }
            l_run += ps;
#pragma unroll
            for (int n = 0; n < 3; ++n) {
              u32x4 hi;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                hi[i] = pack_hi(__builtin_bit_cast(uint32_t, e[2 * i]), __builtin_bit_cast(uint32_t, e[2 * i + 1]));
              pt[n] = __builtin_bit_cast(bf16x8, hi);
#pragma unroll
              for (int i = 0; i < 8; ++i)   // exact
                e[i] -= __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, e[i]) & 0xffff0000u);
            }
#pragma unroll
            for (int dt = 0; dt < NDT; ++dt) {
              const int z = NDT * half + dt;
              if (z + 2 < 2 * NDT) xt[z + 2] = lds_read_xt<RSD>(vx, (z + 2) / NDT, (z + 2) % NDT);
#pragma unroll
              for (int n = 0; n < 3; ++n) oacc[dt] = mfma32x32x16(__builtin_bit_cast(bf16x8, xt[z]), pt[n], oacc[dt]);
            }
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
  bool bad = false;
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad = bad || !(fabsf(oacc[dt][r]) < INFINITY);
  if (bad || (seen != 0.f && (l_run != l_run || m_run < 200.f - 3e38f * fabsf(P.scale_log2))))
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
  float* const part = sc.template partial<D>(P);
  if (s_bad) {
    walk_rows<D>(P, b, h, r0, r1, k0, k1, len, down, part);
  } else if (kw == 0 && active) {
    if (!part) {
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
      float* dst = part + (row - r0) * kPart<D>;
      if (hh == 0) *reinterpret_cast<f32x4*>(dst) = f32x4{m_run, l_run, seen, 0.f};
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
        for (int m = 0; m < 4; ++m)
          *reinterpret_cast<f32x4*>(dst + 4 + 32 * dt + 8 * m + 4 * hh) =
              f32x4{oacc[dt][4 * m], oacc[dt][4 * m + 1], oacc[dt][4 * m + 2], oacc[dt][4 * m + 3]};
    }
  }
  append_share<D>(P, b, h, len, sc.rb * sc.pieces + sc.piece, P.nrb * sc.pieces);
}

// One wave per (b, h, r) of a unit of several pieces: lane i weighs the i-th, and D / 4 lanes a piece add their four
// columns, 64 pieces at a time. Bound by its loads one after another, what the sequence's units were cut into, then the
// pieces: 3.8 us with the launch for 16 rows of 13 pieces, 4.6 for 768 of five.
template <int D, int RB>
__global__ __launch_bounds__(256) void combine_kernel(Params P) {
  constexpr int L4 = D / 4, NG = 64 / L4;
  const int R = P.S * P.G;
  const int lane = threadIdx.x & 63, col = lane % L4, grp = lane / L4;
  const int u = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (u >= P.B * P.Hkv * R) return;
  const int bh = u / R, r = u - bh * R, b = bh / P.Hkv, h = bh - b * P.Hkv, rb = r / RB;
  uniform_i32* const pre = uniform(P.pre);
  const int base = pre[b], n = (pre[b + 1] - base) / (P.Hkv * P.nrb);
  if (n == 1) return;
  const float* src = P.part + ((int64_t)(base + (h * P.nrb + rb) * n) * RB + (r - rb * RB)) * kPart<D>;
  constexpr int64_t kNext = (int64_t)RB * kPart<D>;
  float M = -INFINITY, L = 0.f;
  bool seen = false;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = 0; p0 < n; p0 += 64) {
    const int m = min(64, n - p0);
    f32x4 head = {-INFINITY, 0.f, 0.f, 0.f};
    if (lane < m) head = *reinterpret_cast<const f32x4*>(src + (p0 + lane) * kNext);
    const float before = M;
    M = fmaxf(M, wave_max(head[0]));
    const float ref = max_ref(M), alpha = __builtin_amdgcn_exp2f(before - ref);   // 0 at first
    const float wgt = __builtin_amdgcn_exp2f(head[0] - ref);
    L = L * alpha + wgt * head[1];
    acc *= alpha;
    seen = seen || __builtin_amdgcn_ballot_w64(head[2] != 0.f) != 0;
    for (int s0 = 0; s0 < m; s0 += 8 * NG) {
      // eight loads in flight; past the last piece it again, not added (it may be inf)
      f32x4 o[8];
#pragma unroll
      for (int x = 0; x < 8; ++x)
        o[x] = *reinterpret_cast<const f32x4*>(src + (p0 + min(s0 + grp + NG * x, m - 1)) * kNext + 4 + 4 * col);
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int at = s0 + grp + NG * x;
        const f32x4 y = acc + __shfl(wgt, at & 63) * o[x];
        acc = at < m ? y : acc;
      }
    }
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) L += __shfl_xor(L, m);
#pragma unroll
  for (int m = L4; m < 64; m <<= 1)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], m);
  const float inv = row_inv(seen, L);
  if (grp == 0)
    *reinterpret_cast<bf16x4*>(P.out + b * P.o_sb + (r / P.G) * P.o_ss + (h * P.G + r % P.G) * P.o_sh + 4 * col) =
        cvt4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
}

}  // namespace pkv
}  // namespace prefixlm
