// The pages of a key-value cache: handing out, sharing, taking back, moving and copying them.
//
// refs[p] counts the entries of the table [N, M] that hold page p; 0: the page is free. All sums are of
// integers and every choice goes by an order of rows, columns or page numbers, so a call always
// ends the same. Page contents (all layers' keys and values) move in copy_kernel, from lists that the
// kernels before it leave in the workspace: how many, the host need not know.
#pragma once
#include "common.h"

namespace prefixlm {
namespace pages {

constexpr int NTH = 1024;          // of the kernels that are one workgroup
constexpr int kMaxSeqs = 8192;     // sequences of a table: their numbers of columns fit LDS

// What a workgroup writes and reads again, or counts with atomics, goes past the L1 cache
__device__ __forceinline__ int32_t fresh(const int32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void put(int32_t* p, int32_t x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void add(int32_t* p, int32_t x) { __hip_atomic_fetch_add(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void lower(int32_t* p, int32_t x) { __hip_atomic_fetch_min(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A barrier behind which what the workgroup wrote and added before it has arrived
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}

// Sum of x over the threads before this one, and over all (NTH threads). s: 16 ints
__device__ __forceinline__ int scan(int x, int* s, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, y = wave_scan(x);
  __syncthreads();   // s may be in use
  if (lane == 63) s[w] = y;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < NTH / 64; ++i) {
    before += i < w ? s[i] : 0;
    all += s[i];
  }
  *total = all;
  return y - x + before;
}

// 16 counts a thread, 16384 pages the workgroup: from page `base` on, 0 past the end
constexpr int kPer = 16, kLook = NTH * kPer;
__device__ __forceinline__ void look(const int32_t* refs, int P, int base, int32_t (&x)[kPer]) {
  typedef int32_t i32x4 __attribute__((ext_vector_type(4), aligned(4)));
  const int p0 = base + kPer * (int)threadIdx.x;
  if (p0 + kPer <= P) {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) {
      const i32x4 y = *reinterpret_cast<const i32x4*>(refs + p0 + i);
      x[i] = y[0], x[i + 1] = y[1], x[i + 2] = y[2], x[i + 3] = y[3];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = p0 + i < P ? refs[p0 + i] : 0;
  }
}
// Bit i: pick(p, x[i]) for the page p = base + 16 thread + i
template <class Pick>
__device__ __forceinline__ uint32_t picked(int P, int base, const int32_t (&x)[kPer], Pick pick) {
  const int p0 = base + kPer * (int)threadIdx.x;
  uint32_t mask = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) mask |= (p0 + i < P && pick(p0 + i, x[i]) ? 1u : 0u) << i;
  return mask;
}
// The pages for which pick(p, refs[p]), in order, 16384 at a time (the first of them given in x), by put_one(rank, p):
// ends after the first 16384 that bring the count to `want`. Returns the count.
template <class Pick, class Put>
__device__ __forceinline__ int list_pages(const int32_t* refs, int P, int want, int32_t (&x)[kPer], int* s, Pick pick, Put put_one) {
  int n = 0;
  for (int base = 0; base < P && n < want; base += kLook) {
    if (base) look(refs, P, base, x);
    uint32_t mask = picked(P, base, x, pick);
    int total;
    int at = n + scan(__popc(mask), s, &total);
    while (mask) {
      const int i = __ffs(mask) - 1;
      mask &= mask - 1;
      put_one(at++, base + kPer * (int)threadIdx.x + i);
    }
    n += total;
  }
  return n;
}

// ---- reserve ------------------------------------------------------------------------------
struct ReserveParams {
  int32_t* refs;            // [P]
  int32_t* table;           // [N, M]
  const int32_t* seqlens;   // device [N]; null: seqlen_const
  const int32_t* new_rows;  // device [N]; null: new_const
  int32_t* short_;          // [N]: columns that are left without a page of the sequence's own
  int32_t* free_list;       // workspace [min(P, N M)]
  int32_t* was;             // workspace [P, 3]: holders before, entries that ask, the first of them
  int32_t* copies;          // workspace [1 + 3 N]: how many, then (from, to, rows) each
  int64_t table_sb;
  int N, M, P, ps_log2, seqlen_const, new_const;
};

// The columns [c0, c1) that rows len .. len + new - 1 of sequence n lie in
__device__ __forceinline__ void columns(const ReserveParams& P, int n, int* c0, int* c1, int* len) {
  const int cap = P.M << P.ps_log2;
  const int a = min(max(P.seqlens ? P.seqlens[n] : P.seqlen_const, 0), cap);
  const int more = max(P.new_rows ? P.new_rows[n] : P.new_const, 0);
  const int end = a + min(more, cap - a);
  *len = a;
  *c0 = a >> P.ps_log2;
  *c1 = end > a ? (end + (1 << P.ps_log2) - 1) >> P.ps_log2 : *c0;
}

// One workgroup. The columns of all sequences, in order, are its items. An item needs a page if it has
// none, or one that others hold too: unless all who hold it ask here and it is the first of them. The k-th
// that needs one gets the k-th lowest free page. Bound by the chain of dependent loads and barriers: lengths,
// entries, their counts, and the scan of the free pages meanwhile. Up to 1024 items keep what they know in
// registers and meet in a table in LDS; more go through the workspace, round after round. 64 columns that share pages,
// of 800 pages, 6.0 us; 925 columns of 4300 pages 6.7 (13.0 through the workspace).
constexpr int kSlots = 2 * NTH;    // of the table
__global__ __launch_bounds__(NTH) void reserve_kernel(ReserveParams P) {
  __shared__ int s_off[kMaxSeqs + 1];   // items before sequence n
  __shared__ int s_scan[NTH / 64], s_copies;
  __shared__ int s_page[kSlots], s_asks[kSlots], s_first[kSlots], s_free[NTH];
  const int tid = threadIdx.x;
  int32_t refs[kPer];
  look(P.refs, P.P, 0, refs);
  for (int i = tid; i < kSlots; i += NTH) s_page[i] = -1, s_asks[i] = 0, s_first[i] = 0x7fffffff;
  if (tid == 0) s_copies = 0;
  int W = 0;
  for (int base = 0; base < P.N; base += NTH) {
    int c0 = 0, c1 = 0, len;
    const int n = base + tid;
    if (n < P.N) {
      columns(P, n, &c0, &c1, &len);
      put(P.short_ + n, 0);
    }
    int total;
    const int at = scan(c1 - c0, s_scan, &total);
    if (n < P.N) s_off[n] = W + at;
    W += total;
  }
  if (tid == 0) s_off[P.N] = W;
  __syncthreads();
  // item -> its sequence, column, entry
  auto item = [&](int it, int* n, int* c, int32_t** e, int* rest) {
    int lo = 0, hi = P.N;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_off[mid] <= it) lo = mid; else hi = mid;
    }
    int c0, c1, len;
    columns(P, lo, &c0, &c1, &len);
    *n = lo;
    *c = c0 + it - s_off[lo];
    *e = P.table + lo * P.table_sb + *c;
    *rest = *c == c0 ? len & ((1 << P.ps_log2) - 1) : 0;
  };
  int n = 0, c, rest = 0;
  int32_t* e = nullptr;
  auto grant = [&](int to, int p, bool leaves) {
    put(e, to);
    put(P.refs + to, 1);
    if (!leaves) return;
    add(P.refs + p, -1);
    if (!rest) return;
    int32_t* q = P.copies + 1 + 3 * atomicAdd(&s_copies, 1);
    q[0] = p, q[1] = to, q[2] = rest;
  };
  auto is_free = [](int, int32_t r) { return r == 0; };
  int needed = 0, nfree = 0;
  if (W <= NTH) {
    int p = -1;
    if (tid < W) {
      item(tid, &n, &c, &e, &rest);
      p = *e;
    }
    if (W) nfree = list_pages(P.refs, P.P, W, refs, s_scan, is_free, [&](int k, int page) { if (k < NTH) s_free[k] = page; });
    const bool held = (unsigned)p < (unsigned)P.P;
    const int holders = tid < W && held ? P.refs[p] : 0;
    int at = (int)(((uint32_t)p * 2654435761u) >> 21);   // of 2048 slots, which at most half are taken
    if (holders > 1) {
      for (;; at = (at + 1) & (kSlots - 1)) {
        const int old = atomicCAS(&s_page[at], -1, p);
        if (old == -1 || old == p) break;
      }
      atomicAdd(&s_asks[at], 1);
      atomicMin(&s_first[at], tid);
    }
    __syncthreads();
    const bool leaves = holders > 1 && !(s_asks[at] == holders && s_first[at] == tid);
    const bool needs = tid < W && (!held || leaves);
    const int rank = scan(needs ? 1 : 0, s_scan, &needed);
    if (needs && rank < nfree) grant(s_free[rank], p, leaves);
  } else {
    for (int it = tid; it < W; it += NTH) {
      item(it, &n, &c, &e, &rest);
      const int p = *e;
      if ((unsigned)p >= (unsigned)P.P) continue;
      put(P.was + 3 * (int64_t)p, P.refs[p]);
      put(P.was + 3 * (int64_t)p + 1, 0);
      put(P.was + 3 * (int64_t)p + 2, 0x7fffffff);
    }
    arrive();
    for (int it = tid; it < W; it += NTH) {
      item(it, &n, &c, &e, &rest);
      const int p = *e;
      if ((unsigned)p >= (unsigned)P.P) continue;
      add(P.was + 3 * (int64_t)p + 1, 1);
      lower(P.was + 3 * (int64_t)p + 2, it);
    }
    nfree = list_pages(P.refs, P.P, W, refs, s_scan, is_free, [&](int k, int page) { if (k < W) put(P.free_list + k, page); });
    arrive();
    for (int base = 0; base < W; base += NTH) {
      const int it = base + tid;
      bool needs = false, leaves = false;
      int p = -1;
      if (it < W) {
        item(it, &n, &c, &e, &rest);
        p = *e;
        needs = (unsigned)p >= (unsigned)P.P;
        if (!needs) {
          const int32_t* was = P.was + 3 * (int64_t)p;
          const int holders = fresh(was), asks = fresh(was + 1), first = fresh(was + 2);
          needs = leaves = holders > 1 && !(asks == holders && first == it);
        }
      }
      int total;
      const int rank = needed + scan(needs ? 1 : 0, s_scan, &total);
      needed += total;
      if (needs && rank < nfree) grant(fresh(P.free_list + rank), p, leaves);
    }
  }
  arrive();
  if (tid == 0) P.copies[0] = s_copies;
  if (needed > nfree)
    for (int it = tid; it < W; it += NTH) {
      item(it, &n, &c, &e, &rest);
      const int p = fresh(e);
      if ((unsigned)p >= (unsigned)P.P || fresh(P.refs + p) > 1) add(P.short_ + n, 1);
    }
}
static_assert(kSlots == 2048, "the slot is 11 bits");

// ---- fork -----------------------------------------------------------------------------------
struct ForkParams {
  int32_t* refs;
  int32_t* table;
  const int32_t* parents;   // [N]
  int64_t table_sb;
  int N, M, P, TC;          // TC: columns a workgroup
};
// A workgroup has TC columns of every sequence: all entries are read before one is written. Latency: 64 sequences of 37
// columns 3.2 us. Counts change by integer atomics, whose order changes nothing.
__global__ __launch_bounds__(NTH) void fork_kernel(ForkParams P) {
  extern __shared__ int32_t s_new[];   // [N, TC]
  const int c0 = blockIdx.x * P.TC, total = P.N * P.TC;
  for (int i = threadIdx.x; i < total; i += NTH) {
    const int n = i / P.TC, c = c0 + i - n * P.TC, from = P.parents[n];
    if (c >= P.M || from == n || (unsigned)from >= (unsigned)P.N) continue;
    const int before = P.table[n * P.table_sb + c], x = P.table[from * P.table_sb + c];
    s_new[i] = x;
    if (before == x) continue;
    if ((unsigned)x < (unsigned)P.P) add(P.refs + x, 1);
    if ((unsigned)before < (unsigned)P.P) add(P.refs + before, -1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += NTH) {
    const int n = i / P.TC, c = c0 + i - n * P.TC, from = P.parents[n];
    if (c >= P.M || from == n || (unsigned)from >= (unsigned)P.N) continue;
    P.table[n * P.table_sb + c] = s_new[i];
  }
}

// ---- free -------------------------------------------------------------------------------------
struct FreeParams {
  int32_t* refs;
  int32_t* table;
  const int32_t* keep;      // [N]; null: keep_const
  int64_t table_sb;
  int N, M, P, ps_log2, keep_const;
};
// thread = one entry: 64 x 32 in 4.4 us, of which the launch is most
__global__ __launch_bounds__(256) void free_kernel(FreeParams P) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)P.N * P.M) return;
  const int n = (int)(i / P.M), c = (int)(i - (int64_t)n * P.M);
  if (((int64_t)c << P.ps_log2) < (P.keep ? P.keep[n] : P.keep_const)) return;
  int32_t* e = P.table + n * P.table_sb + c;
  const int p = *e;
  if ((unsigned)p < (unsigned)P.P) add(P.refs + p, -1);
  if (p != -1) *e = -1;
}

// ---- compact ---------------------------------------------------------------------------------
struct CompactParams {
  int32_t* refs;
  int32_t* table;
  int32_t* used;            // [1]
  int32_t* moves;           // workspace [1 + P + P]: how many, the free pages below `used`, the pages above
  int32_t* to;              // workspace [P]: where a page from `used` on goes
  int64_t table_sb;
  int N, M, P;
};
// One workgroup. U pages are in use: the i-th of them from U on moves to the i-th free one below U. Pools of up to
// 16384 pages stay in registers between the two looks at their counts; the free ones meet the others in LDS. Bound by
// its loads, two scans and stores: 1500 pages 6.0 us, 400 5.5.
__global__ __launch_bounds__(NTH) void compact_kernel(CompactParams P) {
  __shared__ int s_scan[NTH / 64];
  __shared__ uint16_t s_hole[kLook / 2];
  const int tid = threadIdx.x;
  int32_t* const list = P.moves + 1;
  int32_t x[kPer];
  look(P.refs, P.P, 0, x);
  int mine = 0, U, half;
#pragma unroll
  for (int i = 0; i < kPer; ++i) mine += x[i] > 0;
  for (int p = kLook + tid; p < P.P; p += NTH) mine += P.refs[p] > 0;
  (void)scan(mine, s_scan, &U);
  // free below U, then used above: as many of one as of the other, and in this order by number
  auto pick = [U](int p, int32_t r) { return (p < U) != (r > 0); };
  if (P.P <= kLook) {
    const uint32_t mask = picked(P.P, 0, x, pick);
    int total;
    const int at0 = scan(__popc(mask), s_scan, &total);
    half = total >> 1;
    int at = at0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = kPer * tid + i;
      if ((mask >> i & 1) && p < U) s_hole[at++] = (uint16_t)p;
    }
    __syncthreads();
    at = at0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int p = kPer * tid + i;
      if (p >= U && p < P.P) {
        int dst = p;
        if (mask >> i & 1) {
          dst = s_hole[at - half];
          list[at - half] = dst;
          list[at++] = p;
          P.refs[dst] = x[i];
          P.refs[p] = 0;
        }
        P.to[p] = dst;
      } else {
        at += mask >> i & 1;
      }
    }
  } else {
    const int n = list_pages(P.refs, P.P, 0x7fffffff, x, s_scan, pick, [&](int k, int p) { put(list + k, p); });
    half = n >> 1;
    for (int p = U + tid; p < P.P; p += NTH) put(P.to + p, p);
    arrive();
    for (int i = tid; i < half; i += NTH) {
      const int dst = fresh(list + i), src = fresh(list + half + i);
      put(P.to + src, dst);
      P.refs[dst] = P.refs[src];
      P.refs[src] = 0;
    }
  }
  if (tid == 0) {
    P.moves[0] = half;
    *P.used = U;
  }
}

// ---- contents ---------------------------------------------------------------------------------
struct CopyParams {
  const bf16* from[2];      // keys' and values' pages, all layers
  bf16* to[2];
  const int32_t* src;       // pairs; with rows: (from, to, rows) three words apart; null: behind dst's
  const int32_t* dst;
  const int32_t* count;     // how many, on the device; null: n
  int64_t from_layer, to_layer;   // elements of a layer
  int n, P_from, P_to, heads, head_elems, row_elems, rows;
  int pieces;               // of a head, 4 KB each
  // compact: entries of the table from `used` on become to_page's
  int32_t* table;
  const int32_t* to_page;
  const int32_t* used;
  int64_t table_sb;
  int N, M, n_remap;        // workgroups that do so, before the others
};
typedef const __attribute__((address_space(4))) int32_t uniform_i32;   // through the scalar cache
// A wave has 4 KB of one head of one pair's page at a time, four loads of 16 bytes a lane, and loads the next before
// it stores these. blockIdx.y: layer and keys or values. heads = 1: a page's heads as one. Bound by memory (1.26
// GB in and out 247 us, 5.1 TB/s); little by its chain of count, pair, load and store.
__global__ __launch_bounds__(256) void copy_kernel(CopyParams P) {
  int blk = blockIdx.x;
  if (blk < P.n_remap) {
    if (blockIdx.y) return;
    const int used = *P.used;
    for (int64_t i = (int64_t)blk * 256 + threadIdx.x; i < (int64_t)P.N * P.M; i += (int64_t)P.n_remap * 256) {
      const int n = (int)(i / P.M);
      int32_t* e = P.table + n * P.table_sb + (i - (int64_t)n * P.M);
      if (*e >= used && *e < P.P_to) *e = P.to_page[*e];
    }
    return;
  }
  blk -= P.n_remap;
  const int lane = threadIdx.x & 63;
  const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane(blk * 4 + (threadIdx.x >> 6));
  const uint32_t nw = 4 * (gridDim.x - P.n_remap);
  const int n = P.count ? *(uniform_i32*)(uintptr_t)P.count : P.n, kv = blockIdx.y & 1;
  const int64_t layer = blockIdx.y >> 1;
  const bf16* from = P.from[kv] + layer * P.from_layer;
  bf16* to = P.to[kv] + layer * P.to_layer;
  uniform_i32 *const src = (uniform_i32*)(uintptr_t)P.src, *const dst = (uniform_i32*)(uintptr_t)P.dst;
  const uint32_t per = (uint32_t)P.heads * P.pieces, total = n * per;   // n per < 2^31
  struct Piece {
    bf16* d;
    int elems;               // of the head from this piece on; 0: nothing
    u32x4 v[4];
  };
  auto load = [&](uint32_t u, Piece& x) {
    x.elems = 0;
    if (u >= total) return;
    const uint32_t pair = u / per, y = u - pair * per, head = y / P.pieces, piece = y - head * P.pieces;
    int a, b, elems = P.head_elems;
    if (P.rows) {
      a = src[3 * pair], b = src[3 * pair + 1];
      elems = src[3 * pair + 2] * P.row_elems;
    } else {
      b = dst[pair], a = P.src ? src[pair] : dst[n + pair];
    }
    if ((unsigned)a >= (unsigned)P.P_from || (unsigned)b >= (unsigned)P.P_to) return;
    const bf16* s = from + ((int64_t)a * P.heads + head) * P.head_elems + piece * 2048;
    x.d = to + ((int64_t)b * P.heads + head) * P.head_elems + piece * 2048;
    x.elems = elems - (int)piece * 2048;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 8 * (64 * i + lane);
      if (at < x.elems) x.v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s + at));
    }
  };
  auto store = [&](const Piece& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = 8 * (64 * i + lane);
      if (at < x.elems) __builtin_nontemporal_store(x.v[i], reinterpret_cast<u32x4*>(x.d + at));
    }
  };
  // total < 2^31 and a step is below 2^17: no overflow
  Piece x, y;
  load(w, x);
  for (uint32_t u = w; u < total; u += 2 * nw) {
    load(u + nw, y);
    store(x);
    load(u + 2 * nw, x);
    store(y);
  }
}

}  // namespace pages
}  // namespace prefixlm
