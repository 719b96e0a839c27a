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

// Sum of x over the threads before this one, and over all (NTH threads). s: 17 ints
__device__ __forceinline__ int scan(int x, int* s, int* total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int y = x;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int z = __shfl_up(y, d);
    if (lane >= d) y += z;
  }
  __syncthreads();   // s may be in use
  if (lane == 63) s[w] = y;
  __syncthreads();
  if (threadIdx.x < 64) {
    int v = lane < NTH / 64 ? s[lane] : 0;
#pragma unroll
    for (int d = 1; d < NTH / 64; d <<= 1) {
      const int z = __shfl_up(v, d);
      if (lane >= d) v += z;
    }
    if (lane < NTH / 64) s[lane] = v;
  }
  __syncthreads();
  *total = s[NTH / 64 - 1];
  return y - x + (w ? s[w - 1] : 0);
}

// The numbers p of [p0, P) for which pick(p, refs[p]), in order, 16384 at a time, into list[0, n): ends after
// the first 16384 that bring the count to `want`. Returns the count, which may pass `cap` numbers: those are
// counted, not written.
constexpr int kPer = 16;           // of one thread
template <class Pick>
__device__ __forceinline__ int list_pages(const int32_t* refs, int P, int want, int cap, int32_t* list, int* s, Pick pick) {
  int n = 0;
  for (int base = 0; base < P && n < want; base += NTH * kPer) {
    const int p0 = base + kPer * (int)threadIdx.x;
    int32_t x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = p0 + i < P ? refs[p0 + i] : 0;
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mask |= (p0 + i < P && pick(p0 + i, x[i]) ? 1u : 0u) << i;
    int total;
    int at = n + scan(__popc(mask), s, &total);
    while (mask) {
      const int i = __ffs(mask) - 1;
      mask &= mask - 1;
      if (at < cap) put(list + at, p0 + i);
      ++at;
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
// that needs one gets the k-th lowest free page.
__global__ __launch_bounds__(NTH) void reserve_kernel(ReserveParams P) {
  __shared__ int s_off[kMaxSeqs + 1];   // items before sequence n
  __shared__ int s_scan[NTH / 64 + 1], s_copies;
  const int tid = threadIdx.x;
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
  arrive();
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
  int n, c, rest;
  int32_t* e;
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
  const int nfree = W ? list_pages(P.refs, P.P, W, W, P.free_list, s_scan, [](int, int32_t r) { return r == 0; }) : 0;
  arrive();
  int needed = 0;
  for (int base = 0; base < W; base += NTH) {
    const int it = base + tid;
    bool needs = false, leaves = false;
    int p = -1;
    if (it < W) {
      item(it, &n, &c, &e, &rest);
      p = *e;
      if ((unsigned)p < (unsigned)P.P) {
        const int32_t* was = P.was + 3 * (int64_t)p;
        const int holders = fresh(was);
        leaves = holders > 1 && !(fresh(was + 1) == holders && fresh(was + 2) == it);
        needs = leaves;
      } else {
        needs = true;
      }
    }
    int total;
    const int rank = needed + scan(needs ? 1 : 0, s_scan, &total);
    needed += total;
    if (needs && rank < nfree) {
      const int to = fresh(P.free_list + rank);
      put(e, to);
      put(P.refs + to, 1);
      if (leaves) {
        add(P.refs + p, -1);
        if (rest) {
          int32_t* q = P.copies + 1 + 3 * atomicAdd(&s_copies, 1);
          q[0] = p, q[1] = to, q[2] = rest;
        }
      }
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

// ---- fork -----------------------------------------------------------------------------------
struct ForkParams {
  int32_t* refs;
  int32_t* table;
  const int32_t* parents;   // [N]
  int64_t table_sb;
  int N, M, P, TC;          // TC: columns a workgroup
};
// A workgroup has TC columns of every sequence: all entries are read before one is written.
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
// thread = one entry
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
// One workgroup. U pages are in use: the i-th of them from U on moves to the i-th free one below U.
__global__ __launch_bounds__(NTH) void compact_kernel(CompactParams P) {
  __shared__ int s_scan[NTH / 64 + 1];
  const int tid = threadIdx.x;
  int mine = 0, U;
  for (int p = tid; p < P.P; p += NTH) mine += P.refs[p] > 0;
  (void)scan(mine, s_scan, &U);
  int32_t* const list = P.moves + 1;
  // free below U, then used above: as many of one as of the other, and in this order by number
  const int n = list_pages(P.refs, P.P, 0x7fffffff, 2 * P.P, list, s_scan, [U](int p, int32_t r) { return (p < U) != (r > 0); });
  for (int p = U + tid; p < P.P; p += NTH) put(P.to + p, p);
  arrive();
  const int half = n >> 1;
  for (int i = tid; i < half; i += NTH) {
    const int dst = fresh(list + i), src = fresh(list + half + i);
    put(P.to + src, dst);
    P.refs[dst] = P.refs[src];
    P.refs[src] = 0;
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
// A wave has 4 KB of one head of one pair's page: four loads of 16 bytes a lane on their way
// together. blockIdx.y: layer and keys or values. heads = 1: a page's heads as one.
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
  const int n = P.count ? *P.count : P.n, kv = blockIdx.y & 1;
  const int64_t layer = blockIdx.y >> 1;
  const bf16* from = P.from[kv] + layer * P.from_layer;
  bf16* to = P.to[kv] + layer * P.to_layer;
  const uint32_t per = (uint32_t)P.heads * P.pieces;   // of a pair; n per < 2^31
  for (uint32_t u = w; u < n * per; u += nw) {
    const uint32_t pair = u / per, x = u - pair * per, head = x / P.pieces, piece = x - head * P.pieces;
    int a, b, elems = P.head_elems;
    if (P.rows) {
      a = P.src[3 * pair], b = P.src[3 * pair + 1];
      elems = P.src[3 * pair + 2] * P.row_elems;
    } else {
      a = P.src ? P.src[pair] : P.dst[n + pair], b = P.dst[pair];
    }
    if ((unsigned)a >= (unsigned)P.P_from || (unsigned)b >= (unsigned)P.P_to) continue;
    const bf16* s = from + ((int64_t)a * P.heads + head) * P.head_elems;
    bf16* d = to + ((int64_t)b * P.heads + head) * P.head_elems;
    u32x4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = piece * 2048 + 8 * (64 * i + lane);
      if (at < elems) v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s + at));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = piece * 2048 + 8 * (64 * i + lane);
      if (at < elems) __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4*>(d + at));
    }
  }
}

}  // namespace pages
}  // namespace prefixlm
