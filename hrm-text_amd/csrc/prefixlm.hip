// C ABI of the gfx950 PrefixLM attention library (declared in include/prefixlm.h).
//
// Host-side validation, workspace carving and kernel launches. The library keeps
// no state between calls except (a) a thread-local error string and (b) a one-time
// per-process kernel attribute setup; timing records live in caller-owned timers.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>
#include <mutex>
#include <new>
#include <vector>

#include "prefixlm.h"
#include "common.h"
#include "worklist.h"
#include "fwd.h"
#include "bwd.h"
#include "plan.h"
#include "rope.h"
#include "kvcache.h"
#include "kvcache8.h"
#include "norm_mlp.h"
#include "gemm.h"
#include "logprob.h"
#include "embed.h"
#include "paged.h"
#include "pages.h"

using namespace prefixlm;

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

constexpr size_t kAlign = 256;
size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

// Stored dS of the dQ-from-dS backward: per head, one 4 KB block (32 queries x 64 keys)
// per attended (key group, query tile) of every segment, in the layout of ds_blk_off
// (worklist.h), from ds_base[s] on. The host scalars bound the blocks per head by
// sum_s ceil(L_s / 32) * ceil(L_s / 64) <= (num_tokens / 32 + numseqs + 1) *
// ceil(max_seqlen_all / 64); a plan knows the exact count. Scales: one per 128-key tile,
// slot (cu_seqlens[s] + k) / 128 + s, below num_tokens / 128 + numseqs + 1.
int64_t ds_bound_blocks(int32_t T, int32_t numseqs, int32_t max_all) {
  return ((int64_t)T / 32 + numseqs + 1) * (((int64_t)max_all + 63) / 64);
}
int64_t ds_nkslot(int32_t T, int32_t numseqs) { return (int64_t)T / 128 + numseqs + 1; }

int64_t max_items(int32_t total, int32_t numseqs, int tile) {
  return (int64_t)(total + tile - 1) / tile + numseqs;
}

// The three lists of a host plan, in the order and with the parameters of the
// device-built lists (forward; backward dK/dV; backward dQ).
const plan::ListDesc kPlanLists[plan::kLists] = {
    {0, fwd::BM, fwd::BN}, {1, bwd::kv::BK, bwd::kv::BQ}, {0, bwd::qk::BQ, bwd::qk::BKT}};

// Checks a caller's plan against this call's scalars; returns its layout.
int check_plan(const void* p, size_t bytes, int32_t total, int32_t numseqs, plan::Layout* l) {
  *l = plan::layout(kPlanLists, total, numseqs);
  if (!p) return fail(PREFIXLM_ERR_INVALID, "plan pointer is null");
  if ((reinterpret_cast<uintptr_t>(p) & 255u) != 0)
    return fail(PREFIXLM_ERR_INVALID, "plan must be 256-byte aligned");
  if (bytes != l->bytes)
    return fail(PREFIXLM_ERR_INVALID,
                "plan of %zu bytes, a batch with total_seqlen=%d and numseqs=%d has %zu: the plan was "
                "built for other metadata",
                bytes, total, numseqs, l->bytes);
  return PREFIXLM_OK;
}

// ---- optional per-kernel timing ---------------------------------------------------
// Caller-owned: a prefixlm_timer (prefixlm_timer_create) passed in the args collects
// one pair of HIP events around each launch; the library itself keeps no records.
struct TimingRec {
  int id;
  hipEvent_t a, b;
};

}  // namespace

struct prefixlm_timer {
  std::vector<TimingRec> recs;
  std::vector<hipEvent_t> pool;
  hipEvent_t get() {
    if (!pool.empty()) {
      hipEvent_t e = pool.back();
      pool.pop_back();
      return e;
    }
    hipEvent_t e = nullptr;
    if (hipEventCreate(&e) != hipSuccess) return nullptr;
    return e;
  }
};

namespace {

struct KernelTimer {
  prefixlm_timer* t;
  int id;
  hipStream_t s;
  hipEvent_t a = nullptr, b = nullptr;
  KernelTimer(void* timer, int id_, hipStream_t s_) : t(static_cast<prefixlm_timer*>(timer)), id(id_), s(s_) {
    if (!t) return;
    a = t->get();
    b = t->get();
    if (a && b && hipEventRecord(a, s) != hipSuccess) a = b = nullptr;
  }
  ~KernelTimer() {
    if (!(a && b)) return;
    if (hipEventRecord(b, s) == hipSuccess) t->recs.push_back({id, a, b});
  }
};

std::once_flag g_attr_once;
hipError_t g_attr_err = hipSuccess;
void set_kernel_attrs() {
  std::call_once(g_attr_once, [] {
    g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd::prefixlm_fwd_kernel<128>),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, fwd::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd::prefixlm_fwd_kernel<64>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, fwd::Geo<64>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&bwd::prefixlm_bwd_dkdv_kernel<128>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bwd::kv::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&bwd::prefixlm_bwd_dkdv_kernel<64>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bwd::kv::Geo<64>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&bwd::prefixlm_bwd_dq_kernel<128>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bwd::qk::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&bwd::prefixlm_bwd_dq_kernel<64>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bwd::qk::Geo<64>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&bwd::prefixlm_bwd_dq_ds_kernel<128>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bwd::q2::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&bwd::prefixlm_bwd_dq_ds_kernel<64>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, bwd::q2::Geo<64>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd::prefixlm_fwd_kernel<128, true>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, fwd::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd::prefixlm_fwd_kernel<128, true, 2>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, 2 * fwd::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd::prefixlm_fwd_kernel<128, false, 2>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, 2 * fwd::Geo<128>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&fwd::prefixlm_fwd_kernel<64, false, 2>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, 2 * fwd::Geo<64>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&kvc::extend_kernel<1>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, kvc::ExtGeo<1>::LDS_BYTES);
    if (g_attr_err == hipSuccess)
      g_attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(&kvc::extend_kernel<2>),
                                       hipFuncAttributeMaxDynamicSharedMemorySize, kvc::ExtGeo<2>::LDS_BYTES);
  });
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Workgroups of a persistent grid with one workgroup per CU: the current device's CU
// count rounded down to a multiple of 8 (the XCD count; the kernels take work from
// per-XCD counters). Cached per device.
std::mutex g_cu_mu;
int g_cu_count[64] = {};
int persistent_grid(int* out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
  if (dev < 0 || dev >= 64) return fail(PREFIXLM_ERR_INVALID, "device %d >= 64", dev);
  std::lock_guard<std::mutex> g(g_cu_mu);
  if (!g_cu_count[dev]) {
    int n = 0;
    e = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev);
    if (e != hipSuccess || n < 1)
      return fail(PREFIXLM_ERR_HIP, "hipDeviceGetAttribute(multiprocessor count): %s", hipGetErrorString(e));
    g_cu_count[dev] = n >= 8 ? n / 8 * 8 : 8;
  }
  *out = g_cu_count[dev];
  return PREFIXLM_OK;
}

// Whether the forward deals each item's key tiles to two groups of waves: its grid leaves every
// CU one workgroup at most, and the segments are long enough (8 key tiles) for half the tiles to
// outweigh the merge.
int fwd_splits_keys(int64_t grid, int32_t max_all, bool* split) {
  int cus = 0;
  const int rc = persistent_grid(&cus);
  *split = grid <= cus && max_all >= 8 * fwd::BN;
  return rc;
}

// Whether the forward's workgroups find their items themselves instead of reading a cost-ordered
// list, which a launch before it would have to build (about 4.8 us). The order only matters once
// workgroups wait for others: grids of up to 1.25 workgroups per CU gain the whole launch (H 16 x
// d128, us with and without the list: 2048 rows in 4 segments, 320 workgroups, 33.2 and 28.1; 280
// 53.9 and 49.0; but 536 with segments of up to 4096 rows 128 and 142), and where no segment is
// longer than 1024 rows, grids of up to three per CU (416 workgroups 21.3 and 16.2, 640 39.5 and
// 36.7; at 1280 56.1 and 56.4). One wave reads the metadata: 64 segments.
int fwd_finds_items(int64_t grid, int32_t numseqs, int32_t max_all, bool* self) {
  int cus = 0;
  const int rc = persistent_grid(&cus);
  *self = grid > 0 && numseqs <= 64 && (4 * grid <= 5 * (int64_t)cus || (max_all <= 1024 && grid <= 3 * (int64_t)cus));
  return rc;
}

// The forward's and backward's buffer offsets inside one segment are 32-bit byte offsets:
// (rows + 256) rows of 16-bit elements take less than 2^31 bytes
bool segment_fits(int64_t rows, int64_t token_stride) { return token_stride <= (((int64_t)1 << 30) - 1) / (rows + 256); }

// Checks shared by forward and backward. `strides` lists (stride_t, stride_h) pairs.
int check_common(const void* const* ptrs, int nptr, const int64_t* strides, int nstr,
                 int32_t T, int32_t H, int32_t D, int32_t total, int32_t numseqs,
                 int32_t max_all, int64_t meta_len, const int32_t* pre, const int32_t* cau,
                 const int32_t* cu) {
  if (D != 128 && D != 64) return fail(PREFIXLM_ERR_INVALID, "head_dim must be 64 or 128 (got %d)", D);
  if (T < 1 || H < 1) return fail(PREFIXLM_ERR_INVALID, "num_tokens=%d num_heads=%d must be >= 1", T, H);
  if (total < 0 || total > T)
    return fail(PREFIXLM_ERR_INVALID, "total_seqlen=%d outside [0, num_tokens=%d]", total, T);
  if (numseqs < 0) return fail(PREFIXLM_ERR_INVALID, "numseqs=%d < 0", numseqs);
  if (numseqs > 0 && (int64_t)numseqs + 1 > meta_len)
    return fail(PREFIXLM_ERR_INVALID, "numseqs=%d needs %d cu_seqlens entries, arrays hold %lld",
                numseqs, numseqs + 1, (long long)meta_len);
  if (numseqs > 0 && (!pre || !cau || !cu))
    return fail(PREFIXLM_ERR_INVALID, "metadata pointers must be non-null");
  if (max_all < 0 || max_all > total)
    return fail(PREFIXLM_ERR_INVALID, "max_seqlen_all=%d outside [0, total_seqlen=%d]", max_all, total);
  for (int i = 0; i < nptr; ++i) {
    if (!ptrs[i]) return fail(PREFIXLM_ERR_INVALID, "tensor pointer %d is null", i);
    if (!aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "tensor pointer %d is not 16-byte aligned", i);
  }
  for (int i = 0; i < nstr; ++i) {
    const int64_t st = strides[2 * i], sh = strides[2 * i + 1];
    if (st < D || sh < 0 || (st % 8) != 0 || (sh % 8) != 0)
      return fail(PREFIXLM_ERR_INVALID,
                  "tensor %d strides (token %lld, head %lld) must be multiples of 8 with token "
                  "stride >= head_dim and head stride >= 0",
                  i, (long long)st, (long long)sh);
    if (!segment_fits(max_all, st))
      return fail(PREFIXLM_ERR_INVALID, "segment of %d rows x token stride %lld exceeds 2 GiB",
                  max_all, (long long)st);
  }
  return PREFIXLM_OK;
}

}  // namespace

// ---- scratch of the zero-allocation backward ------------------------------------
// Device memory of prefixlm_bwd_noalloc: a file-scope array each GPU holds (at its own
// address) from the library's load until the process ends. Its host-side name is not a
// device address: kernels only ever receive the address hipGetSymbolAddress returns,
// fetched once per device with that device current.
constexpr size_t kNoallocScratchBytes = (size_t)16 << 20;
static __device__ __align__(256) unsigned char scratch[kNoallocScratchBytes];

namespace {
constexpr int kMaxDevices = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[kMaxDevices] = {};

// Address of this device's scratch array (the current device's).
int scratch_for_current_device(void** out) {
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
  if (dev < 0 || dev >= kMaxDevices) return fail(PREFIXLM_ERR_INVALID, "device %d >= %d", dev, kMaxDevices);
  std::lock_guard<std::mutex> g(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p)
      return fail(PREFIXLM_ERR_HIP, "hipGetSymbolAddress(scratch) on device %d: %s", dev, hipGetErrorString(e));
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return PREFIXLM_OK;
}
}  // namespace

extern "C" {

int32_t prefixlm_version(void) { return PREFIXLM_VERSION; }

const char* prefixlm_last_error(void) { return g_err; }

size_t prefixlm_fwd_workspace_size(int32_t num_tokens, int32_t num_heads, int32_t head_dim,
                                   int32_t total_seqlen, int32_t numseqs) {
  // the work list (either head dim runs its own kernel)
  (void)num_tokens;
  (void)num_heads;
  (void)head_dim;
  return align_up(sizeof(WsHeader)) + align_up(sizeof(int2) * (size_t)max_items(total_seqlen, numseqs, fwd::BM));
}

size_t prefixlm_fwd_q_amax_count(int32_t num_tokens, int32_t num_heads) {
  // a slot per wave of the forward grid, for any numseqs <= num_tokens
  if (num_tokens < 0 || num_heads < 1) return 0;
  return (size_t)(fwd::NT / 64) * unit_grid(max_items(num_tokens, num_tokens, fwd::BM), num_heads);
}

size_t prefixlm_bwd_workspace_size(int32_t num_tokens, int32_t num_heads, int32_t head_dim,
                                   int32_t total_seqlen, int32_t numseqs) {
  // the same for either head dim: work lists (the dK/dV list's header, which carries the
  // error word, first), stored-dS bases, statistics, counters and delta
  (void)head_dim;
  return align_up(sizeof(WsHeader)) +                                                   // dK/dV list
         align_up(sizeof(int2) * (size_t)max_items(total_seqlen, numseqs, bwd::kv::BK)) +
         align_up(sizeof(WsHeader)) +                                                   // dQ list
         align_up(sizeof(int2) * (size_t)max_items(total_seqlen, numseqs, bwd::qk::BQ)) +
         align_up(sizeof(int32_t) * ((size_t)numseqs + 1)) +                            // dS bases
         align_up(sizeof(float) * ((size_t)num_heads * bwd::kStats +                    // statistics
                                   (size_t)numseqs * num_heads * bwd::kSegStats + bwd::kCounters)) +
         align_up(sizeof(float) * (size_t)num_heads * num_tokens);                      // delta
}

size_t prefixlm_bwd_ds_bytes_blocks(int32_t num_tokens, int32_t num_heads, int32_t numseqs, int64_t ds_blocks) {
  if (num_tokens < 1 || num_heads < 1 || numseqs < 0 || ds_blocks < 1) return 0;
  const int64_t hb = ds_blocks * 4096;
  if (hb >= ((int64_t)1 << 31)) return 0;   // one head's blocks must fit 32-bit offsets
  return align_up((size_t)hb * num_heads) + align_up(sizeof(float) * (size_t)num_heads * ds_nkslot(num_tokens, numseqs));
}

size_t prefixlm_bwd_ds_bytes(int32_t num_tokens, int32_t num_heads, int32_t numseqs, int32_t max_seqlen_all) {
  if (max_seqlen_all < 1 || max_seqlen_all > 128 * bwd::q2::MAX_KT) return 0;   // the dQ kernel holds a segment's tile scales in LDS
  return prefixlm_bwd_ds_bytes_blocks(num_tokens, num_heads, numseqs, ds_bound_blocks(num_tokens, numseqs, max_seqlen_all));
}

}  // extern "C"

template <int HD>
static int fwd_launch(const prefixlm_fwd_args* a, void* stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (a->struct_size != sizeof(prefixlm_fwd_args))
    return fail(PREFIXLM_ERR_INVALID, "prefixlm_fwd_args.struct_size is %u, this library's is %zu: the caller was "
                "built against another version of prefixlm.h", a->struct_size, sizeof(prefixlm_fwd_args));
  const int has_lo = a->out_lo != nullptr;
  const bool use_plan = a->plan != nullptr;
  const bool gated = a->gate != nullptr;
  if (gated && !has_lo) return fail(PREFIXLM_ERR_INVALID, "a gated forward needs out_lo");
  if (gated && HD != 128) return fail(PREFIXLM_ERR_INVALID, "the output gate needs head_dim 128");
  // with a plan the forward needs no workspace
  const void* ptrs[] = {a->q,       a->k,    a->v, a->out, a->lse, use_plan ? a->q : a->workspace,
                        a->out_lo,  a->gate, a->out_gated};
  const int64_t strides[] = {a->q_stride_t,       a->q_stride_h,       a->k_stride_t,        a->k_stride_h,
                             a->v_stride_t,       a->v_stride_h,       a->out_stride_t,      a->out_stride_h,
                             a->out_lo_stride_t,  a->out_lo_stride_h,  a->gate_stride_t,     a->gate_stride_h,
                             a->out_gated_stride_t, a->out_gated_stride_h};
  int rc = check_common(ptrs, 6 + has_lo + 2 * gated, strides, 4 + has_lo + 2 * gated, a->num_tokens,
                        a->num_heads, a->head_dim, a->total_seqlen, a->numseqs, a->max_seqlen_all, a->meta_len,
                        a->prefix_lens, a->causal_lens, a->cu_seqlens);
  if (rc) return rc;
  // out_lo rows (int8, head_dim bytes) leave the kernel as 16-byte chunks
  if (has_lo && ((a->out_lo_stride_t % 16) != 0 || (a->out_lo_stride_h % 16) != 0))
    return fail(PREFIXLM_ERR_INVALID, "out_lo strides (token %lld, head %lld) must be multiples of 16",
                (long long)a->out_lo_stride_t, (long long)a->out_lo_stride_h);
  plan::Layout pl{};
  if (use_plan) {
    rc = check_plan(a->plan, a->plan_bytes, a->total_seqlen, a->numseqs, &pl);
    if (rc) return rc;
  } else {
    const size_t need = prefixlm_fwd_workspace_size(a->num_tokens, a->num_heads, HD, a->total_seqlen, a->numseqs);
    if (a->workspace_bytes < need)
      return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes, %zu needed", a->workspace_bytes, need);
  }
  if (a->q_amax != nullptr && a->numseqs > a->num_tokens)
    return fail(PREFIXLM_ERR_INVALID, "q_amax holds prefixlm_fwd_q_amax_count(num_tokens, num_heads) slots, "
                "which assumes numseqs <= num_tokens (got numseqs=%d, num_tokens=%d)", a->numseqs, a->num_tokens);
  set_kernel_attrs();
  if (g_attr_err != hipSuccess)
    return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(g_attr_err));

  const char* lists = use_plan ? static_cast<const char*>(a->plan) : static_cast<const char*>(a->workspace);
  WsHeader* hdr = reinterpret_cast<WsHeader*>(const_cast<char*>(lists) + (use_plan ? pl.hdr_off[0] : 0));
  int2* items = reinterpret_cast<int2*>(const_cast<char*>(lists) +
                                        (use_plan ? pl.items_off[0] : align_up(sizeof(WsHeader))));
  const int64_t nmax = max_items(a->total_seqlen, a->numseqs, fwd::BM);
  const int T = a->num_tokens, H = a->num_heads;

  (void)hipGetLastError();
  const int64_t nblk = unit_grid(nmax, H);
  bool self = false;
  if (!use_plan) {
    rc = fwd_finds_items(nblk, a->numseqs, a->max_seqlen_all, &self);
    if (rc) return rc;
  }
  if (!use_plan && !self) {
    // one of the two always runs, so the workspace header (item count, error word) is fresh
    MetaParams m{a->prefix_lens, a->causal_lens, a->cu_seqlens, a->numseqs, a->total_seqlen, T,
                 a->is_causal ? 1 : 0, a->max_seqlen_all};
    KernelTimer tm(a->timer, 0, stream);
    ListSpecs specs{};
    specs.l[0] = ListSpec{0, fwd::BM, fwd::BN, (int)nmax, items, hdr, nullptr, 0};
    hipLaunchKernelGGL(build_worklist_kernel, dim3(1), dim3(kPrepThreads), 0, stream, m, specs,
                       (float*)nullptr, 0);
  }
  if (nmax > 0 || a->total_seqlen < T) {
    fwd::Params P{};
    P.q = static_cast<const bf16*>(a->q);
    P.k = static_cast<const bf16*>(a->k);
    P.v = static_cast<const bf16*>(a->v);
    P.o = static_cast<bf16*>(a->out);
    P.o_lo = static_cast<int8_t*>(a->out_lo);
    P.lse = a->lse;
    P.gate = static_cast<const bf16*>(a->gate);
    P.y = gated ? static_cast<bf16*>(a->out_gated) : nullptr;   // ignored without a gate
    P.q_st = a->q_stride_t; P.q_sh = a->q_stride_h;
    P.k_st = a->k_stride_t; P.k_sh = a->k_stride_h;
    P.v_st = a->v_stride_t; P.v_sh = a->v_stride_h;
    P.o_st = a->out_stride_t; P.o_sh = a->out_stride_h;
    P.lo_st = a->out_lo_stride_t; P.lo_sh = a->out_lo_stride_h;
    P.g_st = a->gate_stride_t; P.g_sh = a->gate_stride_h;
    P.y_st = a->out_gated_stride_t; P.y_sh = a->out_gated_stride_h;
    P.prefix = a->prefix_lens;
    P.causal = a->causal_lens;
    P.cu = a->cu_seqlens;
    P.items = self ? nullptr : items;
    P.hdr = hdr;
    P.q_amax = a->q_amax;
    P.max_items = (int)nmax;
    P.max_all = a->max_seqlen_all;
    P.T = T;
    P.H = H;
    P.is_causal = a->is_causal ? 1 : 0;
    P.numseqs = a->numseqs;
    P.scale_log2 = a->softmax_scale * kLog2e;
    bool split = false;
    rc = fwd_splits_keys(nblk, a->max_seqlen_all, &split);
    if (rc) return rc;
    const int nt = fwd::NT * (split ? 2 : 1), groups = nt / (HD / 8);   // padding (row, head) pairs per workgroup
    const int64_t npad = ((int64_t)(T - a->total_seqlen) * H + groups - 1) / groups;
    if (nblk + npad > 0x7fffffff)
      return fail(PREFIXLM_ERR_INVALID, "grid of %lld blocks too large", (long long)(nblk + npad));
    P.n_main = (int)nblk;
    P.total = a->total_seqlen;
    {
      KernelTimer tm(a->timer, 1, stream);
      if (split)
        hipLaunchKernelGGL((fwd::prefixlm_fwd_kernel<HD, false, 2>), dim3((unsigned)(nblk + npad)), dim3(nt),
                           2 * fwd::Geo<HD>::LDS_BYTES, stream, P);
      else
        hipLaunchKernelGGL(fwd::prefixlm_fwd_kernel<HD>, dim3((unsigned)(nblk + npad)), dim3(nt),
                           fwd::Geo<HD>::LDS_BYTES, stream, P);
    }
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "forward launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

template <int HD>
static int bwd_launch(const prefixlm_bwd_args* a, void* stream_) {
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (a->struct_size != sizeof(prefixlm_bwd_args))
    return fail(PREFIXLM_ERR_INVALID, "prefixlm_bwd_args.struct_size is %u, this library's is %zu: the caller was "
                "built against another version of prefixlm.h", a->struct_size, sizeof(prefixlm_bwd_args));
  const void* ptrs[] = {a->q,  a->k,  a->v,  a->out,       a->dout, a->lse,
                        a->dq, a->dk, a->dv, a->workspace, a->out_lo};
  const int64_t strides[] = {a->q_stride_t,    a->q_stride_h,    a->k_stride_t,    a->k_stride_h,
                             a->v_stride_t,    a->v_stride_h,    a->out_stride_t,  a->out_stride_h,
                             a->dout_stride_t, a->dout_stride_h, a->dq_stride_t,   a->dq_stride_h,
                             a->dk_stride_t,   a->dk_stride_h,   a->dv_stride_t,   a->dv_stride_h,
                             a->out_lo_stride_t, a->out_lo_stride_h};
  const int has_lo = a->out_lo != nullptr;
  int rc = check_common(ptrs, 10 + has_lo, strides, 8 + has_lo, a->num_tokens, a->num_heads, a->head_dim,
                        a->total_seqlen, a->numseqs, a->max_seqlen_all, a->meta_len,
                        a->prefix_lens, a->causal_lens, a->cu_seqlens);
  if (rc) return rc;
  const bool gated = a->gate != nullptr;
  if (gated && HD != 128) return fail(PREFIXLM_ERR_INVALID, "the output gate needs head_dim 128");
  if (gated) {
    const void* gp[] = {a->gate, a->dgate, a->dout_attn};
    const int64_t gs[] = {a->gate_stride_t,  a->gate_stride_h,      a->dgate_stride_t,
                          a->dgate_stride_h, a->dout_attn_stride_t, a->dout_attn_stride_h};
    rc = check_common(gp, 3, gs, 3, a->num_tokens, a->num_heads, a->head_dim, a->total_seqlen, a->numseqs,
                      a->max_seqlen_all, a->meta_len, a->prefix_lens, a->causal_lens, a->cu_seqlens);
    if (rc) return rc;
  }
  const bool use_plan = a->plan != nullptr;
  plan::Layout pl{};
  if (use_plan) {
    rc = check_plan(a->plan, a->plan_bytes, a->total_seqlen, a->numseqs, &pl);
    if (rc) return rc;
  }
  const size_t need =
      prefixlm_bwd_workspace_size(a->num_tokens, a->num_heads, HD, a->total_seqlen, a->numseqs);
  if (a->workspace_bytes < need)
    return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes, %zu needed", a->workspace_bytes, need);
  // dQ from the stored dS when the caller gave a buffer and the layout fits: a->ds_blocks
  // blocks per head, or the bound the scalars give
  if (a->ds_blocks < 0) return fail(PREFIXLM_ERR_INVALID, "ds_blocks=%lld < 0", (long long)a->ds_blocks);
  const int64_t ds_cap =
      a->ds_blocks > 0 ? a->ds_blocks : ds_bound_blocks(a->num_tokens, a->numseqs, a->max_seqlen_all);
  const size_t ds_need = a->max_seqlen_all > 128 * bwd::q2::MAX_KT
                             ? 0
                             : prefixlm_bwd_ds_bytes_blocks(a->num_tokens, a->num_heads, a->numseqs, ds_cap);
  const bool use_ds = a->ds_buf != nullptr && ds_need > 0;
  if (use_ds) {
    if (a->ds_buf_bytes < ds_need)
      return fail(PREFIXLM_ERR_INVALID, "ds_buf of %zu bytes, %zu needed", a->ds_buf_bytes, ds_need);
    if ((reinterpret_cast<uintptr_t>(a->ds_buf) & 255u) != 0)
      return fail(PREFIXLM_ERR_INVALID, "ds_buf must be 256-byte aligned");
  }
  if (a->num_heads > bwd::kPreMaxHeads)
    return fail(PREFIXLM_ERR_INVALID, "num_heads=%d exceeds %d", a->num_heads, bwd::kPreMaxHeads);
  if (a->q_amax == nullptr)
    return fail(PREFIXLM_ERR_INVALID, "q_amax is null: the backward needs the forward's per-workgroup max |Q| "
                "(prefixlm_fwd_args.q_amax)");
  {
    // the pre-pass addresses kPreRows rows x all heads of out, out_lo and dout with
    // 32-bit byte offsets
    const int64_t st[6] = {a->out_stride_t, a->out_lo_stride_t, a->dout_stride_t,
                           a->gate_stride_t, a->dgate_stride_t, a->dout_attn_stride_t};
    const int64_t sh[6] = {a->out_stride_h, a->out_lo_stride_h, a->dout_stride_h,
                           a->gate_stride_h, a->dgate_stride_h, a->dout_attn_stride_h};
    for (int i = 0; i < 6; ++i) {
      if ((i == 1 && !has_lo) || (i >= 3 && !gated)) continue;
      if (((int64_t)bwd::kPreRows * st[i] + (int64_t)(a->num_heads - 1) * sh[i] + a->head_dim) * 2 >=
          (int64_t)1 << 31)
        return fail(PREFIXLM_ERR_INVALID, "tensor %d spans more than 2 GiB over %d rows", i, bwd::kPreRows);
    }
  }
  set_kernel_attrs();
  if (g_attr_err != hipSuccess)
    return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(g_attr_err));

  const int T = a->num_tokens, H = a->num_heads;
  const int64_t nkv = max_items(a->total_seqlen, a->numseqs, bwd::kv::BK);
  const int64_t nq = max_items(a->total_seqlen, a->numseqs, bwd::qk::BQ);
  if (unit_grid(nkv, H) > 0x7fffffff || unit_grid(nq, H) > 0x7fffffff)
    return fail(PREFIXLM_ERR_INVALID, "grid of %lld blocks too large", (long long)unit_grid(nq, H));
  char* ws = static_cast<char*>(a->workspace);
  size_t off = 0;
  WsHeader* hdr_kv = reinterpret_cast<WsHeader*>(ws + off);
  off += align_up(sizeof(WsHeader));
  int2* items_kv = reinterpret_cast<int2*>(ws + off);
  off += align_up(sizeof(int2) * (size_t)nkv);
  WsHeader* hdr_q = reinterpret_cast<WsHeader*>(ws + off);
  off += align_up(sizeof(WsHeader));
  int2* items_q = reinterpret_cast<int2*>(ws + off);
  off += align_up(sizeof(int2) * (size_t)nq);
  int32_t* ds_base = reinterpret_cast<int32_t*>(ws + off);
  off += align_up(sizeof(int32_t) * ((size_t)a->numseqs + 1));
  float* stats = reinterpret_cast<float*>(ws + off);
  float* segstats = stats + (size_t)H * bwd::kStats;
  // statistics, then the work-item counters of the persistent kernels (all zeroed below)
  const size_t n_stats = (size_t)H * bwd::kStats + (size_t)a->numseqs * H * bwd::kSegStats + bwd::kCounters;
  int* counters = reinterpret_cast<int*>(segstats + (size_t)a->numseqs * H * bwd::kSegStats);
  off += align_up(sizeof(float) * n_stats);
  float* delta = reinterpret_cast<float*>(ws + off);
  if (n_stats > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "too many segments");
  if (use_plan) {
    char* pb = static_cast<char*>(const_cast<void*>(a->plan));
    hdr_kv = reinterpret_cast<WsHeader*>(pb + pl.hdr_off[1]);
    items_kv = reinterpret_cast<int2*>(pb + pl.items_off[1]);
    hdr_q = reinterpret_cast<WsHeader*>(pb + pl.hdr_off[2]);
    items_q = reinterpret_cast<int2*>(pb + pl.items_off[2]);
    ds_base = reinterpret_cast<int32_t*>(pb + pl.ds_off);
  }

  (void)hipGetLastError();
  // the forward's max |Q| slots (its grid: one per workgroup), reduced per head by the
  // pre-pass into statistics slot 3, for the dK/dV kernel's fp16 scale of Q
  const int q_slots = (fwd::NT / 64) * (int)unit_grid(max_items(a->total_seqlen, a->numseqs, fwd::BM), H);
  if (use_plan) {
    // the work-list kernel is skipped; clear the statistics it would have cleared
    KernelTimer tm(a->timer, 3, stream);
    const int nb = (int)std::min<size_t>((n_stats + 255) / 256, 1024);
    if (nb > 0)
      hipLaunchKernelGGL(bwd::zero_floats_kernel, dim3(nb), dim3(256), 0, stream, stats, (int)n_stats);
  } else {
    // both work lists; also zeroes the statistics the next kernels accumulate
    MetaParams m{a->prefix_lens, a->causal_lens, a->cu_seqlens, a->numseqs, a->total_seqlen, T,
                 a->is_causal ? 1 : 0, a->max_seqlen_all};
    ListSpecs specs{};
    specs.l[0] = ListSpec{1, bwd::kv::BK, bwd::kv::BQ, (int)nkv, items_kv, hdr_kv, use_ds ? ds_base : nullptr,
                          (int)std::min<int64_t>(ds_cap, 0x7fffffff)};
    specs.l[1] = ListSpec{0, bwd::qk::BQ, bwd::qk::BKT, (int)nq, items_q, hdr_q, nullptr, 0};
    KernelTimer tm(a->timer, 3, stream);
    hipLaunchKernelGGL(build_worklist_kernel, dim3(2), dim3(kPrepThreads), 0, stream, m, specs, stats,
                       (int)n_stats);
  }
  // the dK/dV and dQ kernels read dO: the caller's dout, or with a gate the
  // pre-pass's dout * sigmoid(gate)
  const bf16* dO = static_cast<const bf16*>(gated ? a->dout_attn : a->dout);
  const int64_t dO_st = gated ? a->dout_attn_stride_t : a->dout_stride_t;
  const int64_t dO_sh = gated ? a->dout_attn_stride_h : a->dout_stride_h;
  {
    KernelTimer tm(a->timer, 4, stream);
    bwd::GateBwd G{static_cast<const bf16*>(a->gate), static_cast<bf16*>(a->dgate), static_cast<bf16*>(a->dout_attn),
                   a->gate_stride_t, a->gate_stride_h, a->dgate_stride_t, a->dgate_stride_h,
                   a->dout_attn_stride_t, a->dout_attn_stride_h};
    const bwd::PadBwd pad{static_cast<bf16*>(a->dq), static_cast<bf16*>(a->dk), static_cast<bf16*>(a->dv),
                          a->dq_stride_t, a->dq_stride_h, a->dk_stride_t, a->dk_stride_h, a->dv_stride_t, a->dv_stride_h};
    int cus = 0;
    rc = persistent_grid(&cus);
    if (rc) return rc;
    // 32 rows per workgroup, or as few (8 at least) as still give every CU one (700 rows x 8
    // heads x d64: 8.8 us with 32, 5.6 with 8)
    const int rows = std::min(bwd::kPreRows, std::max(8, (T + cus - 1) / cus));
    const dim3 grid((T + rows - 1) / rows);
    if constexpr (HD == 128) {
      if (gated)
        hipLaunchKernelGGL((bwd::prefixlm_bwd_pre_kernel<128, true>), grid, dim3(256), 0, stream,
                           static_cast<const bf16*>(a->out), static_cast<const int8_t*>(a->out_lo),
                           static_cast<const bf16*>(a->dout), a->out_stride_t, a->out_stride_h,
                           a->out_lo_stride_t, a->out_lo_stride_h, a->dout_stride_t, a->dout_stride_h, delta,
                           stats, T, H, a->total_seqlen, G, a->q_amax, q_slots, pad, rows);
    }
    if (!gated)
      hipLaunchKernelGGL((bwd::prefixlm_bwd_pre_kernel<HD, false>), grid, dim3(256), 0, stream,
                         static_cast<const bf16*>(a->out), static_cast<const int8_t*>(a->out_lo),
                         static_cast<const bf16*>(a->dout), a->out_stride_t, a->out_stride_h, a->out_lo_stride_t,
                         a->out_lo_stride_h, a->dout_stride_t, a->dout_stride_h, delta, stats, T, H,
                         a->total_seqlen, G, a->q_amax, q_slots, pad, rows);
  }
  const float scale_log2 = a->softmax_scale * kLog2e;
  if (nkv > 0) {
    bwd::KvParams P;
    P.q = static_cast<const bf16*>(a->q);
    P.k = static_cast<const bf16*>(a->k);
    P.v = static_cast<const bf16*>(a->v);
    P.dout = dO;
    P.lse = a->lse;
    P.delta = delta;
    P.stats = stats;
    P.segstats = segstats;
    P.counters = counters;
    P.ds = nullptr;
    P.ds_scale = nullptr;
    P.ds_base = nullptr;
    P.ds_hbytes = 0;
    P.ds_nkslot = 0;
    if (use_ds) {
      const int64_t hb = ds_cap * 4096;
      P.ds = static_cast<char*>(a->ds_buf);
      P.ds_scale = reinterpret_cast<float*>(P.ds + align_up((size_t)hb * H));
      P.ds_base = ds_base;
      P.ds_hbytes = (uint32_t)hb;
      P.ds_nkslot = (int)ds_nkslot(T, a->numseqs);
    }
    P.dk = static_cast<bf16*>(a->dk);
    P.dv = static_cast<bf16*>(a->dv);
    P.q_st = a->q_stride_t; P.q_sh = a->q_stride_h;
    P.k_st = a->k_stride_t; P.k_sh = a->k_stride_h;
    P.v_st = a->v_stride_t; P.v_sh = a->v_stride_h;
    P.do_st = dO_st; P.do_sh = dO_sh;
    P.dk_st = a->dk_stride_t; P.dk_sh = a->dk_stride_h;
    P.dv_st = a->dv_stride_t; P.dv_sh = a->dv_stride_h;
    P.prefix = a->prefix_lens;
    P.causal = a->causal_lens;
    P.cu = a->cu_seqlens;
    P.items = items_kv;
    P.hdr = hdr_kv;
    P.T = T;
    P.H = H;
    P.is_causal = a->is_causal ? 1 : 0;
    P.numseqs = a->numseqs;
    P.scale_log2 = scale_log2;
    P.scale = a->softmax_scale;
    // persistent: one workgroup per CU (a multiple of 8, see the kernel), fewer when the
    // list is shorter
    int grid = 0;
    rc = persistent_grid(&grid);
    if (rc) return rc;
    const int64_t nblk = std::min<int64_t>(unit_grid(nkv, H), grid);
    KernelTimer tm(a->timer, 5, stream);
    hipLaunchKernelGGL(bwd::prefixlm_bwd_dkdv_kernel<HD>, dim3((unsigned)nblk), dim3(bwd::kv::NT),
                       bwd::kv::Geo<HD>::LDS_BYTES, stream, P);
  }
  if (nq > 0 && use_ds) {
    // dQ = scale dS K from the blocks the dK/dV kernel stored, with its max |K| per
    // (segment, head)
    const int64_t hb = ds_cap * 4096;
    bwd::Q2Params P;
    P.k = static_cast<const bf16*>(a->k);
    P.segstats = segstats;
    P.ds = static_cast<const char*>(a->ds_buf);
    P.ds_scale = reinterpret_cast<const float*>(P.ds + align_up((size_t)hb * H));
    P.ds_base = ds_base;
    P.dq = static_cast<bf16*>(a->dq);
    P.k_st = a->k_stride_t; P.k_sh = a->k_stride_h;
    P.dq_st = a->dq_stride_t; P.dq_sh = a->dq_stride_h;
    P.prefix = a->prefix_lens;
    P.causal = a->causal_lens;
    P.cu = a->cu_seqlens;
    P.items = items_q;
    P.hdr = hdr_q;
    P.T = T;
    P.H = H;
    P.is_causal = a->is_causal ? 1 : 0;
    P.numseqs = a->numseqs;
    P.ds_hbytes = (uint32_t)hb;
    P.ds_nkslot = (int)ds_nkslot(T, a->numseqs);
    P.scale = a->softmax_scale;
    KernelTimer tm(a->timer, 7, stream);
    hipLaunchKernelGGL(bwd::prefixlm_bwd_dq_ds_kernel<HD>, dim3((unsigned)unit_grid(nq, H)), dim3(bwd::q2::NT),
                       bwd::q2::Geo<HD>::LDS_BYTES, stream, P);
  } else if (nq > 0) {
    // reads the per-(segment, head) maxima of |K| and ||V|| the dK/dV kernel wrote
    bwd::QParams P;
    P.q = static_cast<const bf16*>(a->q);
    P.k = static_cast<const bf16*>(a->k);
    P.v = static_cast<const bf16*>(a->v);
    P.dout = dO;
    P.lse = a->lse;
    P.delta = delta;
    P.segstats = segstats;
    P.dq = static_cast<bf16*>(a->dq);
    P.q_st = a->q_stride_t; P.q_sh = a->q_stride_h;
    P.k_st = a->k_stride_t; P.k_sh = a->k_stride_h;
    P.v_st = a->v_stride_t; P.v_sh = a->v_stride_h;
    P.do_st = dO_st; P.do_sh = dO_sh;
    P.dq_st = a->dq_stride_t; P.dq_sh = a->dq_stride_h;
    P.prefix = a->prefix_lens;
    P.causal = a->causal_lens;
    P.cu = a->cu_seqlens;
    P.items = items_q;
    P.hdr = hdr_q;
    P.T = T;
    P.H = H;
    P.is_causal = a->is_causal ? 1 : 0;
    P.numseqs = a->numseqs;
    P.scale_log2 = scale_log2;
    P.scale = a->softmax_scale;
    KernelTimer tm(a->timer, 7, stream);
    hipLaunchKernelGGL(bwd::prefixlm_bwd_dq_kernel<HD>, dim3((unsigned)unit_grid(nq, H)), dim3(bwd::qk::NT),
                       bwd::qk::Geo<HD>::LDS_BYTES, stream, P);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "backward launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

extern "C" {

int prefixlm_fwd(const prefixlm_fwd_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  // each head dim runs its own instantiation of the forward kernel
  return a->head_dim == 64 ? fwd_launch<64>(a, stream_) : fwd_launch<128>(a, stream_);
}

int prefixlm_bwd(const prefixlm_bwd_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  // each head dim runs its own instantiation of the backward kernels
  return a->head_dim == 64 ? bwd_launch<64>(a, stream_) : bwd_launch<128>(a, stream_);
}

size_t prefixlm_bwd_noalloc_max_scratch(void) { return kNoallocScratchBytes; }

int prefixlm_bwd_noalloc(const prefixlm_bwd_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  if (a->workspace || a->workspace_bytes)
    return fail(PREFIXLM_ERR_INVALID, "prefixlm_bwd_noalloc uses the library's scratch: workspace must be NULL/0");
  if (a->timer)
    return fail(PREFIXLM_ERR_INVALID, "prefixlm_bwd_noalloc takes no timer (its events would be allocated)");
  const size_t need =
      prefixlm_bwd_workspace_size(a->num_tokens, a->num_heads, a->head_dim, a->total_seqlen, a->numseqs);
  if (need > kNoallocScratchBytes)
    return fail(PREFIXLM_ERR_INVALID,
                "prefixlm_bwd_noalloc: this call needs %zu bytes of scratch, the library's scratch holds %zu "
                "(num_tokens=%d num_heads=%d head_dim=%d numseqs=%d); use prefixlm_bwd with a workspace",
                need, kNoallocScratchBytes, a->num_tokens, a->num_heads, a->head_dim, a->numseqs);
  void* ws = nullptr;
  const int rc = scratch_for_current_device(&ws);
  if (rc) return rc;
  prefixlm_bwd_args b = *a;
  b.workspace = ws;
  b.workspace_bytes = kNoallocScratchBytes;
  return prefixlm_bwd(&b, stream_);
}

int prefixlm_check_workspace(const void* workspace, void* stream_, int32_t* error_word) {
  if (!workspace) return fail(PREFIXLM_ERR_INVALID, "workspace is null");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  WsHeader h;
  hipError_t e = hipMemcpyAsync(&h, workspace, sizeof(h), hipMemcpyDeviceToHost, stream);
  if (e == hipSuccess) e = hipStreamSynchronize(stream);
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "reading workspace header: %s", hipGetErrorString(e));
  if (error_word) *error_word = h.error;
  if (h.error != 0)
    return fail(PREFIXLM_ERR_METADATA,
                "inconsistent metadata (flags 0x%x): segments must satisfy cu_seqlens[0]=0, "
                "cu_seqlens[s+1]=cu_seqlens[s]+prefix_lens[s]+causal_lens[s] <= total_seqlen",
                h.error);
  return PREFIXLM_OK;
}

int prefixlm_rope(const prefixlm_rope_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (a->head_dim != rope::D) return fail(PREFIXLM_ERR_INVALID, "head_dim must be 128 (got %d)", a->head_dim);
  if (a->num_tokens < 0 || a->num_heads < 1)
    return fail(PREFIXLM_ERR_INVALID, "num_tokens=%d num_heads=%d", a->num_tokens, a->num_heads);
  const void* ptrs[] = {a->x, a->y, a->cos, a->sin};
  for (int i = 0; i < 4; ++i)
    if (!ptrs[i] || !aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "pointer %d is null or not 16-byte aligned", i);
  const int64_t st[] = {a->x_stride_t, a->x_stride_h, a->y_stride_t, a->y_stride_h};
  for (int i = 0; i < 2; ++i)
    if (st[2 * i] < rope::D || st[2 * i + 1] < 0 || st[2 * i] % 8 || st[2 * i + 1] % 8)
      return fail(PREFIXLM_ERR_INVALID, "tensor %d strides (token %lld, head %lld) must be multiples of 8 "
                  "with token stride >= head_dim", i, (long long)st[2 * i], (long long)st[2 * i + 1]);
  if (a->cs_stride_t < rope::D || a->cs_stride_t % 4)
    return fail(PREFIXLM_ERR_INVALID, "cos/sin row stride %lld must be a multiple of 4 and >= head_dim",
                (long long)a->cs_stride_t);
  const int64_t threads = (int64_t)a->num_tokens * a->num_heads * 8;
  if (threads == 0) return PREFIXLM_OK;
  if ((threads + 255) / 256 > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "too many rows");
  rope::Params P{static_cast<const bf16*>(a->x), static_cast<bf16*>(a->y), a->cos, a->sin,
                 a->x_stride_t, a->x_stride_h, a->y_stride_t, a->y_stride_h, a->cs_stride_t,
                 a->num_tokens, a->num_heads, a->backward ? 1 : 0};
  (void)hipGetLastError();
  hipLaunchKernelGGL(rope::rope_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, P);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "rope launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

static int swiglu_launch(const prefixlm_swiglu_args* a, void* stream_, bool backward) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  if (a->rows < 0 || a->cols < 8 || a->cols % 8)
    return fail(PREFIXLM_ERR_INVALID, "rows=%lld cols=%lld: cols must be a positive multiple of 8",
                (long long)a->rows, (long long)a->cols);
  if (a->rows == 0) return PREFIXLM_OK;   // empty tensors may have null pointers
  const void* ptrs[] = {a->gu, backward ? a->dy : a->y, backward ? a->dgu : nullptr};
  for (int i = 0; i < (backward ? 3 : 2); ++i)
    if (!ptrs[i] || !aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "pointer %d is null or not 16-byte aligned", i);
  const int64_t st[] = {a->gu_stride, backward ? a->dy_stride : a->y_stride, a->dgu_stride};
  const int64_t need[] = {2 * a->cols, a->cols, 2 * a->cols};
  for (int i = 0; i < (backward ? 3 : 2); ++i)
    if (st[i] < need[i] || st[i] % 8)
      return fail(PREFIXLM_ERR_INVALID, "row stride %d (%lld) must be a multiple of 8 and >= %lld", i,
                  (long long)st[i], (long long)need[i]);
  const int64_t threads = a->rows * (a->cols / 8);
  if (threads == 0) return PREFIXLM_OK;
  if ((threads + 255) / 256 > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "too many elements");
  nm::SwigluParams P{static_cast<const bf16*>(a->gu), static_cast<const bf16*>(a->dy), static_cast<bf16*>(a->y),
                     static_cast<bf16*>(a->dgu), a->gu_stride, a->y_stride, a->dy_stride, a->dgu_stride,
                     a->rows, a->cols};
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  (void)hipGetLastError();
  const bool nt = a->rows * a->cols * (backward ? 10 : 6) > nm::kNtBytes;
  hipLaunchKernelGGL(backward ? (nt ? nm::swiglu_bwd_kernel<true> : nm::swiglu_bwd_kernel<false>)
                              : (nt ? nm::swiglu_fwd_kernel<true> : nm::swiglu_fwd_kernel<false>),
                     dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, P);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "swiglu launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

int prefixlm_swiglu_fwd(const prefixlm_swiglu_args* a, void* stream) { return swiglu_launch(a, stream, false); }
int prefixlm_swiglu_bwd(const prefixlm_swiglu_args* a, void* stream) { return swiglu_launch(a, stream, true); }

// The RMSNorm kernel for rows of `cols` elements: 16-byte chunks per lane, the smallest
// power of two with 64 * nch * 8 >= cols.
static void (*rmsnorm_kernel(int cols, bool backward))(nm::NormParams) {
  const int need = (cols / 8 + 63) / 64;
  int nch = 1;
  while (nch < need) nch *= 2;
  static_assert(nm::kNormMaxChunks == 16, "the dispatch covers up to 16 chunks per lane");
  switch (nch) {
    case 1: return backward ? nm::rmsnorm_bwd_kernel<1> : nm::rmsnorm_fwd_kernel<1>;
    case 2: return backward ? nm::rmsnorm_bwd_kernel<2> : nm::rmsnorm_fwd_kernel<2>;
    case 4: return backward ? nm::rmsnorm_bwd_kernel<4> : nm::rmsnorm_fwd_kernel<4>;
    case 8: return backward ? nm::rmsnorm_bwd_kernel<8> : nm::rmsnorm_fwd_kernel<8>;
    default: return backward ? nm::rmsnorm_bwd_kernel<16> : nm::rmsnorm_fwd_kernel<16>;
  }
}

static void (*add_rmsnorm_kernel(int cols))(nm::NormParams) {
  const int need = (cols / 8 + 63) / 64;
  return need <= 1   ? nm::rmsnorm_fwd_kernel<1, true>
         : need <= 2 ? nm::rmsnorm_fwd_kernel<2, true>
         : need <= 4 ? nm::rmsnorm_fwd_kernel<4, true>
         : need <= 8 ? nm::rmsnorm_fwd_kernel<8, true>
                     : nm::rmsnorm_fwd_kernel<16, true>;
}

static int rmsnorm_launch(const prefixlm_rmsnorm_args* a, void* stream_, bool backward) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  if (a->rows < 0 || a->cols < 8 || a->cols % 8 || a->cols > nm::kNormMaxCols)
    return fail(PREFIXLM_ERR_INVALID, "rows=%lld cols=%d: cols must be a multiple of 8 in [8, %d]",
                (long long)a->rows, a->cols, nm::kNormMaxCols);
  if (!backward && !(a->eps >= 0.f)) return fail(PREFIXLM_ERR_INVALID, "eps must be >= 0");
  if (a->rows == 0) return PREFIXLM_OK;   // empty tensors may have null pointers
  const void* ptrs[] = {a->x, backward ? a->dy : a->y, backward ? a->dx : nullptr};
  for (int i = 0; i < (backward ? 3 : 2); ++i)
    if (!ptrs[i] || !aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "pointer %d is null or not 16-byte aligned", i);
  if (!a->rstd) return fail(PREFIXLM_ERR_INVALID, "rstd is null");
  const int64_t st[] = {a->x_stride, backward ? a->dy_stride : a->y_stride, a->dx_stride};
  for (int i = 0; i < (backward ? 3 : 2); ++i)
    if (st[i] < a->cols || st[i] % 8)
      return fail(PREFIXLM_ERR_INVALID, "row stride %d (%lld) must be a multiple of 8 and >= cols", i,
                  (long long)st[i]);
  if ((a->rows + 3) / 4 > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "too many rows");
  nm::NormParams P{static_cast<const bf16*>(a->x), static_cast<const bf16*>(a->dy), static_cast<bf16*>(a->y),
                   static_cast<bf16*>(a->dx), a->rstd, a->x_stride, a->y_stride, a->dy_stride, a->dx_stride,
                   a->rows, a->cols, a->eps, nullptr, nullptr, 0, 0};
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  (void)hipGetLastError();
  hipLaunchKernelGGL(rmsnorm_kernel(a->cols, backward), dim3((unsigned)((a->rows + 3) / 4)), dim3(256), 0, stream, P);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "rmsnorm launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

int prefixlm_rmsnorm_fwd(const prefixlm_rmsnorm_args* a, void* stream) { return rmsnorm_launch(a, stream, false); }
int prefixlm_rmsnorm_bwd(const prefixlm_rmsnorm_args* a, void* stream) { return rmsnorm_launch(a, stream, true); }

int prefixlm_add_rmsnorm(const prefixlm_add_rmsnorm_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  if (a->rows < 0 || a->cols < 8 || a->cols % 8 || a->cols > nm::kNormMaxCols)
    return fail(PREFIXLM_ERR_INVALID, "rows=%lld cols=%d: cols must be a multiple of 8 in [8, %d]",
                (long long)a->rows, a->cols, nm::kNormMaxCols);
  if (!(a->eps >= 0.f)) return fail(PREFIXLM_ERR_INVALID, "eps must be >= 0");
  if (a->rows == 0) return PREFIXLM_OK;   // empty tensors may have null pointers
  const void* ptrs[] = {a->x, a->r, a->s, a->y};
  const int64_t st[] = {a->x_stride, a->r_stride, a->s_stride, a->y_stride};
  for (int i = 0; i < (a->y ? 4 : 3); ++i) {
    if (!ptrs[i] || !aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "pointer %d is null or not 16-byte aligned", i);
    if ((st[i] < a->cols && !(i < 2 && st[i] == 0)) || st[i] % 8)
      return fail(PREFIXLM_ERR_INVALID, "row stride %d (%lld) must be a multiple of 8 and >= cols", i, (long long)st[i]);
  }
  if (!a->rstd) return fail(PREFIXLM_ERR_INVALID, "rstd is null");
  if ((a->rows + 3) / 4 > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "too many rows");
  const nm::NormParams P{static_cast<const bf16*>(a->x), nullptr, static_cast<bf16*>(a->y), nullptr, a->rstd, a->x_stride,
                         a->y_stride, 0, 0, a->rows, a->cols, a->eps, static_cast<const bf16*>(a->r),
                         static_cast<bf16*>(a->s), a->r_stride, a->s_stride};
  (void)hipGetLastError();
  hipLaunchKernelGGL(add_rmsnorm_kernel(a->cols), dim3((unsigned)((a->rows + 3) / 4)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream_), P);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "add + rmsnorm launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

}  // extern "C"

// Projections of at most 128 rows: the kernel that streams W (see gemm.h).
template <int MB, int NWV>
static int proj_skinny_launch(const mlp::Params& P, bool sw, bool norm, float* rstd, float eps, hipStream_t stream) {
  using Kernel = void (*)(mlp::Params, float*, float);
  using G = mlp::SkinnyGeo<MB, NWV>;
  const Kernel kernels[4] = {mlp::proj_skinny_kernel<MB, NWV, false, false>, mlp::proj_skinny_kernel<MB, NWV, false, true>,
                             mlp::proj_skinny_kernel<MB, NWV, true, false>, mlp::proj_skinny_kernel<MB, NWV, true, true>};
  static std::once_flag once;
  static hipError_t attr_err = hipSuccess;
  std::call_once(once, [&kernels] {
    for (int i = 0; i < 4 && attr_err == hipSuccess; ++i)
      attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernels[i]), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     G::lds(i >= 2));
  });
  if (attr_err != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(attr_err));
  hipLaunchKernelGGL(kernels[2 * (sw ? 1 : 0) + (norm ? 1 : 0)], dim3((unsigned)((sw ? P.N / 2 : P.N) / 32)), dim3(64 * NWV),
                     G::lds(sw), stream, P, rstd, eps);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "projection launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}
static int proj_skinny(const prefixlm_proj_gemm_args* a, bool given, hipStream_t stream) {
  const mlp::Params P{static_cast<const bf16*>(a->x), static_cast<const bf16*>(a->w), static_cast<bf16*>(a->y),
                      given ? a->rstd : nullptr, a->x_stride, a->w_stride, a->y_stride, a->M, a->K, a->N, 0, 0};
  const bool sw = a->swiglu != 0, norm = a->norm != 0;
  float* const rstd = given ? nullptr : a->rstd;   // where the scales found from x go
  if (a->M <= 32) return proj_skinny_launch<1, 8>(P, sw, norm, rstd, a->eps, stream);
  if (a->M <= 64) return proj_skinny_launch<2, 8>(P, sw, norm, rstd, a->eps, stream);
  return proj_skinny_launch<4, 4>(P, sw, norm, rstd, a->eps, stream);
}

extern "C" {

// given: the row scales are in a->rstd already
static int proj_gemm_launch(const prefixlm_proj_gemm_args* a, void* stream_, bool given) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  const bool sw = a->swiglu != 0;
  if (a->M < 0 || a->K < mlp::KT || a->K % mlp::KT || a->N < mlp::WT || a->N % mlp::WT)
    return fail(PREFIXLM_ERR_INVALID, "M=%d K=%d N=%d: K must be a positive multiple of %d and N of %d", a->M, a->K,
                a->N, mlp::KT, mlp::WT);
  const int64_t nout = sw ? a->N / 2 : a->N;
  if (a->M == 0) return PREFIXLM_OK;
  const void* ptrs[] = {a->x, a->w, a->y};
  for (int i = 0; i < 3; ++i)
    if (!ptrs[i] || !aligned16(ptrs[i])) return fail(PREFIXLM_ERR_INVALID, "pointer %d is null or not 16-byte aligned", i);
  if (a->x_stride < a->K || a->x_stride % 8 || a->w_stride < a->K || a->w_stride % 8 || a->y_stride < nout ||
      a->y_stride % 8)
    return fail(PREFIXLM_ERR_INVALID, "strides (x %lld, w %lld, y %lld) must be multiples of 8 covering the rows",
                (long long)a->x_stride, (long long)a->w_stride, (long long)a->y_stride);
  if (!(a->eps >= 0.f)) return fail(PREFIXLM_ERR_INVALID, "eps must be >= 0");
  if (given && !a->norm) return fail(PREFIXLM_ERR_INVALID, "row scales without norm");
  if (a->norm) {
    if (!a->rstd) return fail(PREFIXLM_ERR_INVALID, "norm needs rstd (M floats)");
    if (a->K > nm::kNormMaxCols) return fail(PREFIXLM_ERR_INVALID, "norm: K=%d exceeds %d", a->K, nm::kNormMaxCols);
  }
  // 32-bit byte offsets: within a 256-row tile of x and y, and over all of W
  if ((int64_t)256 * a->x_stride * 2 >= ((int64_t)1 << 31) ||
      (int64_t)256 * a->y_stride * 2 >= ((int64_t)1 << 31) || (int64_t)a->N * a->w_stride * 2 >= ((int64_t)1 << 32))
    return fail(PREFIXLM_ERR_INVALID, "operands exceed the 32-bit offsets of the kernel");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  (void)hipGetLastError();
  if (a->M <= 128) return proj_skinny(a, given, stream);
  int cus = 0;
  const int rc = persistent_grid(&cus);
  if (rc) return rc;
  mlp::Params P{static_cast<const bf16*>(a->x), static_cast<const bf16*>(a->w), static_cast<bf16*>(a->y),
                a->rstd, a->x_stride, a->w_stride, a->y_stride, a->M, a->K, a->N, 0, 0};
  P.n_tiles = a->N / mlp::WT;
  // 256 x rows per tile, or 128 where that needs fewer or shorter rounds over the CUs: a round
  // of 128-row tiles takes 0.6 (many rounds) to 0.8 (one) of a round of 256-row ones, the W
  // tile's loads staying the same (K 2048, N 11264: M 512 37 us with 128 rows, 47 with 256;
  // M 700 67 and 49; M 1100 74 and 54; M 16384 748 and 614)
  const int64_t t256 = (int64_t)((a->M + 255) / 256) * P.n_tiles, t128 = (int64_t)((a->M + 127) / 128) * P.n_tiles;
  if (t128 > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "grid too large");
  const bool half = 7 * ((t128 + cus - 1) / cus) < 10 * ((t256 + cus - 1) / cus);
  P.m_tiles = (a->M + (half ? 127 : 255)) / (half ? 128 : 256);
  const int tiles = (int)(half ? t128 : t256);
  const unsigned grid = (unsigned)std::min(cus, (tiles + 7) / 8 * 8);
  static std::once_flag once;
  static hipError_t attr_err = hipSuccess;
  void (*const kernels[8])(mlp::Params) = {
      mlp::proj_gemm_kernel<256, false, false>, mlp::proj_gemm_kernel<256, false, true>,
      mlp::proj_gemm_kernel<256, true, false>,  mlp::proj_gemm_kernel<256, true, true>,
      mlp::proj_gemm_kernel<128, false, false>, mlp::proj_gemm_kernel<128, false, true>,
      mlp::proj_gemm_kernel<128, true, false>,  mlp::proj_gemm_kernel<128, true, true>};
  std::call_once(once, [&kernels] {
    for (int i = 0; i < 8 && attr_err == hipSuccess; ++i)
      attr_err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernels[i]), hipFuncAttributeMaxDynamicSharedMemorySize,
                                     i < 4 ? mlp::Geo<256>::LDS_BYTES : mlp::Geo<128>::LDS_BYTES);
  });
  if (attr_err != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(attr_err));
  if (a->norm && !given) {
    // the row scales first (a wave per row, x read once; the normalized x is not written)
    nm::NormParams N{static_cast<const bf16*>(a->x), nullptr, nullptr, nullptr, a->rstd, a->x_stride, 0, 0, 0,
                     a->M, a->K, a->eps, nullptr, nullptr, 0, 0};
    hipLaunchKernelGGL(rmsnorm_kernel(a->K, false), dim3((unsigned)((a->M + 3) / 4)), dim3(256), 0, stream, N);
  }
  hipLaunchKernelGGL(kernels[4 * (half ? 1 : 0) + 2 * (sw ? 1 : 0) + (a->norm ? 1 : 0)], dim3(grid), dim3(mlp::NTH),
                     half ? mlp::Geo<128>::LDS_BYTES : mlp::Geo<256>::LDS_BYTES, stream, P);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "projection gemm launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

int prefixlm_proj_gemm(const prefixlm_proj_gemm_args* a, void* stream) { return proj_gemm_launch(a, stream, false); }

int prefixlm_proj_gemm_scaled(const prefixlm_proj_gemm_args* a, void* stream) {
  return proj_gemm_launch(a, stream, true);
}

// Whether the 256-byte rows of a [B, N, H] cache with these element strides are all apart:
// with the dimensions ordered by stride, each stride covers the extent of the smaller ones.
static bool rows_apart(int64_t B, int64_t N, int64_t H, int64_t sb, int64_t sn, int64_t sh) {
  std::pair<int64_t, int64_t> d[3] = {{sb, B}, {sn, N}, {sh, H}};   // (stride, count)
  std::sort(d, d + 3);
  int64_t extent = kvc::D;
  for (const auto& x : d) {
    if (x.second == 1) continue;
    if (x.first < extent) return false;
    extent += x.first * (x.second - 1);
  }
  return true;
}

// Query waves of the extend kernel for S new rows, its query blocks, and the key splits of
// either kernel. one_round (the 8-bit cache's): above six splits, 512 workgroups at most.
static int ext_qw(int S) { return S <= 32 ? 1 : S <= 64 ? 2 : 4; }
static int kv_nqb(int S) { return S == 1 ? 1 : (S + 32 * ext_qw(S) - 1) / (32 * ext_qw(S)); }
static int64_t kv_nsplit(int64_t B, int S, int64_t H, int64_t Smax, bool one_round = false) {
  if (S == 1) {
    // Few (row, head) pairs: 512 workgroups, at least one 64-key step each (16 pairs x 4096
    // keys 13.1 us at 512, 14.2 at 1024, 12.0 at 256; 64 pairs 26.1, 26.7, 28.4). Many: 1024,
    // and two splits each of 512 keys or more, which even out ragged lengths (1024 pairs x
    // 4096: 272 us at one split, 263 at two, 266 at four; 2048 pairs x 256: 41 at one, 46 at
    // two).
    // Caches of up to 384 rows: one split, whose keys take less time than the combine's launch
    // (16 pairs x 128 keys 4.2 us, 6.9 with two splits; x 384 5.8 and 7.2; 128 pairs x 384 8.4
    // and 10.1; 32 pairs x 512 8.6 and 7.4).
    const int64_t units = B * H;
    if (units <= 128 && Smax <= 384) return 1;
    if (units <= 128)
      return std::max<int64_t>(1, std::min({(512 + units - 1) / units, (Smax + kvc::kStep - 1) / kvc::kStep,
                                            (int64_t)kvc::kMaxSplits}));
    // Caches of 1088 to 1535 rows: three splits where up to 1024 workgroups allow them (144 pairs x
    // 1300 rows 20% less than with two, 320 pairs 8%), not two of up to 750 keys.
    const int64_t most = Smax < 1088 ? Smax / 512 : std::max<int64_t>(3, Smax / 512);
    return std::max<int64_t>(1, std::min(std::max<int64_t>(2, (1024 + units - 1) / units), most));
  }
  const int64_t tk = 32 * (4 / ext_qw(S)), units = B * H * kv_nqb(S);
  // 512 workgroups fill the chip (two per CU); more splits mostly add partials to write and
  // merge: 4 x 16 heads x 45 queries 31 us at 512, 41 at 1024, 58 at 2048, and 2 x 16 x 300 on
  // 8192 rows 119 us at 256, 103 at 512, 97 at 1024, 115 at 2048
  int64_t want = (512 + units - 1) / units;
  const int64_t most = (Smax + tk - 1) / tk;
  if (one_round && want > 6) want = 512 / units;
  const int64_t n = std::max<int64_t>(1, std::min({want, most, (int64_t)kvc::kMaxSplits}));
  // One split instead where the tiles it walks more cost less than the combine's launch and the
  // partials, which n splits write and read for every query. The estimate: a tile of 32, 64 or 128
  // keys takes 1.27, 1.5 or 2.1 us with up to 512 workgroups, the launch 2.1 us at the least,
  // a partial 0.2 ns. 256 pairs x 64 queries, one split against two: 128-row caches 15.0 and
  // 32.6 us, 512 29.3 and 41.5; 64 pairs x 128 queries on 256 rows 24.9, and 29.8 with eight; 8
  // pairs x 64 queries on 256 rows 16.4, and 13.8 with the four it keeps. It errs beside its line
  // (256 pairs x 64 queries on 1024 rows 53.5 with the two it keeps, 44.0 with one), but 0.35 ns a
  // partial, right there, makes others worse (12 pairs x 200 queries on 200 rows 17.1 -> 22.1).
  const double c = ext_qw(S) == 1 ? 2100 : ext_qw(S) == 2 ? 1500 : 1270;   // ns
  const double one = (double)most * c * std::max(1.0, (double)units / 512);
  const double split = (double)((most + n - 1) / n) * c * std::max(1.0, (double)units * (double)n / 512) + 2100 +
                       0.2 * (double)B * S * (double)H * (double)n;
  return one <= split ? 1 : n;
}

// The reference's prefill, an empty cache and a packed batch of new rows: the varlen forward over
// them; with `append` the launch also writes them to the bf16 caches. Prompts whose rows lie further
// apart than that forward's offsets reach take the extend kernel, whose strides have 64 bits, and so do
// softmax scales that are not positive: the forward masks scores, and takes their maximum, before it scales.
static bool kv_prefills(const kvc::Params& P) {
  const int64_t S = P.S;
  const bool packed = P.B == 1 || (P.q_sb == S * P.q_ss && P.k_sb == S * P.k_ss && P.v_sb == S * P.v_ss &&
                                   P.o_sb == S * P.o_ss);
  return !P.seqlens && P.seqlen_const == 0 && P.s_new && P.scale_log2 > 0.f && packed && P.S <= P.Smax &&
         (int64_t)P.B * P.S < 0x7fffffff && P.q_ss >= kvc::D && P.k_ss >= kvc::D && P.v_ss >= kvc::D && P.o_ss >= kvc::D &&
         segment_fits(S, std::max(std::max(P.q_ss, P.k_ss), std::max(P.v_ss, P.o_ss)));
}
static int kv_prefill(const kvc::Params& P, bool append, hipStream_t stream) {
  const int B = P.B, S = P.S, H = P.H;
  const int64_t T = (int64_t)B * S;
  // one launch: the sequences are equal, so the forward needs no metadata and no work list, and
  // workgroups past its items append the new rows (append, metadata, work list and forward as
  // four launches took 46.8 us a call for 2 x 1021 rows x 16 heads, now 32.7)
  const void* fp[] = {P.q, P.k, P.v, P.out};
  const int64_t fs[] = {P.q_ss, P.q_sh, P.k_ss,   P.k_sh,
                        P.v_ss, P.v_sh, P.o_ss, P.o_sh};
  const int rc = check_common(fp, 4, fs, 4, (int32_t)T, H, kvc::D, (int32_t)T, 0, S, 0, nullptr, nullptr, nullptr);
  if (rc) return rc;
  fwd::Params F{};
  F.q = P.q;
  F.k = P.k;
  F.v = P.v;
  F.o = P.out;
  F.q_st = P.q_ss; F.q_sh = P.q_sh;
  F.k_st = P.k_ss; F.k_sh = P.k_sh;
  F.v_st = P.v_ss; F.v_sh = P.v_sh;
  F.o_st = P.o_ss; F.o_sh = P.o_sh;
  F.T = F.total = (int)T;
  F.H = H;
  F.is_causal = P.causal;
  F.numseqs = B;
  F.scale_log2 = P.scale_log2;
  F.seq_len = S;
  F.kc = P.kc;
  F.vc = P.vc;
  F.kc_sb = P.kc_sb; F.kc_ss = P.kc_ss; F.kc_sh = P.kc_sh;
  F.vc_sb = P.vc_sb; F.vc_ss = P.vc_ss; F.vc_sh = P.vc_sh;
  const int64_t items = (int64_t)B * ((S + fwd::BM - 1) / fwd::BM), nblk = unit_grid(items, H);
  bool split = false;
  int cus = 0;
  int rc2 = fwd_splits_keys(nblk, S, &split);
  if (!rc2) rc2 = persistent_grid(&cus);
  if (rc2) return rc2;
  // More workgroups than the CUs hold at once (three each), all with the same keys to walk: one
  // sequence after another, so that those running together share its keys and values in L2 (8 x
  // 4100 rows x 16 heads 1327 us with the tiles of all sequences mixed, 1205 so; below that
  // number 8 x 300 rows 18.5 and 19.1)
  F.seq_major = !P.causal && nblk > 3 * (int64_t)cus;
  const int nt = fwd::NT * (split ? 2 : 1), per = nt * fwd::kAppend;
  const int64_t nappend = append ? (T * H * 16 + per - 1) / per : 0;
  if (nblk + nappend > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "grid too large");
  F.n_main = (int)nblk;
  if (split)
    hipLaunchKernelGGL((fwd::prefixlm_fwd_kernel<kvc::D, true, 2>), dim3((unsigned)(nblk + nappend)), dim3(nt),
                       2 * fwd::Geo<kvc::D>::LDS_BYTES, stream, F);
  else
    hipLaunchKernelGGL((fwd::prefixlm_fwd_kernel<kvc::D, true>), dim3((unsigned)(nblk + nappend)), dim3(nt),
                       fwd::Geo<kvc::D>::LDS_BYTES, stream, F);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "prefill launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

size_t prefixlm_kvcache_workspace_size(int32_t batch, int32_t seqlen_q, int32_t num_heads, int32_t head_dim,
                                       int32_t max_seqlen_cache) {
  (void)head_dim;
  if (batch < 1 || seqlen_q < 1 || num_heads < 1 || max_seqlen_cache < 1) return 0;
  const int64_t nsplit = kv_nsplit(batch, seqlen_q, num_heads, max_seqlen_cache);
  if (nsplit == 1) return kAlign;   // written directly
  return align_up(sizeof(float) * (size_t)batch * seqlen_q * num_heads * nsplit * kvc::kPart);
}

int prefixlm_kvcache_fwd(const prefixlm_kvcache_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int B = a->batch, S = a->seqlen_q, H = a->num_heads, Smax = a->max_seqlen_cache;
  if (a->head_dim != kvc::D) return fail(PREFIXLM_ERR_INVALID, "head_dim must be 128 (got %d)", a->head_dim);
  if (B < 1 || S < 1 || H < 1 || Smax < 1)
    return fail(PREFIXLM_ERR_INVALID, "batch=%d seqlen_q=%d num_heads=%d max_seqlen_cache=%d must be >= 1", B, S,
                H, Smax);
  const bool has_new = a->k != nullptr;
  if ((a->k == nullptr) != (a->v == nullptr)) return fail(PREFIXLM_ERR_INVALID, "k and v must be given together");
  if (!a->cache_seqlens && (a->cache_seqlen < 0 || a->cache_seqlen > Smax))
    return fail(PREFIXLM_ERR_INVALID, "cache_seqlen=%d outside [0, %d]", a->cache_seqlen, Smax);
  const void* ptrs[] = {a->q, a->k_cache, a->v_cache, a->out, a->workspace, a->k, a->v};
  const int nptr = has_new ? 7 : 5;
  for (int i = 0; i < nptr; ++i)
    if (!ptrs[i] || !aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "tensor pointer %d is null or not 16-byte aligned", i);
  const int64_t st[] = {a->q_stride_b,       a->q_stride_s,       a->q_stride_h,       a->k_cache_stride_b,
                        a->k_cache_stride_s, a->k_cache_stride_h, a->v_cache_stride_b, a->v_cache_stride_s,
                        a->v_cache_stride_h, a->out_stride_b,     a->out_stride_s,     a->out_stride_h,
                        a->k_stride_b,       a->k_stride_s,       a->k_stride_h,       a->v_stride_b,
                        a->v_stride_s,       a->v_stride_h};
  for (int i = 0; i < (has_new ? 18 : 12); ++i)
    if (st[i] < 0 || st[i] % 8)
      return fail(PREFIXLM_ERR_INVALID, "stride %d (%lld) must be a non-negative multiple of 8", i, (long long)st[i]);
  const size_t need = prefixlm_kvcache_workspace_size(B, S, H, a->head_dim, Smax);
  if (a->workspace_bytes < need)
    return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes, %zu needed", a->workspace_bytes, need);

  kvc::Params P{};
  P.q = static_cast<const bf16*>(a->q);
  P.k = static_cast<const bf16*>(a->k);
  P.v = static_cast<const bf16*>(a->v);
  P.kc = static_cast<bf16*>(a->k_cache);
  P.vc = static_cast<bf16*>(a->v_cache);
  P.out = static_cast<bf16*>(a->out);
  P.part = static_cast<float*>(a->workspace);
  P.seqlens = a->cache_seqlens;
  P.q_sb = a->q_stride_b; P.q_ss = a->q_stride_s; P.q_sh = a->q_stride_h;
  P.k_sb = a->k_stride_b; P.k_ss = a->k_stride_s; P.k_sh = a->k_stride_h;
  P.v_sb = a->v_stride_b; P.v_ss = a->v_stride_s; P.v_sh = a->v_stride_h;
  P.kc_sb = a->k_cache_stride_b; P.kc_ss = a->k_cache_stride_s; P.kc_sh = a->k_cache_stride_h;
  P.vc_sb = a->v_cache_stride_b; P.vc_ss = a->v_cache_stride_s; P.vc_sh = a->v_cache_stride_h;
  P.o_sb = a->out_stride_b; P.o_ss = a->out_stride_s; P.o_sh = a->out_stride_h;
  P.B = B; P.S = S; P.H = H; P.Smax = Smax;
  P.nsplit = (int)kv_nsplit(B, S, H, Smax);
  P.nqb = kv_nqb(S);
  P.causal = a->is_causal ? 1 : 0;
  P.seqlen_const = a->cache_seqlen;
  P.s_new = has_new ? S : 0;
  P.scale_log2 = a->softmax_scale * kLog2e;

  (void)hipGetLastError();
  const bool prefill = kv_prefills(P);
  // The decode and extend kernels read the new rows from k, v and write them to the caches in
  // one launch; that needs cache rows of its own for every (b, row, head) and two caches (a
  // row shared between batch rows would be read by one while the other writes it).
  P.fused = !prefill && has_new &&
            rows_apart(B, Smax, H, a->k_cache_stride_b, a->k_cache_stride_s, a->k_cache_stride_h) &&
            rows_apart(B, Smax, H, a->v_cache_stride_b, a->v_cache_stride_s, a->v_cache_stride_h) &&
            a->k_cache != a->v_cache;
  if (has_new && !P.fused && !prefill) {
    const int64_t threads = (int64_t)B * S * H * 16;
    if ((threads + 255) / 256 > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "too many rows");
    hipLaunchKernelGGL(kvc::append_kernel, dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, stream, P);
  }
  set_kernel_attrs();
  if (g_attr_err != hipSuccess)
    return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(g_attr_err));
  if (prefill) {
    return kv_prefill(P, true, stream);
  }
  {
    const int64_t units = (int64_t)B * H * P.nsplit, nblk = S == 1 ? units : (units + 7) / 8 * 8 * P.nqb;
    if (nblk > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "grid too large");
    if (S == 1 && P.nsplit == 1 && (int64_t)B * H <= 256 && Smax > kvc::kStep)
      // one workgroup per CU at most: eight waves each (256 pairs x 256 keys 7.5 -> 6.4 us, x 768
      // 18.5 -> 15.8; 512 pairs x 192 8.7 and 9.1; x 64 keys, one step of four waves, 4.0 and 4.4;
      // sixteen waves are slower than eight everywhere below 512 keys)
      hipLaunchKernelGGL(kvc::decode_kernel<512>, dim3((unsigned)nblk), dim3(512), 0, stream, P);
    else if (S == 1)
      hipLaunchKernelGGL(kvc::decode_kernel<kvc::NT>, dim3((unsigned)nblk), dim3(kvc::NT), 0, stream, P);
    else if (ext_qw(S) == 1)
      hipLaunchKernelGGL(kvc::extend_kernel<1>, dim3((unsigned)nblk), dim3(kvc::NT), kvc::ExtGeo<1>::LDS_BYTES, stream, P);
    else if (ext_qw(S) == 2)
      hipLaunchKernelGGL(kvc::extend_kernel<2>, dim3((unsigned)nblk), dim3(kvc::NT), kvc::ExtGeo<2>::LDS_BYTES, stream, P);
    else
      hipLaunchKernelGGL(kvc::extend_kernel<4>, dim3((unsigned)nblk), dim3(kvc::NT), kvc::ExtGeo<4>::LDS_BYTES, stream, P);
    if (P.nsplit > 1) {
      const int64_t waves = (int64_t)B * S * H;
      hipLaunchKernelGGL(kvc::combine_kernel<>, dim3((unsigned)((waves * 64 + 255) / 256)), dim3(256), 0, stream, P);
    }
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "kv-cache launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

size_t prefixlm_plan_size(int32_t total_seqlen, int32_t numseqs) {
  if (total_seqlen < 0 || numseqs < 0) return 0;
  return plan::layout(kPlanLists, total_seqlen, numseqs).bytes;
}

int prefixlm_plan_build(const int32_t* prefix_lens, const int32_t* causal_lens, const int32_t* cu_seqlens,
                        int32_t numseqs, int32_t total_seqlen, int32_t num_tokens, int32_t is_causal,
                        void* plan_out, size_t plan_bytes) {
  if (numseqs < 0 || total_seqlen < 0 || total_seqlen > num_tokens)
    return fail(PREFIXLM_ERR_INVALID, "numseqs=%d, total_seqlen=%d, num_tokens=%d are inconsistent", numseqs,
                total_seqlen, num_tokens);
  if (numseqs > 0 && (!prefix_lens || !causal_lens || !cu_seqlens))
    return fail(PREFIXLM_ERR_INVALID, "metadata pointers must be non-null");
  const plan::Layout l = plan::layout(kPlanLists, total_seqlen, numseqs);
  if (!plan_out || plan_bytes != l.bytes)
    return fail(PREFIXLM_ERR_INVALID, "plan buffer of %zu bytes, %zu needed", plan_bytes, l.bytes);
  const int32_t err = plan::build(kPlanLists, l, prefix_lens, causal_lens, cu_seqlens, numseqs, total_seqlen,
                                  num_tokens, is_causal ? 1 : 0, static_cast<unsigned char*>(plan_out));
  if (err)
    return fail(PREFIXLM_ERR_METADATA,
                "inconsistent metadata (flags 0x%x): segments must satisfy cu_seqlens[0]=0, "
                "cu_seqlens[s+1]=cu_seqlens[s]+prefix_lens[s]+causal_lens[s] <= total_seqlen",
                err);
  return PREFIXLM_OK;
}

int64_t prefixlm_plan_ds_blocks(const void* plan_p, size_t plan_bytes) {
  if (!plan_p || plan_bytes < sizeof(WsHeader)) return -1;
  WsHeader h;
  memcpy(&h, plan_p, sizeof(h));
  if (h.pad[0] != plan::kPlanMagic || h.pad[1] < 0 || h.pad[2] < 0) return -1;
  if (plan::layout(kPlanLists, h.pad[2], h.pad[1]).bytes != plan_bytes) return -1;
  return h.pad[4];
}

void* prefixlm_timer_create(void) { return new (std::nothrow) prefixlm_timer(); }

void prefixlm_timer_destroy(void* timer) {
  prefixlm_timer* t = static_cast<prefixlm_timer*>(timer);
  if (!t) return;
  for (auto& r : t->recs) {
    (void)hipEventDestroy(r.a);
    (void)hipEventDestroy(r.b);
  }
  for (hipEvent_t e : t->pool) (void)hipEventDestroy(e);
  delete t;
}

int prefixlm_timer_read(void* timer, float* total_ms, int32_t* launches) {
  prefixlm_timer* t = static_cast<prefixlm_timer*>(timer);
  if (!t) return fail(PREFIXLM_ERR_INVALID, "timer is null");
  for (int i = 0; i < PREFIXLM_NUM_KERNELS; ++i) {
    if (total_ms) total_ms[i] = 0.f;
    if (launches) launches[i] = 0;
  }
  int rc = PREFIXLM_OK;
  for (auto& r : t->recs) {
    float ms = 0.f;
    hipError_t e = hipEventSynchronize(r.b);
    if (e == hipSuccess) e = hipEventElapsedTime(&ms, r.a, r.b);
    if (e != hipSuccess) {
      rc = fail(PREFIXLM_ERR_HIP, "timing event: %s", hipGetErrorString(e));
    } else if (r.id >= 0 && r.id < PREFIXLM_NUM_KERNELS) {
      if (total_ms) total_ms[r.id] += ms;
      if (launches) launches[r.id] += 1;
    }
    t->pool.push_back(r.a);
    t->pool.push_back(r.b);
  }
  t->recs.clear();
  return rc;
}

}  // extern "C"

// A launch has fewer than 2^32 threads
static bool launchable(int64_t blocks, int64_t threads) { return blocks <= 0xffffffffll / threads && blocks <= 0x7fffffff; }

// ---- log probabilities ---------------------------------------------------------------
// Splits of a row, where the rows alone are far fewer than the CUs and long enough to pay for the second
// launch: 512 workgroups, of at least 8192 logits each. One split against several: 8 rows of 98304 logits
// 8.2 and 9.1 us, of 131072 9.8 and 9.2, of 262144 16.8 and 9.1; with five alternatives, whose search is
// shorter in a split, of 65536 10.3 and 11.0, of 98304 12.1 and 11.6 (64 rows 12.3 and 13.7), of 131072
// 14.2 and 11.7; with 20, 8 rows of 98304 13.0 and 14.5, of 131072 15.0 and 14.5. 64 rows of 262144 17.2
// and 9.5, 200 rows 18.0 and 26.4. The alternatives of all splits are ranked together, each by one of 256
// threads: with more of them than that 8 rows of 262144 with 20 took 37.2 us, now 15.5, one split 22.8.
static int lp_nsplit(int64_t rows, int64_t V, int32_t top) {
  if (rows < 1 || rows > 64 || V < (top > 0 && top <= 8 && rows <= 16 ? 98304 : 131072)) return 1;
  const int64_t most = V / (16 * lp::NT), want = (512 + rows - 1) / rows;
  const int64_t fit = top > 0 ? 256 / top : lp::kMaxSplits;
  return (int)std::min({most, want, fit, (int64_t)lp::kMaxSplits});
}
static_assert(256 / lp::kMaxTop >= 1 && 256 <= lp::kCand, "a split at least, and the combine's candidates fit");

static size_t lp_workspace(int64_t rows, int64_t vocab, int32_t top_k) {
  if (rows < 1 || vocab < 1 || top_k < 0) return 0;
  const int n = lp_nsplit(rows, vocab, top_k);
  return n == 1 ? 0 : align_up((size_t)rows * n * 16) + align_up((size_t)rows * n * top_k * 8);
}

template <class T, bool ENT, bool TOP>
static void lp_fwd_launch(const lp::Params& P, hipStream_t stream) {
  hipLaunchKernelGGL((lp::forward_kernel<T, ENT, TOP>), dim3((unsigned)(P.rows * P.nsplit)), dim3(lp::NT), 0, stream, P);
  if (P.nsplit > 1)
    hipLaunchKernelGGL((lp::combine_kernel<T, ENT, TOP>), dim3((unsigned)P.rows), dim3(256), 0, stream, P);
}
template <class T>
static void lp_fwd_launch(const lp::Params& P, hipStream_t stream) {
  if (P.entropy)
    P.top ? lp_fwd_launch<T, true, true>(P, stream) : lp_fwd_launch<T, true, false>(P, stream);
  else
    P.top ? lp_fwd_launch<T, false, true>(P, stream) : lp_fwd_launch<T, false, false>(P, stream);
}

template <class T>
static void lp_bwd_launch(const lp::Params& P, bool nt, int nblk, hipStream_t stream) {
  auto* k = P.h ? (nt ? lp::backward_kernel<T, true, true> : lp::backward_kernel<T, true, false>)
                : (nt ? lp::backward_kernel<T, false, true> : lp::backward_kernel<T, false, false>);
  hipLaunchKernelGGL(k, dim3((unsigned)(P.rows * nblk)), dim3(256), 0, stream, P, nblk);
}

static int lp_call(const prefixlm_logprob_args* a, void* stream_, bool backward) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  if (a->rows < 0 || a->vocab < 1 || a->vocab > 0x7fffffff)
    return fail(PREFIXLM_ERR_INVALID, "rows=%lld vocab=%lld: vocab must be in [1, 2^31)", (long long)a->rows,
                (long long)a->vocab);
  if (!backward && (a->top_k < 0 || a->top_k > lp::kMaxTop || a->top_k > a->vocab))
    return fail(PREFIXLM_ERR_INVALID, "top_k=%d must be in [0, min(%d, vocab)]", a->top_k, lp::kMaxTop);
  if (a->rows == 0) return PREFIXLM_OK;   // empty tensors may have null pointers
  const uintptr_t size = a->x_fp32 ? 4 : 2;
  if (!a->x || (uintptr_t)a->x % size) return fail(PREFIXLM_ERR_INVALID, "x is null or not aligned to its element");
  if (a->x_stride < 0) return fail(PREFIXLM_ERR_INVALID, "x_stride (%lld) must be >= 0", (long long)a->x_stride);
  if (!a->stats) return fail(PREFIXLM_ERR_INVALID, "stats is null");
  if (!a->targets && (a->logprob || (backward && a->dlogprob)))
    return fail(PREFIXLM_ERR_INVALID, "targets is null");
  lp::Params P{};
  P.x = a->x;
  P.targets = a->targets;
  P.stats = a->stats;
  P.entropy = a->entropy;
  P.x_st = a->x_stride;
  P.rows = a->rows;
  P.V = a->vocab;
  P.ignore = a->ignore_index;
  P.wide_targets = !a->targets_int32;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  if (backward) {
    if (!a->dx || (uintptr_t)a->dx % size) return fail(PREFIXLM_ERR_INVALID, "dx is null or not aligned to its element");
    if (a->dx_stride < a->vocab)
      return fail(PREFIXLM_ERR_INVALID, "dx_stride (%lld) must be >= vocab", (long long)a->dx_stride);
    if (a->dentropy && !a->entropy) return fail(PREFIXLM_ERR_INVALID, "dentropy needs the forward's entropy");
    P.dx = a->dx;
    P.dx_st = a->dx_stride;
    P.g = a->dlogprob;
    P.h = a->dentropy;
    const int64_t nblk = (a->vocab + 8 * 256 * lp::kUnroll - 1) / (8 * 256 * lp::kUnroll);
    if (a->rows > 0x7fffffff || !launchable(a->rows * nblk, 256)) return fail(PREFIXLM_ERR_INVALID, "too many elements");
    (void)hipGetLastError();
    const bool nt = 2 * a->rows * a->vocab * (int64_t)size > lp::kNtBytes;
    if (a->x_fp32)
      lp_bwd_launch<float>(P, nt, (int)nblk, stream);
    else
      lp_bwd_launch<bf16>(P, nt, (int)nblk, stream);
  } else {
    if (a->targets && !a->logprob) return fail(PREFIXLM_ERR_INVALID, "logprob is null");
    if (a->top_k && (!a->top_logprobs || !a->top_ids))
      return fail(PREFIXLM_ERR_INVALID, "top_logprobs or top_ids is null");
    P.logprob = a->logprob;
    P.top = a->top_k;
    P.top_val = a->top_logprobs;
    P.top_id = a->top_ids;
    P.nsplit = lp_nsplit(a->rows, a->vocab, a->top_k);
    if (P.nsplit > 1) {
      const size_t need = lp_workspace(a->rows, a->vocab, a->top_k);
      if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need)
        return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes is null, unaligned or below %zu", a->workspace_bytes, need);
      P.part = static_cast<float*>(a->workspace);
      P.part_top = reinterpret_cast<unsigned long long*>(static_cast<char*>(a->workspace) +
                                                         align_up((size_t)a->rows * P.nsplit * 16));
    }
    if (a->rows > 0x7fffffff || !launchable(a->rows * P.nsplit, lp::NT)) return fail(PREFIXLM_ERR_INVALID, "too many rows");
    (void)hipGetLastError();
    if (a->x_fp32)
      lp_fwd_launch<float>(P, stream);
    else
      lp_fwd_launch<bf16>(P, stream);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "log probabilities launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

extern "C" {

size_t prefixlm_logprob_workspace_size(int64_t rows, int64_t vocab, int32_t top_k) {
  return lp_workspace(rows, vocab, top_k);
}
int prefixlm_logprob_fwd(const prefixlm_logprob_args* a, void* stream) { return lp_call(a, stream, false); }
int prefixlm_logprob_bwd(const prefixlm_logprob_args* a, void* stream) { return lp_call(a, stream, true); }

}  // extern "C"

// ---- embedding -----------------------------------------------------------------------
// The sort's tiles: 2048 tokens, or more where that would be over kMaxTiles of them
static int emb_tile(int64_t T) {
  const int64_t per = (T + emb::kMaxTiles - 1) / emb::kMaxTiles;
  return (int)std::max<int64_t>(2048, (per + emb::kSortThreads - 1) / emb::kSortThreads * emb::kSortThreads);
}
// Sorted tokens per wave of the sum: 32, or 16 where that leaves fewer than 2048 waves (4999 tokens x
// 1280 columns 13.6 and 9.0 us; 16384 x 2048 the sum takes 41.8 and 40.9, the join of the twice as many
// partials 6.6 and 9.0).
static int emb_run(int64_t T, int32_t cols) {
  return T * ((cols + 511) / 512) < 2048 * 2 * emb::kMinRun ? emb::kMinRun : 2 * emb::kMinRun;
}

struct EmbWorkspace {
  size_t key[2], pos[2], hist, part, total;
};
static EmbWorkspace emb_workspace(int64_t T, int32_t cols) {
  EmbWorkspace w{};
  size_t at = 0;
  auto take = [&at](size_t n) {
    const size_t here = at;
    at += align_up(n);
    return here;
  };
  const int tile = emb_tile(T);
  for (int i = 0; i < 2; ++i) {
    w.key[i] = take((size_t)T * 4);
    w.pos[i] = take((size_t)T * 4);
  }
  w.hist = take((size_t)((T + tile - 1) / tile) * emb::kBins * 4);
  w.part = take((size_t)((T + emb_run(T, cols) - 1) / emb_run(T, cols)) * 2 * (size_t)cols * 4);
  w.total = at;
  return w;
}

extern "C" {

size_t prefixlm_embedding_workspace_size(int64_t tokens, int64_t vocab, int32_t cols) {
  (void)vocab;
  return tokens < 1 || cols < 1 ? 0 : emb_workspace(tokens, cols).total;
}

static int emb_check(const prefixlm_embedding_args* a) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  if (a->tokens < 0 || a->tokens > 0x7fffffff || a->vocab < 1 || a->vocab >= (1 << 27))
    return fail(PREFIXLM_ERR_INVALID, "tokens=%lld vocab=%lld: tokens must be below 2^31, vocab in [1, 2^27)",
                (long long)a->tokens, (long long)a->vocab);
  if (a->cols < 8 || a->cols % 8) return fail(PREFIXLM_ERR_INVALID, "cols=%d must be a positive multiple of 8", a->cols);
  return PREFIXLM_OK;
}
static int emb_rows(const void* p, int64_t stride, int32_t fp32, int32_t cols, bool repeats, const char* name) {
  if (!p || !aligned16(p)) return fail(PREFIXLM_ERR_INVALID, "%s is null or not 16-byte aligned", name);
  if ((stride < cols && !(repeats && stride == 0)) || stride % (fp32 ? 4 : 8))
    return fail(PREFIXLM_ERR_INVALID, "row stride of %s (%lld) must be 16-byte rows and >= cols", name, (long long)stride);
  return PREFIXLM_OK;
}

int prefixlm_embedding_fwd(const prefixlm_embedding_args* a, void* stream_) {
  int rc = emb_check(a);
  if (rc) return rc;
  if (a->tokens == 0) return PREFIXLM_OK;
  if (!a->ids) return fail(PREFIXLM_ERR_INVALID, "ids is null");
  rc = emb_rows(a->table, a->table_stride, a->table_fp32, a->cols, true, "table");
  if (!rc) rc = emb_rows(a->y, a->y_stride, a->y_fp32, a->cols, false, "y");
  if (rc) return rc;
  const int64_t nblk = (a->tokens * (a->cols / 8) + 255) / 256;
  if (!launchable(nblk, 256)) return fail(PREFIXLM_ERR_INVALID, "too many elements");
  const emb::FwdParams P{a->table, a->ids, a->y, a->table_stride, a->y_stride, a->tokens, a->vocab, a->cols,
                         !a->ids_int32, a->scale};
  (void)hipGetLastError();
  auto* k = a->table_fp32 ? (a->y_fp32 ? emb::lookup_kernel<float, float> : emb::lookup_kernel<float, bf16>)
                          : (a->y_fp32 ? emb::lookup_kernel<bf16, float> : emb::lookup_kernel<bf16, bf16>);
  hipLaunchKernelGGL(k, dim3((unsigned)nblk), dim3(256), 0, reinterpret_cast<hipStream_t>(stream_), P);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "embedding launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

int prefixlm_embedding_bwd(const prefixlm_embedding_args* a, void* stream_) {
  int rc = emb_check(a);
  if (rc) return rc;
  rc = emb_rows(a->grad, a->cols, a->table_fp32, a->cols, false, "grad");
  if (!rc && a->tokens) rc = emb_rows(a->dy, a->dy_stride, a->y_fp32, a->cols, true, "dy");
  if (rc) return rc;
  if (a->tokens && !a->ids) return fail(PREFIXLM_ERR_INVALID, "ids is null");
  const size_t need = prefixlm_embedding_workspace_size(a->tokens, a->vocab, a->cols);
  if (a->tokens && (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need))
    return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes is null, unaligned or below %zu", a->workspace_bytes, need);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int64_t T = a->tokens, units = a->vocab * a->cols * (a->table_fp32 ? 4 : 2) / 16;
  int bits = 1, passes = 1;
  while ((a->vocab >> bits) != 0) ++bits;   // keys up to vocab
  passes = T ? (bits + emb::kBits - 1) / emb::kBits : 0;
  const int run = emb_run(T, a->cols);
  const int64_t waves = (T + run - 1) / run * ((a->cols + 511) / 512);
  if (!launchable((waves + 3) / 4, 256)) return fail(PREFIXLM_ERR_INVALID, "too many elements");
  const EmbWorkspace w = emb_workspace(T, a->cols);
  char* ws = static_cast<char*>(a->workspace);
  emb::SortParams P{};
  P.zero = a->grad;
  P.T = T;
  P.V = a->vocab;
  P.padding = a->padding_id;
  P.wide_ids = !a->ids_int32;
  P.tile = emb_tile(T);
  P.tiles = (int)((T + P.tile - 1) / P.tile);
  (void)hipGetLastError();
  const bool one = T > 0 && T <= emb::kRankTokens && a->vocab <= emb::kRankIds;
  const int launches = std::max(1, 2 * passes);
  int done = 0;
  auto share = [&] {   // of the clearing, for the next launch; and its workgroups
    P.zero_begin = units * done / launches;
    P.zero_end = units * ++done / launches;
    return (unsigned)(P.tiles + std::min<int64_t>(2048, (P.zero_end - P.zero_begin + 255) / 256));
  };
  if (one) {
    P.ids = a->ids;
    P.key_out = reinterpret_cast<uint32_t*>(ws + w.key[0]);
    P.pos_out = reinterpret_cast<uint32_t*>(ws + w.pos[0]);
    P.zero_begin = 0;
    P.zero_end = units;
    // one workgroup a CU at most: 4999 tokens 13.4 us (64 a workgroup 20.9)
    P.tile = (int)std::max<int64_t>(16, (T + 511) / 512 * 2);
    P.tiles = (int)((T + P.tile - 1) / P.tile);
    const int64_t n = P.tiles + std::min<int64_t>(256, (units + 4 * emb::kRankThreads - 1) / (4 * emb::kRankThreads));
    auto* k = T <= 1024   ? emb::rank_kernel<1>
              : T <= 2048 ? emb::rank_kernel<2>
              : T <= 4096 ? emb::rank_kernel<4>
              : T <= 6144 ? emb::rank_kernel<6>
              : T <= 8192 ? emb::rank_kernel<8>
              : T <= 12288 ? emb::rank_kernel<12>
                           : emb::rank_kernel<16>;
    hipLaunchKernelGGL(k, dim3((unsigned)n), dim3(emb::kRankThreads), 0, stream, P);
  } else if (T == 0) {
    const unsigned n = share();
    hipLaunchKernelGGL(emb::histogram_kernel, dim3(n), dim3(emb::kSortThreads), 0, stream, P);
  }
  for (int p = 0; p < (one ? 0 : passes); ++p) {
    P.ids = p == 0 ? a->ids : nullptr;
    P.key_in = reinterpret_cast<const uint32_t*>(ws + w.key[(p + 1) & 1]);
    P.pos_in = reinterpret_cast<const uint32_t*>(ws + w.pos[(p + 1) & 1]);
    P.key_out = reinterpret_cast<uint32_t*>(ws + w.key[p & 1]);
    P.pos_out = reinterpret_cast<uint32_t*>(ws + w.pos[p & 1]);
    P.hist = reinterpret_cast<uint32_t*>(ws + w.hist);
    P.shift = p * emb::kBits;
    unsigned n = share();
    hipLaunchKernelGGL(emb::histogram_kernel, dim3(n), dim3(emb::kSortThreads), 0, stream, P);
    n = share();
    hipLaunchKernelGGL(emb::scatter_kernel, dim3(n), dim3(emb::kSortThreads), 0, stream, P);
  }
  if (T > 0) {
    emb::SumParams S{};
    S.key = P.key_out;
    S.pos = P.pos_out;
    S.dy = a->dy;
    S.grad = a->grad;
    S.part = reinterpret_cast<float*>(ws + w.part);
    S.dy_st = a->dy_stride;
    S.T = T;
    S.V = a->vocab;
    S.cols = a->cols;
    S.run = run;
    S.chunks = (int)((T + run - 1) / run);
    S.scale = a->scale;
    auto* k = a->table_fp32 ? (a->y_fp32 ? emb::sum_kernel<float, float> : emb::sum_kernel<bf16, float>)
                            : (a->y_fp32 ? emb::sum_kernel<float, bf16> : emb::sum_kernel<bf16, bf16>);
    hipLaunchKernelGGL(k, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream, S);
    if (S.chunks > 1)
      hipLaunchKernelGGL(a->table_fp32 ? emb::join_kernel<float> : emb::join_kernel<bf16>,
                         dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, stream, S);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "embedding gradient launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

}  // extern "C"

// ---- attention over an 8-bit cache -----------------------------------------------------------
// Splits of the keys. Several queries: as for bf16 (the tiles are the same), but above six splits no
// more than 512 workgroups, as a second round of a few costs more than the longer splits (24 units x
// 10569 keys, 100 queries, 67.7 us with 22 splits, 51 with 21, of ragged rows 63.8 and 47.4; 60 x 4006, 90
// queries 63.5 and 50.7, ragged 62.9 and 53.8). Not from five splits down, where it depends on the rows: 120
// units x 4178 keys of ragged rows took 95 with five and 110 with four in one batch, 101 and 92 in another
// (90 queries), 66 and 58 (45). One query:
// one split for caches of up to 1536 rows, whose keys take less time than the combine's launch (16
// pairs x 920 of 1536 rows 8.7 us, 11.3 with three splits; 128 x 800 of 1024 9.9 and 12.8; 64 x 1800
// of 2048 14.8, 13.2 with four), and from 192 pairs on, one for each CU nearly (256 x 12288 of 16384
// ragged rows 128.7, 131.3 with twelve; 256 x 1500 of 2048 19.8 and 22.7). Else 768 workgroups (48
// pairs x 23000 of 32768 rows 51.3 with 16 splits, 54.8 with eight; 80 x 4096 20.1 with twelve, 24.2
// with two), of at least two blocks each.
static int64_t kv8_nsplit(int64_t B, int S, int64_t H, int64_t Smax) {
  if (S > 1) return kv_nsplit(B, S, H, Smax, true);
  const int64_t units = B * H;
  if (Smax <= 1536 || units >= 192) return 1;
  return std::min({(768 + units - 1) / units, Smax / (2 * kv8::kBlock), (int64_t)kvc::kMaxSplits});
}

template <class C>
static void kv8_launch(const kv8::Params& P, int64_t nblk, hipStream_t stream) {
  const dim3 g((unsigned)nblk), n(kvc::NT);
  // one split: eight waves (16 pairs x 920 rows 10.4 -> 8.7 us, 128 x 800 11.8 -> 9.9, 2048 x 800 70.4
  // -> 67.7), unless many pairs have short caches (1024 x 200 of 256 rows 15.9, with four 12.7)
  if (P.S == 1 && P.nsplit == 1 && !((int64_t)P.B * P.H > 512 && P.Smax <= 512))
    hipLaunchKernelGGL((kv8::decode_kernel<C, 512>), g, dim3(512), 0, stream, P);
  else if (P.S == 1)
    hipLaunchKernelGGL((kv8::decode_kernel<C, kvc::NT>), g, n, 0, stream, P);
  else if (ext_qw(P.S) == 1)
    hipLaunchKernelGGL((kv8::extend_kernel<C, 1>), g, n, kvc::ExtGeo<1>::LDS_BYTES, stream, P);
  else if (ext_qw(P.S) == 2)
    hipLaunchKernelGGL((kv8::extend_kernel<C, 2>), g, n, kvc::ExtGeo<2>::LDS_BYTES, stream, P);
  else
    hipLaunchKernelGGL((kv8::extend_kernel<C, 4>), g, n, kvc::ExtGeo<4>::LDS_BYTES, stream, P);
}

// Dynamic LDS above the default limit has to be allowed once per kernel and device
static int kv8_allow_lds() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
  if (dev < 0 || dev >= 64) return fail(PREFIXLM_ERR_INVALID, "device %d >= 64", dev);
  std::lock_guard<std::mutex> g(mu);
  if (done[dev]) return PREFIXLM_OK;
  const std::pair<const void*, int> kernels[] = {
      {(const void*)kv8::extend_kernel<kv8::E4M3, 1>, kvc::ExtGeo<1>::LDS_BYTES},
      {(const void*)kv8::extend_kernel<kv8::E4M3, 2>, kvc::ExtGeo<2>::LDS_BYTES},
      {(const void*)kv8::extend_kernel<kv8::E4M3, 4>, kvc::ExtGeo<4>::LDS_BYTES},
      {(const void*)kv8::extend_kernel<kv8::Int8, 1>, kvc::ExtGeo<1>::LDS_BYTES},
      {(const void*)kv8::extend_kernel<kv8::Int8, 2>, kvc::ExtGeo<2>::LDS_BYTES},
      {(const void*)kv8::extend_kernel<kv8::Int8, 4>, kvc::ExtGeo<4>::LDS_BYTES}};
  for (const auto& k : kernels) {
    e = hipFuncSetAttribute(k.first, hipFuncAttributeMaxDynamicSharedMemorySize, k.second);
    if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  }
  done[dev] = true;
  return PREFIXLM_OK;
}

extern "C" {

size_t prefixlm_kvcache8_workspace_size(int32_t batch, int32_t seqlen_q, int32_t num_heads, int32_t max_seqlen_cache) {
  if (batch < 1 || seqlen_q < 1 || num_heads < 1 || max_seqlen_cache < 1) return 0;
  const int64_t nsplit = kv8_nsplit(batch, seqlen_q, num_heads, max_seqlen_cache);
  return nsplit == 1 ? 0 : align_up(sizeof(float) * (size_t)batch * seqlen_q * num_heads * nsplit * kvc::kPart);
}

int prefixlm_kvcache8_fwd(const prefixlm_kvcache8_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const int B = a->batch, S = a->seqlen_q, H = a->num_heads, Smax = a->max_seqlen_cache;
  if (a->head_dim != kvc::D) return fail(PREFIXLM_ERR_INVALID, "head_dim must be 128 (got %d)", a->head_dim);
  if (B < 1 || S < 1 || H < 1 || Smax < 1 || Smax % kv8::kBlock)
    return fail(PREFIXLM_ERR_INVALID,
                "batch=%d seqlen_q=%d num_heads=%d must be >= 1 and max_seqlen_cache=%d a positive multiple of %d", B, S, H,
                Smax, kv8::kBlock);
  if (S > 0x7fffffff - Smax) return fail(PREFIXLM_ERR_INVALID, "seqlen_q=%d is too large", S);
  const bool has_new = a->k != nullptr;
  if ((a->k == nullptr) != (a->v == nullptr)) return fail(PREFIXLM_ERR_INVALID, "k and v must be given together");
  if (!a->cache_seqlens && (a->cache_seqlen < 0 || a->cache_seqlen > Smax))
    return fail(PREFIXLM_ERR_INVALID, "cache_seqlen=%d outside [0, %d]", a->cache_seqlen, Smax);
  const void* ptrs[] = {a->q, a->k_codes, a->v_codes, a->k_scale, a->v_scale, a->k_recent, a->v_recent, a->out, a->k, a->v};
  for (int i = 0; i < (has_new ? 10 : 8); ++i)
    if (!ptrs[i] || (i == 3 || i == 4 ? (uintptr_t)ptrs[i] % 4 != 0 : !aligned16(ptrs[i])))
      return fail(PREFIXLM_ERR_INVALID, "tensor pointer %d is null or not aligned (16 bytes, scales 4)", i);
  const int64_t st[] = {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->out_stride_b, a->out_stride_s, a->out_stride_h,
                        a->k_stride_b, a->k_stride_s, a->k_stride_h, a->v_stride_b,   a->v_stride_s,   a->v_stride_h};
  for (int i = 0; i < (has_new ? 12 : 6); ++i)
    if (st[i] < 0 || st[i] % 8)
      return fail(PREFIXLM_ERR_INVALID, "stride %d (%lld) must be a non-negative multiple of 8", i, (long long)st[i]);
  const size_t need = prefixlm_kvcache8_workspace_size(B, S, H, Smax);
  if (need && (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need))
    return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes is null, unaligned or below %zu", a->workspace_bytes, need);

  kv8::Params P{};
  P.q = static_cast<const bf16*>(a->q);
  P.k = static_cast<const bf16*>(a->k);
  P.v = static_cast<const bf16*>(a->v);
  P.kc = static_cast<uint8_t*>(a->k_codes);
  P.vc = static_cast<uint8_t*>(a->v_codes);
  P.ks = a->k_scale;
  P.vs = a->v_scale;
  P.kr = static_cast<bf16*>(a->k_recent);
  P.vr = static_cast<bf16*>(a->v_recent);
  P.out = static_cast<bf16*>(a->out);
  P.part = static_cast<float*>(a->workspace);
  P.seqlens = a->cache_seqlens;
  P.q_sb = a->q_stride_b; P.q_ss = a->q_stride_s; P.q_sh = a->q_stride_h;
  P.k_sb = a->k_stride_b; P.k_ss = a->k_stride_s; P.k_sh = a->k_stride_h;
  P.v_sb = a->v_stride_b; P.v_ss = a->v_stride_s; P.v_sh = a->v_stride_h;
  P.o_sb = a->out_stride_b; P.o_ss = a->out_stride_s; P.o_sh = a->out_stride_h;
  P.B = B; P.S = S; P.H = H; P.Smax = Smax;
  P.nsplit = (int)kv8_nsplit(B, S, H, Smax);
  P.nqb = kv_nqb(S);
  P.causal = a->is_causal ? 1 : 0;
  P.seqlen_const = a->cache_seqlen;
  P.s_new = has_new ? S : 0;
  P.scale_log2 = a->softmax_scale * kLog2e;
  P.touched = (S + kv8::kBlock - 1) / kv8::kBlock;
  // the same queries, rows, lengths and partials, for the kernels shared with the bf16 cache
  kvc::Params Q{};
  Q.q = P.q; Q.k = P.k; Q.v = P.v; Q.out = P.out; Q.part = P.part; Q.seqlens = P.seqlens;
  Q.q_sb = P.q_sb; Q.q_ss = P.q_ss; Q.q_sh = P.q_sh;
  Q.k_sb = P.k_sb; Q.k_ss = P.k_ss; Q.k_sh = P.k_sh;
  Q.v_sb = P.v_sb; Q.v_ss = P.v_ss; Q.v_sh = P.v_sh;
  Q.o_sb = P.o_sb; Q.o_ss = P.o_ss; Q.o_sh = P.o_sh;
  Q.B = B; Q.S = S; Q.H = H; Q.Smax = Smax; Q.nsplit = P.nsplit;
  Q.causal = P.causal; Q.seqlen_const = P.seqlen_const; Q.s_new = P.s_new; Q.scale_log2 = P.scale_log2;

  const int64_t units = (int64_t)B * H * P.nsplit, nblk = S == 1 ? units : (units + 7) / 8 * 8 * P.nqb;
  const int64_t nappend = has_new ? 2 * (int64_t)B * H * P.touched : 0;
  // with rows of one block at most the attention's launch appends (see the kernel)
  const bool prefill = kv_prefills(Q), beside = S > 1 && S <= kv8::kBlock && !prefill;
  P.n_main = (int)std::min<int64_t>(nblk, 0x7fffffff);
  const int64_t waves = (int64_t)B * S * H;
  if (!launchable(nblk + nappend, 512) || !launchable((waves + 3) / 4, 256))
    return fail(PREFIXLM_ERR_INVALID, "grid too large");
  (void)hipGetLastError();
  if (prefill) {
    // the training forward, whose probabilities are rounded to bf16 (2^-9 of each, half the output's own
    // rounding): the extend kernel, which keeps their fp32 bits, takes twice as long (2 x 1021 rows x 16
    // heads 84 us, so 37; 4 x 4100 x 16 1298 and 625)
    set_kernel_attrs();
    if (g_attr_err != hipSuccess)
      return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(g_attr_err));
    const int rc = kv_prefill(Q, false, stream);
    if (rc) return rc;
  } else {
    const int rc = kv8_allow_lds();
    if (rc) return rc;
    if (a->code_int8)
      kv8_launch<kv8::Int8>(P, nblk + (beside ? nappend : 0), stream);
    else
      kv8_launch<kv8::E4M3>(P, nblk + (beside ? nappend : 0), stream);
    if (P.nsplit > 1)
      hipLaunchKernelGGL(kvc::combine_kernel<true>, dim3((unsigned)((waves * 64 + 255) / 256)), dim3(256), 0, stream, Q);
  }
  if (has_new && !beside && (S > 1 || prefill))
    hipLaunchKernelGGL(a->code_int8 ? kv8::append_kernel<kv8::Int8> : kv8::append_kernel<kv8::E4M3>,
                       dim3((unsigned)nappend), dim3(kv8::kAppendThreads), 0, stream, P, P.touched);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "8-bit kv-cache launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

}  // extern "C"

// ---- a cache in pages ------------------------------------------------------------------------
static int pool_check(const prefixlm_page_pool& p, bool contents) {
  if (p.head_dim != 64 && p.head_dim != 128) return fail(PREFIXLM_ERR_INVALID, "head_dim must be 64 or 128 (got %d)", p.head_dim);
  if (p.page_size < 16 || p.page_size > 1024 || (p.page_size & (p.page_size - 1)))
    return fail(PREFIXLM_ERR_INVALID, "page_size must be a power of two from 16 to 1024 (got %d)", p.page_size);
  if (p.layers < 1 || p.layers > 32767 || p.num_pages < 1 || p.num_kv_heads < 1 || p.batch < 1 || p.columns < 1)
    return fail(PREFIXLM_ERR_INVALID, "layers=%d (to 32767) num_pages=%d num_kv_heads=%d batch=%d columns=%d must be >= 1",
                p.layers, p.num_pages, p.num_kv_heads, p.batch, p.columns);
  if ((int64_t)p.columns * p.page_size > (1 << 30))
    return fail(PREFIXLM_ERR_INVALID, "columns=%d x page_size=%d exceeds 2^30 rows", p.columns, p.page_size);
  if ((int64_t)p.num_kv_heads * p.page_size * p.head_dim > (1 << 30))
    return fail(PREFIXLM_ERR_INVALID, "a page of %d heads x %d x %d exceeds 2^30 elements", p.num_kv_heads, p.page_size, p.head_dim);
  if (contents && (!p.k_pages || !p.v_pages || !aligned16(p.k_pages) || !aligned16(p.v_pages)))
    return fail(PREFIXLM_ERR_INVALID, "k_pages or v_pages is null or not 16-byte aligned");
  return PREFIXLM_OK;
}
static int table_check(const prefixlm_page_pool& p) {
  if (!p.refs || !p.page_table || (uintptr_t)p.refs % 4 || (uintptr_t)p.page_table % 4)
    return fail(PREFIXLM_ERR_INVALID, "refs or page_table is null or not 4-byte aligned");
  if (p.table_stride < p.columns)
    return fail(PREFIXLM_ERR_INVALID, "table_stride=%lld is below columns=%d", (long long)p.table_stride, p.columns);
  return PREFIXLM_OK;
}
static int log2_of(int x) { return 31 - __builtin_clz((unsigned)x); }

// R rows share a key-value head's keys. The rows of a block, which picks the kernel: one token of ungrouped heads alone;
// up to 16 (64 x 4 key-value heads of four on 2163-3972 rows 75 us, 80 without the matrix cores); blocks of 64 from 17
// on, most of which may be empty (24 x 4 heads, 20 rows, on 1729-3063 32 us; with 32 rows of 16 in the kernel for 16 it
// took 40 for 34 then); from 65 on 128, or 64 where these start all at once on 256 CUs, two a CU (three of 64 columns), and
// 128 would be one a CU: 4 x 16 heads x 509 rows on 1582-2028 84 us (128: 106), of 64 columns 52 (76); 3 x 16 74 (88); 6 x 16
// x 64 columns 71 (85). More or fewer: 6 x 16 130 by 64, 129 by 128; 5 x 16 123 and 116; 24 x 4 x 400 on 1437-2614 140 and
// 124; 2 x 16 64 and 61; 16 x 16 x 512 on 6053-6782 923 and 807. Only the call's sizes are known here: on few cached rows the
// blocks of 128, which are then cut, cost more than they save (16 heads x 900 rows on 119 41 us, 39 by 64).
static int pg_rows(int64_t B, int64_t Hkv, int64_t R, int D) {
  if (R <= 64) return R == 1 ? 1 : R <= 16 ? 16 : 64;
  if (B >= 512 || Hkv >= 512) return 128;
  const int64_t blocks = B * Hkv * ((R + 63) / 64);
  return blocks > 256 && blocks <= (D == 128 ? 512 : 768) ? 64 : 128;
}
// Keys of a tile
static int pg_tile(int rows, int D) { return rows == 1 ? (D == 128 ? 64 : 128) : rows == 16 ? 4 * pkv::kKeys : 64; }
// The workgroups that the units share, 0: one for each unit. Two a CU, three of the smaller ones for one row (3 x 12 heads
// on 20735-25651 rows 74 us with 768, 71 with 512, 73 with 1024), unless units are as good as enough, or their
// keys, as many as the table has room for, take less time than the combine's launch. One row, one workgroup of 512 threads a unit against 768 that
// share: 16 units of 512 rows 7.5 and 9.5 us, of 1024 11.6 and 9.9; 64 of 1024 13.7 and 14.6, of 1536 18.5 and 16.2;
// 128 of 1024 15.1 and 18.5; 256 of 2048 35.6 and 39. More rows: 16 units of 256 8.8 and 11.0, of 512 13.0 and 11.4; 128 of
// 512 14.6 and 15.3.
static int pg_nwg(int64_t B, int64_t Hkv, int64_t R, int D, int64_t cap) {
  if (B > pkv::kMaxShared || Hkv > 512) return 0;
  const int rows = pg_rows(B, Hkv, R, D), tile = pg_tile(rows, D), most = rows == 1 ? 768 : 512;
  const int64_t units = B * Hkv * ((R + rows - 1) / rows), tiles = units * ((cap + tile - 1) / tile);
  if (2 * units > most || tiles <= units || tiles > 0x7fffffff) return 0;   // the kernels add the tiles up in 32 bits
  if (rows == 1 ? cap <= 768 + 5 * units : cap <= 256 || (units >= 128 && cap <= 512)) return 0;
  return (int)std::min<int64_t>(most, tiles);
}
static size_t pg_workspace(int64_t B, int64_t Hkv, int64_t R, int D, int64_t cap) {
  const int n = pg_nwg(B, Hkv, R, D, cap);
  return n == 0 ? 0 : align_up(sizeof(int32_t) * (B + 1)) + align_up(sizeof(float) * (size_t)n * pg_rows(B, Hkv, R, D) * (D + 4));
}

template <int D>
static void pg_launch(const pkv::Params& P, unsigned nblk, hipStream_t stream) {
  const int64_t R = (int64_t)P.S * P.G;
  const dim3 g(nblk), n(pkv::NT), c((unsigned)((P.B * P.Hkv * R + 3) / 4));
  switch (pg_rows(P.B, P.Hkv, R, D)) {
    case 1:
      if (P.nwg)
        hipLaunchKernelGGL((pkv::decode_kernel<D, pkv::NT>), g, n, 0, stream, P);
      else
        hipLaunchKernelGGL((pkv::decode_kernel<D, 512>), g, dim3(512), 0, stream, P);
      if (P.nwg) hipLaunchKernelGGL((pkv::combine_kernel<D, 1>), c, n, 0, stream, P);
      break;
    case 16:
      hipLaunchKernelGGL((pkv::stream_kernel<D>), g, n, 0, stream, P);
      if (P.nwg) hipLaunchKernelGGL((pkv::combine_kernel<D, 16>), c, n, 0, stream, P);
      break;
    case 64:
      if (P.ps_log2 >= 6)
        hipLaunchKernelGGL((pkv::tile_kernel<D, 2, true>), g, n, (pkv::TileGeo<D, 2>::LDS_BYTES), stream, P);
      else
        hipLaunchKernelGGL((pkv::tile_kernel<D, 2, false>), g, n, (pkv::TileGeo<D, 2>::LDS_BYTES), stream, P);
      if (P.nwg) hipLaunchKernelGGL((pkv::combine_kernel<D, 64>), c, n, 0, stream, P);
      break;
    default:
      if (P.ps_log2 >= 6)
        hipLaunchKernelGGL((pkv::tile_kernel<D, 4, true>), g, n, (pkv::TileGeo<D, 4>::LDS_BYTES), stream, P);
      else
        hipLaunchKernelGGL((pkv::tile_kernel<D, 4, false>), g, n, (pkv::TileGeo<D, 4>::LDS_BYTES), stream, P);
      if (P.nwg) hipLaunchKernelGGL((pkv::combine_kernel<D, 128>), c, n, 0, stream, P);
  }
}
static_assert(pkv::TileGeo<64, 4>::LDS_BYTES <= 65536 && pkv::TileGeo<64, 2>::LDS_BYTES <= 65536, "within the default limit");
// The tiles of 128 columns, whose LDS is above the default limit, allowed once per device
static int pg_allow_lds() {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipGetDevice: %s", hipGetErrorString(e));
  if (dev < 0 || dev >= 64) return fail(PREFIXLM_ERR_INVALID, "device %d >= 64", dev);
  std::lock_guard<std::mutex> g(mu);
  if (done[dev]) return PREFIXLM_OK;
  static_assert(pkv::TileGeo<128, 2>::LDS_BYTES == pkv::TileGeo<128, 4>::LDS_BYTES);
  const void* const tiles[] = {
      reinterpret_cast<const void*>(&pkv::tile_kernel<128, 2, false>), reinterpret_cast<const void*>(&pkv::tile_kernel<128, 2, true>),
      reinterpret_cast<const void*>(&pkv::tile_kernel<128, 4, false>), reinterpret_cast<const void*>(&pkv::tile_kernel<128, 4, true>)};
  for (const void* f : tiles)
    if (e == hipSuccess) e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (pkv::TileGeo<128, 2>::LDS_BYTES));
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  done[dev] = true;
  return PREFIXLM_OK;
}

extern "C" {

size_t prefixlm_paged_workspace_size(int32_t batch, int32_t seqlen_q, int32_t num_heads, int32_t num_kv_heads,
                                     int32_t head_dim, int32_t page_size, int32_t columns) {
  if (batch < 1 || seqlen_q < 1 || num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads || head_dim < 1 ||
      page_size < 1 || columns < 1)
    return 0;
  const int64_t R = (int64_t)seqlen_q * (num_heads / num_kv_heads);
  return pg_workspace(batch, num_kv_heads, R, head_dim, (int64_t)columns * page_size);
}

int prefixlm_paged_fwd(const prefixlm_paged_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  const prefixlm_page_pool& pool = a->pool;
  int rc = pool_check(pool, true);
  if (!rc) rc = table_check(pool);
  if (rc) return rc;
  const int S = a->seqlen_q, cap = pool.columns * pool.page_size;
  if (S < 1 || S > 0x7fffffff - cap) return fail(PREFIXLM_ERR_INVALID, "seqlen_q=%d must be >= 1 and below 2^31 - %d", S, cap);
  if (a->num_heads < 1 || a->num_heads % pool.num_kv_heads)
    return fail(PREFIXLM_ERR_INVALID, "num_heads=%d must be a multiple of num_kv_heads=%d", a->num_heads, pool.num_kv_heads);
  if (a->layer < 0 || a->layer >= pool.layers)
    return fail(PREFIXLM_ERR_INVALID, "layer=%d outside [0, %d)", a->layer, pool.layers);
  const bool has_new = a->k != nullptr;
  if ((a->k == nullptr) != (a->v == nullptr)) return fail(PREFIXLM_ERR_INVALID, "k and v must be given together");
  const void* ptrs[] = {a->q, a->out, a->k, a->v};
  for (int i = 0; i < (has_new ? 4 : 2); ++i)
    if (!ptrs[i] || !aligned16(ptrs[i]))
      return fail(PREFIXLM_ERR_INVALID, "tensor pointer %d is null or not 16-byte aligned", i);
  const int64_t st[] = {a->q_stride_b, a->q_stride_s, a->q_stride_h, a->out_stride_b, a->out_stride_s, a->out_stride_h,
                        a->k_stride_b, a->k_stride_s, a->k_stride_h, a->v_stride_b,   a->v_stride_s,   a->v_stride_h};
  for (int i = 0; i < (has_new ? 12 : 6); ++i)
    if (st[i] < 0 || st[i] % 8)
      return fail(PREFIXLM_ERR_INVALID, "stride %d (%lld) must be a non-negative multiple of 8", i, (long long)st[i]);
  if (!a->cache_seqlens && (a->cache_seqlen < 0 || a->cache_seqlen > cap))
    return fail(PREFIXLM_ERR_INVALID, "cache_seqlen=%d outside [0, %d]", a->cache_seqlen, cap);
  const size_t need = prefixlm_paged_workspace_size(pool.batch, S, a->num_heads, pool.num_kv_heads, pool.head_dim,
                                                    pool.page_size, pool.columns);
  if (need && (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need))
    return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes is null, unaligned or below %zu", a->workspace_bytes, need);

  pkv::Params P{};
  const int64_t layer = (int64_t)pool.num_pages * pool.num_kv_heads * pool.page_size * pool.head_dim * a->layer;
  P.q = static_cast<const bf16*>(a->q);
  P.k = static_cast<const bf16*>(a->k);
  P.v = static_cast<const bf16*>(a->v);
  P.kp = static_cast<bf16*>(pool.k_pages) + layer;
  P.vp = static_cast<bf16*>(pool.v_pages) + layer;
  P.refs = pool.refs;
  P.table = pool.page_table;
  P.out = static_cast<bf16*>(a->out);
  P.part = static_cast<float*>(a->workspace);
  P.seqlens = a->cache_seqlens;
  P.q_sb = a->q_stride_b; P.q_ss = a->q_stride_s; P.q_sh = a->q_stride_h;
  P.k_sb = a->k_stride_b; P.k_ss = a->k_stride_s; P.k_sh = a->k_stride_h;
  P.v_sb = a->v_stride_b; P.v_ss = a->v_stride_s; P.v_sh = a->v_stride_h;
  P.o_sb = a->out_stride_b; P.o_ss = a->out_stride_s; P.o_sh = a->out_stride_h;
  P.table_sb = pool.table_stride;
  P.B = pool.batch; P.S = S; P.Hkv = pool.num_kv_heads; P.G = a->num_heads / pool.num_kv_heads;
  P.P = pool.num_pages; P.cap = cap; P.ps_log2 = log2_of(pool.page_size);
  P.causal = a->is_causal ? 1 : 0;
  P.seqlen_const = a->cache_seqlen;
  P.s_new = has_new ? S : 0;
  P.scale_log2 = a->softmax_scale * kLog2e;
  const int64_t R = (int64_t)S * P.G;
  if (R > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "seqlen_q=%d x %d heads of a group is too large", S, P.G);
  const int rows = pg_rows(P.B, P.Hkv, R, pool.head_dim);
  P.nrb = (int)((R + rows - 1) / rows);
  P.nwg = pg_nwg(P.B, P.Hkv, R, pool.head_dim, cap);
  P.pre = static_cast<int32_t*>(a->workspace);
  P.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + align_up(sizeof(int32_t) * ((size_t)P.B + 1)));
  // pieces and their join are few; without them the first launch is the only one
  const int64_t units = (int64_t)P.B * P.Hkv, eighths = (units + 7) / 8 * 8;
  if (!P.nwg && (units > 0x7ffffff0 || P.nrb > 0x7fffffff / eighths || !launchable(eighths * P.nrb, rows == 1 ? 512 : pkv::NT)))
    return fail(PREFIXLM_ERR_INVALID, "grid too large");
  const int64_t nblk = P.nwg ? P.nwg : eighths * P.nrb;
  rc = pg_allow_lds();
  if (rc) return rc;
  (void)hipGetLastError();
  if (pool.head_dim == 128)
    pg_launch<128>(P, (unsigned)nblk, stream);
  else
    pg_launch<64>(P, (unsigned)nblk, stream);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "paged kv-cache launch: %s", hipGetErrorString(e));
  return PREFIXLM_OK;
}

}  // extern "C"

// Workspace of reserve: free pages, three words a page, copies; of compact: moves, targets
static size_t pages_free_words(const prefixlm_page_pool& p) {
  return (size_t)std::min<int64_t>(p.num_pages, (int64_t)p.batch * p.columns);
}
static int pages_check(const prefixlm_pages_args* a, bool contents, bool workspace) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  int rc = pool_check(a->pool, contents);
  if (!rc) rc = table_check(a->pool);
  if (rc) return rc;
  if (workspace) {
    const size_t need = prefixlm_pages_workspace_size(&a->pool);
    if (!a->workspace || !aligned16(a->workspace) || a->workspace_bytes < need)
      return fail(PREFIXLM_ERR_INVALID, "workspace of %zu bytes is null, unaligned or below %zu", a->workspace_bytes, need);
    if (!a->result || (uintptr_t)a->result % 4) return fail(PREFIXLM_ERR_INVALID, "result is null or not 4-byte aligned");
  }
  return PREFIXLM_OK;
}
static int pages_end(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(PREFIXLM_ERR_HIP, "%s launch: %s", what, hipGetErrorString(e));
  return PREFIXLM_OK;
}
// What all copies of a pool share. by_head: pairs bring rows, else whole pages move.
static pages::CopyParams pages_copy(const prefixlm_page_pool& to, const prefixlm_page_pool& from, bool by_head) {
  pages::CopyParams C{};
  const int64_t page = (int64_t)to.num_kv_heads * to.page_size * to.head_dim;
  C.from[0] = static_cast<const bf16*>(from.k_pages);
  C.from[1] = static_cast<const bf16*>(from.v_pages);
  C.to[0] = static_cast<bf16*>(to.k_pages);
  C.to[1] = static_cast<bf16*>(to.v_pages);
  C.from_layer = page * from.num_pages;
  C.to_layer = page * to.num_pages;
  C.P_from = from.num_pages;
  C.P_to = to.num_pages;
  C.heads = by_head ? to.num_kv_heads : 1;
  C.head_elems = (int)(page / C.heads);
  C.row_elems = to.head_dim;
  C.rows = by_head;
  C.pieces = (C.head_elems + 2047) / 2048;
  return C;
}
// Workgroups of a copy of up to n pairs: eight for each CU over all layers, or what there is to do
static int pages_copy_grid(const pages::CopyParams& C, int64_t n, int layers, dim3* grid) {
  const int64_t most = (int64_t)C.heads * C.pieces;   // waves of a pair
  if (n > 0x7fffffff / most) return fail(PREFIXLM_ERR_INVALID, "too many pages to copy in one call");
  int cus = 0;
  const int rc = persistent_grid(&cus);
  if (rc) return rc;
  const int64_t x = std::min<int64_t>((n * most + 3) / 4, (8 * (int64_t)cus + 2 * layers - 1) / (2 * layers));
  *grid = dim3((unsigned)(std::max<int64_t>(1, x) + C.n_remap), (unsigned)(2 * layers));
  return PREFIXLM_OK;
}

extern "C" {

size_t prefixlm_pages_workspace_size(const prefixlm_page_pool* p) {
  if (!p || p->num_pages < 1 || p->batch < 1 || p->columns < 1) return 0;
  const size_t reserve = pages_free_words(*p) + 3 * (size_t)p->num_pages + 1 + 3 * (size_t)p->batch;
  const size_t compact = 1 + 2 * (size_t)p->num_pages;
  return align_up(sizeof(int32_t) * std::max(reserve, compact));
}

int prefixlm_pages_reserve(const prefixlm_pages_args* a, void* stream_) {
  const int rc = pages_check(a, true, true);
  if (rc) return rc;
  const prefixlm_page_pool& p = a->pool;
  if (p.batch > pages::kMaxSeqs) return fail(PREFIXLM_ERR_INVALID, "batch=%d exceeds %d", p.batch, pages::kMaxSeqs);
  if ((int64_t)p.batch * p.columns > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "a table of %d x %d is too large", p.batch, p.columns);
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  pages::ReserveParams P{};
  P.refs = p.refs;
  P.table = p.page_table;
  P.seqlens = a->rows;
  P.new_rows = a->new_rows;
  P.short_ = a->result;
  P.free_list = static_cast<int32_t*>(a->workspace);
  P.was = P.free_list + pages_free_words(p);
  P.copies = P.was + 3 * (size_t)p.num_pages;
  P.table_sb = p.table_stride;
  P.N = p.batch; P.M = p.columns; P.P = p.num_pages; P.ps_log2 = log2_of(p.page_size);
  P.seqlen_const = a->row_const;
  P.new_const = a->new_row_const;
  pages::CopyParams C = pages_copy(p, p, true);
  C.src = P.copies + 1;
  C.count = P.copies;
  dim3 grid;
  const int rc2 = pages_copy_grid(C, p.batch, p.layers, &grid);   // a sequence's first column alone has rows to be copied
  if (rc2) return rc2;
  (void)hipGetLastError();
  hipLaunchKernelGGL(pages::reserve_kernel, dim3(1), dim3(pages::NTH), 0, stream, P);
  hipLaunchKernelGGL(pages::copy_kernel, grid, dim3(256), 0, stream, C);
  return pages_end("page reserve");
}

int prefixlm_pages_fork(const prefixlm_pages_args* a, void* stream_) {
  const int rc = pages_check(a, false, false);
  if (rc) return rc;
  const prefixlm_page_pool& p = a->pool;
  if (p.batch > pages::kMaxSeqs) return fail(PREFIXLM_ERR_INVALID, "batch=%d exceeds %d", p.batch, pages::kMaxSeqs);
  if (!a->src || (uintptr_t)a->src % 4) return fail(PREFIXLM_ERR_INVALID, "src is null or not 4-byte aligned");
  pages::ForkParams P{};
  P.refs = p.refs;
  P.table = p.page_table;
  P.parents = a->src;
  P.table_sb = p.table_stride;
  P.N = p.batch; P.M = p.columns; P.P = p.num_pages;
  // 64 KB of LDS; as many columns a workgroup as a launch of a very wide table takes
  P.TC = std::min(p.batch <= 1024 ? 16 : p.batch <= 2048 ? 8 : p.batch <= 4096 ? 4 : 2, p.columns);
  auto nblk = [&] { return ((int64_t)p.columns + P.TC - 1) / P.TC; };
  while (!launchable(nblk(), pages::NTH) && 2 * P.TC * p.batch <= 16384) P.TC *= 2;
  if (!launchable(nblk(), pages::NTH)) return fail(PREFIXLM_ERR_INVALID, "a table of %d x %d is too large", p.batch, p.columns);
  (void)hipGetLastError();
  hipLaunchKernelGGL(pages::fork_kernel, dim3((unsigned)nblk()), dim3(pages::NTH), sizeof(int32_t) * P.N * P.TC,
                     reinterpret_cast<hipStream_t>(stream_), P);
  return pages_end("page fork");
}

int prefixlm_pages_free(const prefixlm_pages_args* a, void* stream_) {
  const int rc = pages_check(a, false, false);
  if (rc) return rc;
  const prefixlm_page_pool& p = a->pool;
  pages::FreeParams P{};
  P.refs = p.refs;
  P.table = p.page_table;
  P.keep = a->rows;
  P.keep_const = a->row_const;
  P.table_sb = p.table_stride;
  P.N = p.batch; P.M = p.columns; P.P = p.num_pages; P.ps_log2 = log2_of(p.page_size);
  const int64_t nblk = ((int64_t)P.N * P.M + 255) / 256;
  if (!launchable(nblk, 256)) return fail(PREFIXLM_ERR_INVALID, "a table of %d x %d is too large", P.N, P.M);
  (void)hipGetLastError();
  hipLaunchKernelGGL(pages::free_kernel, dim3((unsigned)nblk), dim3(256), 0, reinterpret_cast<hipStream_t>(stream_), P);
  return pages_end("page free");
}

int prefixlm_pages_compact(const prefixlm_pages_args* a, void* stream_) {
  const int rc = pages_check(a, true, true);
  if (rc) return rc;
  const prefixlm_page_pool& p = a->pool;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_);
  pages::CompactParams P{};
  P.refs = p.refs;
  P.table = p.page_table;
  P.used = a->result;
  P.moves = static_cast<int32_t*>(a->workspace);
  P.to = P.moves + 1 + p.num_pages;
  P.table_sb = p.table_stride;
  P.N = p.batch; P.M = p.columns; P.P = p.num_pages;
  pages::CopyParams C = pages_copy(p, p, false);
  // the moves' targets come first, then as many sources; how many, the kernel before this one knows
  C.dst = P.moves + 1;
  C.src = nullptr;
  C.count = P.moves;
  C.table = p.page_table;
  C.to_page = P.to;
  C.used = a->result;
  C.table_sb = p.table_stride;
  C.N = p.batch; C.M = p.columns;
  C.n_remap = (int)std::min<int64_t>(64, ((int64_t)C.N * C.M + 1023) / 1024);
  dim3 grid;
  const int rc2 = pages_copy_grid(C, p.num_pages / 2, p.layers, &grid);
  if (rc2) return rc2;
  (void)hipGetLastError();
  hipLaunchKernelGGL(pages::compact_kernel, dim3(1), dim3(pages::NTH), 0, stream, P);
  hipLaunchKernelGGL(pages::copy_kernel, grid, dim3(256), 0, stream, C);
  return pages_end("page compact");
}

int prefixlm_pages_copy(const prefixlm_pages_args* a, void* stream_) {
  if (!a) return fail(PREFIXLM_ERR_INVALID, "args is null");
  const prefixlm_page_pool &to = a->pool, &from = a->from ? *a->from : a->pool;
  int rc = pool_check(to, true);
  if (!rc) rc = pool_check(from, true);
  if (rc) return rc;
  if (to.layers != from.layers || to.num_kv_heads != from.num_kv_heads || to.page_size != from.page_size || to.head_dim != from.head_dim)
    return fail(PREFIXLM_ERR_INVALID, "the pools' layers, heads, page_size or head_dim differ");
  if (a->n < 0 || a->n > 0x7fffffff) return fail(PREFIXLM_ERR_INVALID, "n=%lld is negative or too large", (long long)a->n);
  if (a->n == 0) return PREFIXLM_OK;
  if (!a->src || !a->dst || (uintptr_t)a->src % 4 || (uintptr_t)a->dst % 4)
    return fail(PREFIXLM_ERR_INVALID, "src or dst is null or not 4-byte aligned");
  pages::CopyParams C = pages_copy(to, from, false);
  C.src = a->src;
  C.dst = a->dst;
  C.n = (int)a->n;
  dim3 grid;
  rc = pages_copy_grid(C, a->n, to.layers, &grid);
  if (rc) return rc;
  (void)hipGetLastError();
  hipLaunchKernelGGL(pages::copy_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream_), C);
  return pages_end("page copy");
}

}  // extern "C"
