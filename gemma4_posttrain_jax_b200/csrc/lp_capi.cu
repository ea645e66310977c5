// C ABI of liblp_b200.so (declared in include/lp_logprob.h): argument checks, tensor-map
// construction, tile planning and kernel launches. No torch or Python types cross it.
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/lp_logprob.h"
#include "lp_gemm.cuh"
#include "lp_dist_kernels.cuh"
#include "lp_plan.cuh"
#include "lp_small_kernels.cuh"

namespace {

using namespace lpk;

thread_local std::string g_last_error;
std::atomic<long long> g_launches{0};

// Optional per-kernel timing: CUDA events recorded on the launching stream around every
// kernel this library launches, summed per kernel name by lp_profile_read().
struct ProfRecord {
  const char* tag;
  cudaEvent_t start, stop;
};
std::mutex g_prof_mu;
bool g_prof_on = false;
std::vector<ProfRecord> g_prof_records;
std::vector<cudaEvent_t> g_prof_pool;

cudaEvent_t prof_event() {
  if (!g_prof_pool.empty()) {
    cudaEvent_t e = g_prof_pool.back();
    g_prof_pool.pop_back();
    return e;
  }
  cudaEvent_t e = nullptr;
  cudaEventCreate(&e);
  return e;
}

struct ProfScope {
  cudaStream_t st;
  const char* tag;
  cudaEvent_t start = nullptr;
  ProfScope(cudaStream_t s, const char* t) : st(s), tag(t) {
    std::lock_guard<std::mutex> lk(g_prof_mu);
    if (g_prof_on) {
      start = prof_event();
      cudaEventRecord(start, st);
    }
  }
  ~ProfScope() {
    if (start == nullptr) return;
    std::lock_guard<std::mutex> lk(g_prof_mu);
    cudaEvent_t stop = prof_event();
    cudaEventRecord(stop, st);
    g_prof_records.push_back({tag, start, stop});
  }
};

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_last_error = buf;
  return code;
}

#define LP_CUDA_TRY(expr)                                                                   \
  do {                                                                                      \
    cudaError_t e_ = (expr);                                                                \
    if (e_ != cudaSuccess) return fail(LP_ECUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)

#define LP_LAUNCH_CHECK(name)                                                                  \
  do {                                                                                         \
    cudaError_t e_ = cudaGetLastError();                                                       \
    if (e_ != cudaSuccess) return fail(LP_ECUDA, "launch %s: %s", name, cudaGetErrorString(e_)); \
    g_launches.fetch_add(1, std::memory_order_relaxed);                                        \
  } while (0)

constexpr int kMaxDevices = 64;

// Tensor-core CTA group of the GEMMs: 2 = CTA pairs with 256x256 tiles, 1 = single CTAs with
// 128x256 tiles. By default each GEMM uses the group that measured faster for it;
// LP_B200_CTA_GROUP=1|2 or lp_set_cta_group(1|2) forces one group for every GEMM.
// 0 = per-GEMM default (below); 1 / 2 = force every GEMM to that CTA group.
// Optional pipeline counters of the GEMM kernels (a tuning aid): one 8-counter block per CTA
// and per GEMM kind, allocated on the first lp_debug_enable(1) of a device.
constexpr int kDbgKinds = 5;  // fwd, dz, dh, dw, other
std::atomic<bool> g_dbg_on{false};
unsigned long long* g_dbg_buf[kMaxDevices] = {};
int dbg_kind(const char* tag) {
  if (!strcmp(tag, "fwd_lse_gemm")) return 0;
  if (!strcmp(tag, "bwd_dz_gemm")) return 1;
  if (!strcmp(tag, "bwd_dh_gemm")) return 2;
  if (!strcmp(tag, "bwd_dw_gemm")) return 3;
  return 4;
}
unsigned long long* dbg_ptr(const char* tag) {
  if (!g_dbg_on.load()) return nullptr;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices || g_dbg_buf[dev] == nullptr) return nullptr;
  return g_dbg_buf[dev] + (size_t)dbg_kind(tag) * 256 * 8;
}

std::atomic<int> g_cg{-1};

int forced_cta_group() {
  int v = g_cg.load();
  if (v < 0) {
    const char* e = getenv("LP_B200_CTA_GROUP");
    v = (e != nullptr && (e[0] == '1' || e[0] == '2')) ? e[0] - '0' : 0;
    g_cg.store(v);
  }
  return v;
}

// CTA group per GEMM. A pair's 256x256 tile takes a third less operand data from L2 per FLOP
// than two single-CTA 128x256 tiles, and at the 1 kW power cap the energy saved comes back as
// SM clock. With one multicast commit per K block the pair's MMA issue is as fast as a single
// CTA's (forward: 659 vs 652 cycles per K block); a whole config-2 step with every GEMM as
// pairs measured fastest, although the dZ recompute alone is ~2 % faster as single CTAs.
// The sampler head (a few decode rows) and the generic GEMM hook use single CTAs.
enum CgUse { CG_FWD, CG_DZ, CG_DH, CG_DW, CG_HOOK, CG_HEAD };
int cta_group_for(CgUse k) {
  const int f = forced_cta_group();
  if (f) return f;
  // tuning: LP_B200_CG_PER_GEMM="fzhw" (four digits 1 / 2: forward, dZ, dH, dW)
  static const char* per = getenv("LP_B200_CG_PER_GEMM");
  if (per != nullptr && k < CG_HOOK && (int)strlen(per) >= 4 && (per[k] == '1' || per[k] == '2')) return per[k] - '0';
  return (k == CG_HOOK || k == CG_HEAD) ? 1 : 2;
}
int cta_group() { return forced_cta_group(); }

// The dW GEMM's K is the chunk's token count. With few tokens (e.g. T = 256) each tile is a
// few K blocks and the pair's cross-SM hand-offs (both CTAs' loads, both epilogues) are not
// amortised: single CTAs measured faster there (T = 256: 0.35 vs 0.43 ms, the bf16 dW stores
// at 0.86 of the write-only HBM bandwidth), pairs faster at thousands of tokens.
int cta_group_dw(int64_t k_tokens) {
  const int cg = cta_group_for(CG_DW);
  if (forced_cta_group() != 0 || getenv("LP_B200_CG_PER_GEMM") != nullptr) return cg;
  return k_tokens <= 1024 ? 1 : cg;
}

struct DeviceInfo {
  int sms = 0;
  int major = 0, minor = 0;
  int pairs = 0;  // CTA pairs of the pair GEMMs that can be resident at once
  bool ready = false;
};

// Persistent workers of a launch: SMs for CG = 1, co-resident CTA pairs for CG = 2.
// LP_B200_MAX_CTAS caps the CTAs of a GEMM launch (a tuning aid: fewer SMs share L2 / HBM).
int workers(const DeviceInfo* di, int cg) {
  static const int cap = [] {
    const char* e = getenv("LP_B200_MAX_CTAS");
    return (e != nullptr && atoi(e) > 0) ? atoi(e) : 0;
  }();
  const int w = cg == 1 ? di->sms : di->pairs;
  return cap > 0 ? std::max(1, std::min(w, cap / cg)) : w;
}
DeviceInfo g_dev[kMaxDevices];
std::mutex g_dev_mu;

// How many 2-CTA clusters of the largest pair GEMM (most shared memory) fit on the GPU at
// once; the persistent pair kernels launch at most this many pairs.
int max_resident_pairs(int sms, int* pairs) {
  auto kern = tc_gemm_kernel<2, EPI_BWD_DZ, false, false, true>;
  constexpr int smem = gemm_smem_bytes<2, EPI_BWD_DZ>();
  LP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sms, 1, 1);
  cfg.blockDim = dim3(NUM_THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  LP_CUDA_TRY(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
  *pairs = std::max(1, std::min(n, sms / 2));
  return LP_OK;
}

// Host-visible device error codes: one int per device in mapped, pinned host memory, which
// kernels write (besides g_lp_device_error) when they record an error. Reading a slot is a
// plain host load, so callers can check for errors at points where they already wait for
// the GPU without another synchronisation.
int* g_host_errors = nullptr;  // [kMaxDevices], allocated on the first device set-up

int setup_host_error_mirror(int dev) {
  if (g_host_errors == nullptr) {
    void* p = nullptr;
    LP_CUDA_TRY(cudaHostAlloc(&p, kMaxDevices * sizeof(int), cudaHostAllocMapped | cudaHostAllocPortable));
    std::memset(p, 0, kMaxDevices * sizeof(int));
    g_host_errors = static_cast<int*>(p);
  }
  int* dptr = nullptr;
  LP_CUDA_TRY(cudaHostGetDevicePointer(reinterpret_cast<void**>(&dptr), g_host_errors + dev, 0));
  LP_CUDA_TRY(cudaMemcpyToSymbol(g_lp_host_error, &dptr, sizeof(dptr)));
  return LP_OK;
}

int current_device_info(DeviceInfo** out) {
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(LP_EINVAL, "device ordinal %d out of range", dev);
  // a thread that has made no runtime call yet (one of autograd's, say) has a current device but no
  // context, which the driver's tensor-map encoder needs
  static thread_local int bound = -1;
  if (bound != dev) {
    LP_CUDA_TRY(cudaSetDevice(dev));
    bound = dev;
  }
  std::lock_guard<std::mutex> lk(g_dev_mu);
  DeviceInfo& d = g_dev[dev];
  if (!d.ready) {
    LP_CUDA_TRY(cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev));
    LP_CUDA_TRY(cudaDeviceGetAttribute(&d.major, cudaDevAttrComputeCapabilityMajor, dev));
    LP_CUDA_TRY(cudaDeviceGetAttribute(&d.minor, cudaDevAttrComputeCapabilityMinor, dev));
    d.pairs = d.sms / 2;
    if (d.major == 10 && d.minor == 0) {
      int rc = max_resident_pairs(d.sms, &d.pairs);
      if (rc) return rc;
      if ((rc = setup_host_error_mirror(dev))) return rc;
    }
    d.ready = true;
  }
  if (d.major != 10 || d.minor != 0)
    return fail(LP_EUNSUPPORTED, "liblp_b200 needs an sm_100 (B200) device, device %d is sm_%d%d", dev, d.major,
                d.minor);
  *out = &d;
  return LP_OK;
}

// --------------------------------------------------------------------------- tensor maps
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// 2-D tiled map, 128-byte swizzle, zero fill out of bounds. `inner`/`outer` in elements,
// `row_bytes` = byte stride between outer rows.
int make_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, int esize, uint64_t inner, uint64_t outer,
             uint64_t row_bytes, uint32_t box_inner, uint32_t box_outer, const char* what,
             CUtensorMapSwizzle swz = CU_TENSOR_MAP_SWIZZLE_128B) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(LP_ECUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  if (inner == 0 || outer == 0) return fail(LP_EINVAL, "%s: empty tensor", what);
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0) return fail(LP_EINVAL, "%s: base pointer not 16-byte aligned", what);
  if (row_bytes % 16 != 0) return fail(LP_EINVAL, "%s: row stride %llu bytes not a multiple of 16", what,
                                       (unsigned long long)row_bytes);
  if (row_bytes < inner * (uint64_t)esize) return fail(LP_EINVAL, "%s: row stride smaller than a row", what);
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {row_bytes};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(m, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swz,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(LP_ECUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return LP_OK;
}

int map_bf16(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint64_t ld_elems, uint32_t bi,
             uint32_t bo, const char* what) {
  return make_map(m, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, inner, outer, ld_elems * 2, bi, bo, what);
}

// MN-major bf16 operand [k_extent rows][mn_extent columns] (row stride ld_elems) as a 3-D
// map: dims (64 columns, K rows, mn_extent / 64 column chunks), box (64, 64, chunks), 128-byte
// swizzle. One box lands in shared memory as `chunks` consecutive 8 KB [64 K rows x 128 B]
// blocks, the layout of `chunks` 2-D 64x64 boxes side by side. Only for mn_extent % 64 == 0,
// so the box never reaches past the tensor.
int map_mn3d(CUtensorMap* m, const void* base, uint64_t mn_extent, uint64_t k_extent, uint64_t ld_elems,
             uint32_t chunks, const char* what) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(LP_ECUDA, "cuTensorMapEncodeTiled unavailable from the driver");
  if (mn_extent % 64 != 0 || k_extent == 0) return fail(LP_EINVAL, "%s: 3-D map needs 64-column chunks", what);
  if ((reinterpret_cast<uintptr_t>(base) & 15) != 0) return fail(LP_EINVAL, "%s: base pointer not 16-byte aligned", what);
  if ((ld_elems * 2) % 16 != 0 || ld_elems < mn_extent) return fail(LP_EINVAL, "%s: bad row stride", what);
  cuuint64_t dims[3] = {64, k_extent, mn_extent / 64};
  cuuint64_t strides[2] = {ld_elems * 2, 128};
  cuuint32_t box[3] = {64, 64, chunks};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(LP_ECUDA, "%s: cuTensorMapEncodeTiled (3-D) failed (%d)", what, (int)r);
  return LP_OK;
}

// 3-D MN-major operand maps (LP_B200_MN3D=0 keeps the per-chunk 2-D boxes, for tuning).
bool mn3d_enabled() {
  static const bool on = [] {
    const char* e = getenv("LP_B200_MN3D");
    return !(e != nullptr && e[0] == '0');
  }();
  return on;
}

// Epilogue store targets: one 32-row box per warp and piece, rows of `box_row_bytes` (64 or
// 128, the store_row_bytes of the GEMM) with the swizzle of that width, matching the staging
// layout of the GEMM epilogue.
int map_store_bf16(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint64_t ld_elems,
                   const char* what, int box_row_bytes = 64) {
  return make_map(m, base, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, inner, outer, ld_elems * 2, box_row_bytes / 2, 32,
                  what, box_row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}
int map_store_f32(CUtensorMap* m, const void* base, uint64_t inner, uint64_t outer, uint64_t ld_elems,
                  const char* what, int box_row_bytes = 64) {
  return make_map(m, base, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, inner, outer, ld_elems * 4, box_row_bytes / 4, 32,
                  what, box_row_bytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B);
}

// store_row_bytes of the plain-store GEMM (EPI_STORE) at CTA group cg.
int store_box_bytes(int cg) { return cg == 2 ? store_row_bytes<2, EPI_STORE>() : store_row_bytes<1, EPI_STORE>(); }

// Planning (tile plans, split-K, backward token chunks, workspace layout): lp_plan.cuh.

// --------------------------------------------------------------------------- launches
}  // namespace

// Work-unit counters of the GEMM kernels (each launch claims its units with atomicAdd on
// one slot). Slots rotate so that launches in flight on different streams use different
// counters; a launch zeroes its slot on its own stream just before it starts.
constexpr int kSchedSlots = 4096;
static __device__ unsigned int g_lp_sched[kSchedSlots];

namespace {

unsigned int* g_sched_ptr[kMaxDevices] = {};
std::mutex g_sched_mu;
std::atomic<unsigned> g_sched_next{0};

int sched_slot(cudaStream_t st, unsigned int** out) {
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(LP_EINVAL, "device ordinal %d out of range", dev);
  unsigned int* base;
  {
    std::lock_guard<std::mutex> lk(g_sched_mu);
    if (g_sched_ptr[dev] == nullptr) {
      void* p = nullptr;
      const cudaError_t e = cudaGetSymbolAddress(&p, g_lp_sched);
      if (e != cudaSuccess || p == nullptr)
        return fail(LP_ECUDA, "cudaGetSymbolAddress(work counters) on device %d: %s", dev, cudaGetErrorString(e));
      g_sched_ptr[dev] = static_cast<unsigned int*>(p);
    }
    base = g_sched_ptr[dev];
  }
  unsigned int* slot = base + g_sched_next.fetch_add(1u) % kSchedSlots;
  LP_CUDA_TRY(cudaMemsetAsync(slot, 0, sizeof(unsigned int), st));
  *out = slot;
  return LP_OK;
}

template <int CG, int EPI, bool A_MN, bool B_MN, bool CAP>
int launch_gemm_cg(cudaStream_t st, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o,
                   const GemmParams& p, const DeviceInfo* di, const char* tag) {
  auto kern = tc_gemm_kernel<CG, EPI, A_MN, B_MN, CAP>;
  constexpr int smem = gemm_smem_bytes<CG, EPI>();
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured[dev]) {
    LP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (CG == 2) LP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 0));
    configured[dev] = true;
  }
  const int grid = CG * std::max(1, std::min(p.s.num_units, workers(di, CG)));
  GemmParams pp = p;
  pp.dbg = dbg_ptr(tag);
  // A caller that keeps a counter of its own (in its workspace) passes it in. A single M tile's units
  // are alike and share no operand but its few rows, so workers take them in turn: no counter, and no
  // memset before the launch (1 row x 262144 x 2048, the whole top-20 call: 192.2 us, with a counter 193.8).
  if (pp.sched == nullptr) {
    if (int rc = sched_slot(st, &pp.sched)) return rc;
  } else if (p.s.num_units * CG <= grid || (p.s.tiles_m == 1 && p.s.k_splits == 1)) {
    pp.sched = nullptr;
  } else {
    LP_CUDA_TRY(cudaMemsetAsync(pp.sched, 0, sizeof(unsigned), st));
  }
  ProfScope prof(st, tag);
  if constexpr (CG == 1) {
    kern<<<grid, num_threads<EPI>(), smem, st>>>(a, b, o, pp);
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(num_threads<EPI>(), 1, 1);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LP_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, b, o, pp));
  }
  LP_LAUNCH_CHECK("tc_gemm_kernel");
  return LP_OK;
}

template <int EPI, bool A_MN, bool B_MN, bool CAP>
int launch_gemm(cudaStream_t st, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o,
                const GemmParams& p, const DeviceInfo* di, const char* tag) {
  return p.s.bm == 256 ? launch_gemm_cg<2, EPI, A_MN, B_MN, CAP>(st, a, b, o, p, di, tag)
                       : launch_gemm_cg<1, EPI, A_MN, B_MN, CAP>(st, a, b, o, p, di, tag);
}

template <int EPI, bool A_MN, bool B_MN>
int launch_gemm_cap(bool cap, cudaStream_t st, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o,
                    const GemmParams& p, const DeviceInfo* di, const char* tag) {
  return cap ? launch_gemm<EPI, A_MN, B_MN, true>(st, a, b, o, p, di, tag)
             : launch_gemm<EPI, A_MN, B_MN, false>(st, a, b, o, p, di, tag);
}

// L2 eviction priorities of the A / B loads of each GEMM (0 normal = plain load,
// 1 evict_first, 2 evict_last). Measured (ncu DRAM bytes per launch at the config-2 size):
// plain loads keep the forward and the dZ recompute near their algorithmic traffic;
// evict_first on an operand that concurrent CTAs share (W) multiplies HBM reads, and an
// explicit evict_normal policy is not the same as no hint. With the dynamic scheduler the
// dW GEMM is also faster with plain loads than with evict_last on its H chunk (715 vs 734
// cycles per K block, pipeline counters). LP_B200_L2HINTS="fA fB zA zB hA hB wA wB"
// (8 digits: forward, dZ recompute, dH, dW) overrides them for tuning.
enum GemmKind { G_FWD = 0, G_DZ = 1, G_DH = 2, G_DW = 3 };
int l2_hint(GemmKind k, int operand) {
  static int table[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  static std::once_flag once;
  std::call_once(once, [] {
    const char* e = getenv("LP_B200_L2HINTS");
    if (e == nullptr) return;
    int i = 0;
    for (const char* c = e; *c && i < 8; ++c)
      if (*c >= '0' && *c <= '2') table[i++] = *c - '0';
  });
  return table[2 * (int)k + operand];
}

void set_hints(GemmParams& p, GemmKind k) {
  p.e.a_l2 = l2_hint(k, 0);
  p.e.b_l2 = l2_hint(k, 1);
}

// Box height of a K-major B operand: the rows of B one CTA stages.
uint32_t b_box_rows(int cg) { return (uint32_t)(BN / cg); }

int check_common(const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs, const int32_t* y) {
  if (T < 0 || d <= 0 || Vs <= 0) return fail(LP_EINVAL, "bad sizes T=%lld d=%lld Vs=%lld", (long long)T, (long long)d,
                                               (long long)Vs);
  if (T > (int64_t)1 << 30 || Vs > (int64_t)1 << 30) return fail(LP_EINVAL, "T or Vs above 2^30");
  if (d % 8 != 0) return fail(LP_EINVAL, "hidden size d=%lld must be a multiple of 8", (long long)d);
  if (ldh < d || ldh % 8 != 0) return fail(LP_EINVAL, "ldh=%lld must be >= d and a multiple of 8", (long long)ldh);
  if (T > 0 && (H == nullptr || y == nullptr)) return fail(LP_EINVAL, "null hidden or targets");
  if (W == nullptr) return fail(LP_EINVAL, "null embedding");
  return LP_OK;
}

// Few rows for many partials: the forward's finalize runs one block per row instead of one
// thread per row (fewer rows than fill the GPU with 256-row blocks).
bool few_rows(int64_t T, const DeviceInfo* di) { return cdiv(T, 256) < di->sms; }

}  // namespace

// ============================================================================= C ABI
extern "C" {

int lp_version(void) { return 100; }

const char* lp_last_error(void) { return g_last_error.c_str(); }

long long lp_launch_count(void) { return g_launches.load(); }

int lp_debug_enable(int on) {
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(LP_EINVAL, "device ordinal out of range");
  if (on && g_dbg_buf[dev] == nullptr) {
    LP_CUDA_TRY(cudaMalloc(&g_dbg_buf[dev], (size_t)kDbgKinds * 256 * 8 * sizeof(unsigned long long)));
  }
  if (g_dbg_buf[dev] != nullptr)
    LP_CUDA_TRY(cudaMemset(g_dbg_buf[dev], 0, (size_t)kDbgKinds * 256 * 8 * sizeof(unsigned long long)));
  g_dbg_on.store(on != 0);
  return LP_OK;
}

int lp_debug_read(unsigned long long* out) {
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (out == nullptr) return fail(LP_EINVAL, "null out");
  if (dev < 0 || dev >= kMaxDevices || g_dbg_buf[dev] == nullptr) return fail(LP_EINVAL, "debug counters not enabled");
  std::vector<unsigned long long> h((size_t)kDbgKinds * 256 * 8);
  LP_CUDA_TRY(cudaMemcpy(h.data(), g_dbg_buf[dev], h.size() * sizeof(unsigned long long), cudaMemcpyDeviceToHost));
  for (int k = 0; k < kDbgKinds; ++k)
    for (int i = 0; i < 8; ++i) {
      unsigned long long t = 0;
      for (int c = 0; c < 256; ++c) t += h[((size_t)k * 256 + c) * 8 + i];
      out[k * 8 + i] = t;
    }
  return LP_OK;
}

int lp_device_pairs(void) {
  DeviceInfo* di = nullptr;
  return current_device_info(&di) == LP_OK ? di->pairs : -1;
}

int lp_set_cta_group(int cg) {
  if (cg != 0 && cg != 1 && cg != 2) return fail(LP_EINVAL, "cta group must be 0, 1 or 2, got %d", cg);
  g_cg.store(cg);
  return LP_OK;
}

int lp_get_cta_group(void) { return cta_group(); }

int lp_profile_enable(int on) {
  std::lock_guard<std::mutex> lk(g_prof_mu);
  for (auto& r : g_prof_records) {
    g_prof_pool.push_back(r.start);
    g_prof_pool.push_back(r.stop);
  }
  g_prof_records.clear();
  g_prof_on = on != 0;
  return LP_OK;
}

int lp_profile_read(int max_tags, char* names, double* total_ms, long long* launches, int* n_tags) {
  if (max_tags <= 0 || names == nullptr || total_ms == nullptr || launches == nullptr || n_tags == nullptr)
    return fail(LP_EINVAL, "bad lp_profile_read arguments");
  std::lock_guard<std::mutex> lk(g_prof_mu);
  int n = 0;
  std::vector<std::string> tags;
  for (auto& r : g_prof_records) {
    LP_CUDA_TRY(cudaEventSynchronize(r.stop));
    float ms = 0.f;
    LP_CUDA_TRY(cudaEventElapsedTime(&ms, r.start, r.stop));
    int k = 0;
    while (k < n && tags[k] != r.tag) ++k;
    if (k == n) {
      if (n == max_tags) continue;
      tags.push_back(r.tag);
      total_ms[n] = 0.0;
      launches[n] = 0;
      ++n;
    }
    total_ms[k] += ms;
    launches[k] += 1;
  }
  for (int k = 0; k < n; ++k) {
    std::strncpy(names + 32 * k, tags[k].c_str(), 31);
    names[32 * k + 31] = 0;
  }
  *n_tags = n;
  return LP_OK;
}

int lp_device_error(int device, int* code) {
  int prev = 0;
  LP_CUDA_TRY(cudaGetDevice(&prev));
  LP_CUDA_TRY(cudaSetDevice(device));
  int v = 0, zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_lp_device_error, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_lp_device_error, &zero, sizeof(int));
  cudaSetDevice(prev);
  if (e != cudaSuccess) return fail(LP_ECUDA, "lp_device_error: %s", cudaGetErrorString(e));
  if (g_host_errors != nullptr && device >= 0 && device < kMaxDevices) {
    if (v == 0) v = reinterpret_cast<volatile int*>(g_host_errors)[device];
    reinterpret_cast<volatile int*>(g_host_errors)[device] = 0;
  }
  if (code) *code = v;
  return LP_OK;
}

int lp_device_error_poll(int device) {
  if (device < 0 || device >= kMaxDevices || g_host_errors == nullptr) return 0;
  return reinterpret_cast<volatile int*>(g_host_errors)[device];
}

size_t lp_fwd_workspace_bytes(int64_t T, int64_t Vs) {
  DeviceInfo* di = nullptr;
  int sms = 148;
  if (current_device_info(&di) == LP_OK) sms = di->sms;
  if (T <= 0 || Vs <= 0) return 256;
  const int cg = cta_group_for(CG_FWD);
  GemmSched s = plan_fwd(T, Vs, 64, di != nullptr ? workers(di, cg) : (cg == 1 ? sms : sms / 2), 128 * cg);
  // partials, target logits, and the [3, T] triples lp_fwd_sum merges first when T is small
  return align_up((size_t)2 * s.n_groups * T * sizeof(float2), 256) + align_up((size_t)T * 4, 256) +
         align_up((size_t)T * 12, 256);
}

int lp_fwd(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs, int64_t v_off,
           const int32_t* y, float softcap, float* stats, float* logp, void* workspace, size_t workspace_bytes) {
  int rc = check_common(H, T, d, ldh, W, Vs, y);
  if (rc) return rc;
  if (T == 0) return LP_OK;
  if (stats == nullptr) return fail(LP_EINVAL, "null stats");
  DeviceInfo* di = nullptr;
  if ((rc = current_device_info(&di))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int cg = cta_group_for(CG_FWD);
  GemmSched s = plan_fwd(T, Vs, d, workers(di, cg), 128 * cg);
  const size_t part_bytes = align_up((size_t)2 * s.n_groups * T * sizeof(float2), 256);
  const size_t need = part_bytes + align_up((size_t)T * 4, 256);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(LP_EWORKSPACE, "lp_fwd needs %zu workspace bytes, got %zu", need, workspace_bytes);
  float2* part = reinterpret_cast<float2*>(workspace);
  float* tgt = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + part_bytes);

  alignas(64) CUtensorMap ta, tb;
  if ((rc = map_bf16(&ta, H, d, T, ldh, BK, 128, "hidden"))) return rc;
  if ((rc = map_bf16(&tb, W, d, Vs, d, BK, b_box_rows(cg), "embedding"))) return rc;
  GemmParams p{};
  p.s = s;
  p.e.y = y;
  p.e.v_off = v_off;
  p.e.softcap = softcap;
  p.e.part = part;
  p.e.tgt = tgt;
  set_hints(p, G_FWD);
  if ((rc = launch_gemm_cap<EPI_FWD_LSE, false, false>(softcap > 0.f, st, ta, tb, ta, p, di, "fwd_lse_gemm"))) return rc;
  ProfScope prof(st, "fwd_finalize");
  if (few_rows(T, di)) {
    fwd_finalize_rows_kernel<<<(unsigned)T, 128, 0, st>>>(part, 2 * s.n_groups, (int)T, tgt, y, v_off, Vs, stats, logp);
    LP_LAUNCH_CHECK("fwd_finalize_rows_kernel");
  } else {
    fwd_finalize_kernel<<<(unsigned)cdiv(T, 256), 256, 0, st>>>(part, 2 * s.n_groups, (int)T, tgt, y, v_off, Vs, stats,
                                                                logp);
    LP_LAUNCH_CHECK("fwd_finalize_kernel");
  }
  return LP_OK;
}

int lp_fwd_sum(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs,
               int64_t v_off, const int32_t* y, float softcap, void* exchange, void* exchange_multicast,
               int64_t ld_exchange, unsigned* counter, unsigned* counter_multicast, unsigned* arrivals,
               unsigned epoch, int rank, int world, int timeout_ms, float* logp, float* norm, void* workspace,
               size_t workspace_bytes) {
  int rc = check_common(H, T, d, ldh, W, Vs, y);
  if (rc) return rc;
  if (world < 1 || rank < 0 || rank >= world) return fail(LP_EINVAL, "bad rank %d / world %d", rank, world);
  if (exchange == nullptr || exchange_multicast == nullptr || counter == nullptr || counter_multicast == nullptr ||
      arrivals == nullptr)
    return fail(LP_EINVAL, "null exchange buffer, counter or arrival counter");
  if (((reinterpret_cast<uintptr_t>(exchange) | reinterpret_cast<uintptr_t>(exchange_multicast)) & 15) != 0)
    return fail(LP_EINVAL, "the exchange buffer and its multicast address must be 16-byte aligned");
  if (ld_exchange < T) return fail(LP_EINVAL, "ld_exchange=%lld < T=%lld", (long long)ld_exchange, (long long)T);
  if (epoch == 0 || (unsigned long long)epoch * (unsigned)world > 0xffffffffull)
    return fail(LP_EINVAL, "epoch %u out of range for world %d", epoch, world);
  if (timeout_ms <= 0) return fail(LP_EINVAL, "timeout_ms must be positive");
  if (T == 0) return LP_OK;
  if (logp == nullptr && norm == nullptr) return fail(LP_EINVAL, "null logp and norm");
  DeviceInfo* di = nullptr;
  if ((rc = current_device_info(&di))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int cg = cta_group_for(CG_FWD);
  GemmSched s = plan_fwd(T, Vs, d, workers(di, cg), 128 * cg);
  const size_t part_bytes = align_up((size_t)2 * s.n_groups * T * sizeof(float2), 256);
  const size_t tgt_bytes = align_up((size_t)T * 4, 256);
  const size_t need = part_bytes + tgt_bytes + align_up((size_t)T * 12, 256);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(LP_EWORKSPACE, "lp_fwd_sum needs %zu workspace bytes, got %zu", need, workspace_bytes);
  float2* part = reinterpret_cast<float2*>(workspace);
  float* tgt = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + part_bytes);
  float* pre = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + part_bytes + tgt_bytes);

  alignas(64) CUtensorMap ta, tb;
  if ((rc = map_bf16(&ta, H, d, T, ldh, BK, 128, "hidden"))) return rc;
  if ((rc = map_bf16(&tb, W, d, Vs, d, BK, b_box_rows(cg), "embedding"))) return rc;
  GemmParams p{};
  p.s = s;
  p.e.y = y;
  p.e.v_off = v_off;
  p.e.softcap = softcap;
  p.e.part = part;
  p.e.tgt = tgt;
  set_hints(p, G_FWD);
  if ((rc = launch_gemm_cap<EPI_FWD_LSE, false, false>(softcap > 0.f, st, ta, tb, ta, p, di, "fwd_lse_gemm"))) return rc;
  // one block per SM at most: every block must be resident while the blocks wait for the
  // other ranks
  const unsigned grid = (unsigned)std::min<int64_t>(cdiv(T, 256), di->sms);
  ProfScope prof(st, "fwd_finalize_mesh");
  const bool merge_first = few_rows(T, di);
  if (merge_first) {
    fwd_finalize_rows_kernel<<<(unsigned)T, 128, 0, st>>>(part, 2 * s.n_groups, (int)T, tgt, y, v_off, Vs, pre,
                                                          nullptr);
    LP_LAUNCH_CHECK("fwd_finalize_rows_kernel");
  }
  fwd_finalize_mesh_kernel<<<grid, 256, 0, st>>>(
      part, 2 * s.n_groups, (int)T, tgt, y, v_off, Vs, reinterpret_cast<float4*>(exchange_multicast),
      reinterpret_cast<const float4*>(exchange), ld_exchange, counter_multicast, counter, arrivals,
      epoch * (unsigned)world, rank, world, (unsigned long long)timeout_ms * 1000000ull, merge_first ? pre : nullptr,
      logp, norm);
  LP_LAUNCH_CHECK("fwd_finalize_mesh_kernel");
  return LP_OK;
}

}  // extern "C"

namespace {

// Sampler head plan: the forward's chunk-major order with one vocabulary tile per unit, so
// a decode batch (one or two M tiles) still spreads over every SM.
GemmSched plan_head(int64_t B, int64_t V, int64_t d, int bm) {
  GemmSched s = plan_fwd(B, V, d, 0, bm);
  s.n_group = 1;
  s.n_groups = s.tiles_n;
  s.num_units = s.tiles_m * s.n_groups;
  return s;
}

size_t head_part_bytes(const GemmSched& s, int64_t B) { return align_up((size_t)2 * s.n_groups * B * sizeof(float2), 256); }

}  // namespace

extern "C" {

size_t lp_head_workspace_bytes(int64_t B, int64_t V) {
  if (B <= 0 || V <= 0) return 256;
  const int cg = cta_group_for(CG_HEAD);
  return 2 * head_part_bytes(plan_head(B, V, 64, 128 * cg), B);
}

int lp_head(void* stream, const void* H, int64_t B, int64_t d, int64_t ldh, const void* W, int64_t V, float softcap,
            float* logits, int64_t ld_logits, int flags, float* norm, int32_t* argmax, float* argmax_logp,
            void* workspace, size_t workspace_bytes) {
  if (B < 0 || d <= 0 || V <= 0) return fail(LP_EINVAL, "bad sizes B=%lld d=%lld V=%lld", (long long)B, (long long)d,
                                              (long long)V);
  if (B > (int64_t)1 << 30 || V > (int64_t)1 << 30) return fail(LP_EINVAL, "B or V above 2^30");
  if (d % 8 != 0) return fail(LP_EINVAL, "hidden size d=%lld must be a multiple of 8", (long long)d);
  if (ldh < d || ldh % 8 != 0) return fail(LP_EINVAL, "ldh=%lld must be >= d and a multiple of 8", (long long)ldh);
  if (W == nullptr || (B > 0 && H == nullptr)) return fail(LP_EINVAL, "null hidden or embedding");
  if (flags & ~LP_HEAD_LOGPROBS) return fail(LP_EINVAL, "unknown lp_head flags %d", flags);
  if (logits != nullptr) {
    if (ld_logits < V || ld_logits % 4 != 0) return fail(LP_EINVAL, "ld_logits must be >= V and a multiple of 4");
    if ((reinterpret_cast<uintptr_t>(logits) & 15) != 0) return fail(LP_EINVAL, "logits must be 16-byte aligned");
  } else if (flags & LP_HEAD_LOGPROBS) {
    return fail(LP_EINVAL, "LP_HEAD_LOGPROBS needs a logits buffer");
  }
  if ((flags & LP_HEAD_LOGPROBS) && norm == nullptr) return fail(LP_EINVAL, "LP_HEAD_LOGPROBS needs norm");
  if (B == 0) return LP_OK;
  DeviceInfo* di = nullptr;
  int rc = current_device_info(&di);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int cg = cta_group_for(CG_HEAD);
  GemmSched s = plan_head(B, V, d, 128 * cg);
  const size_t pb = head_part_bytes(s, B);
  if (workspace == nullptr || workspace_bytes < 2 * pb)
    return fail(LP_EWORKSPACE, "lp_head needs %zu workspace bytes, got %zu", 2 * pb, workspace_bytes);
  float2* part = reinterpret_cast<float2*>(workspace);
  float2* best = reinterpret_cast<float2*>(reinterpret_cast<char*>(workspace) + pb);

  alignas(64) CUtensorMap ta, tb, to;
  if ((rc = map_bf16(&ta, H, d, B, ldh, BK, 128, "hidden"))) return rc;
  if ((rc = map_bf16(&tb, W, d, V, d, BK, b_box_rows(cg), "embedding"))) return rc;
  if (logits != nullptr) {
    if ((rc = map_store_f32(&to, logits, V, B, ld_logits, "logits store"))) return rc;
  } else {
    to = ta;  // not used: no logits are stored
  }
  GemmParams p{};
  p.s = s;
  p.e.softcap = softcap;
  p.e.part = part;
  p.e.best = best;
  p.e.store_logits = logits != nullptr ? 1 : 0;
  set_hints(p, G_FWD);
  if ((rc = launch_gemm_cap<EPI_HEAD, false, false>(softcap > 0.f, st, ta, tb, to, p, di, "head_gemm"))) return rc;
  {
    ProfScope prof(st, "head_finalize");
    head_finalize_kernel<<<(unsigned)B, 256, 0, st>>>(part, best, 2 * s.n_groups, (int)B, norm, argmax, argmax_logp);
    LP_LAUNCH_CHECK("head_finalize_kernel");
  }
  if (flags & LP_HEAD_LOGPROBS) {
    ProfScope prof(st, "logits_to_logprobs");
    const unsigned gx = (unsigned)std::max<int64_t>(1, std::min<int64_t>(cdiv(V / 4 + 1, 256), 64));
    const unsigned gy = (unsigned)std::min<int64_t>(B, 65535);
    logits_to_logprobs_kernel<<<dim3(gx, gy), 256, 0, st>>>(logits, ld_logits, (int)B, V, norm);
    LP_LAUNCH_CHECK("logits_to_logprobs_kernel");
  }
  return LP_OK;
}

int lp_combine(void* stream, const float* shard_stats, int P, int64_t T, float* logp, float* norm) {
  if (P <= 0 || T < 0) return fail(LP_EINVAL, "bad P=%d or T=%lld", P, (long long)T);
  if (T == 0) return LP_OK;
  if (shard_stats == nullptr) return fail(LP_EINVAL, "null shard_stats");
  DeviceInfo* di = nullptr;
  if (int rc = current_device_info(&di)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope prof(st, "combine");
  combine_kernel<<<(unsigned)cdiv(T, 256), 256, 0, st>>>(shard_stats, P, (int)T, logp, norm);
  LP_LAUNCH_CHECK("combine_kernel");
  return LP_OK;
}

size_t lp_bwd_workspace_bytes(int64_t T, int64_t d, int64_t Vs, int64_t token_chunk, int flags) {
  DeviceInfo* di = nullptr;
  int sms = 148;
  if (current_device_info(&di) == LP_OK) sms = di->sms;
  if (T <= 0 || Vs <= 0 || d <= 0) return 256;
  const int cg = cta_group_for(CG_DH);  // the split-K partials follow the dH GEMM's tiles
  return bwd_layout(T, d, Vs, token_chunk, flags, di != nullptr ? workers(di, cg) : (cg == 1 ? sms : sms / 2),
                    128 * cg).total +
         256;
}

}  // extern "C"

namespace {

// The dH sum over the vocabulary mesh inside the dH GEMM (lp_bwd_sum).
struct MeshSum {
  void* dh_mc;
  unsigned* cnt_local;
  unsigned* cnt_mc;
  int rank, world;
  unsigned long long limit_ns;
};

// CTA group of the distribution operators' GEMMs [M, N]. At equal tile counts pairs are faster (a
// 256-row tile takes 0.94 of the time of two 128-row tiles: 512 rows of the 262144 x 2048 head 434
// against 462 us, 1024 rows 826 / 868), but a last half-empty pair tile or a last round that pairs
// fill badly costs more (128 rows 215 / 179 us, 301 rows 403 / 381, 1100 rows 1110 / 1013). Rounds
// of the persistent workers decide, single CTAs' against 0.94 of the pairs'. Below K = 1024 a tile's
// epilogue takes longer than its product, and single CTAs, whose epilogues wait for no other CTA, are
// faster (2048 rows, 131072 columns, K = 256 / 512 / 768: 242 / 253 / 328 us against 273 / 291 / 334).
int cta_group_dist(int64_t M, int64_t N, int64_t K, const DeviceInfo* di, CgUse use) {
  const int f = forced_cta_group();
  if (f) return f;
  if (K <= 768) return 1;
  const int w1 = di != nullptr ? workers(di, 1) : 148, w2 = di != nullptr ? workers(di, 2) : 74;
  const int64_t tn = cdiv(N, BN);
  const double one = (double)cdiv(cdiv(M, 128) * tn, w1), two = 0.94 * (double)cdiv(cdiv(M, 256) * tn, w2);
  return one <= two ? 1 : cta_group_for(use);
}

// The backward of given tokens' log-probabilities and the entropy (lp_dist_bwd): K tokens per row
// and two row constants take the place of one target and its gradient.
struct DistGrad {
  int K;
  int64_t V;  // the whole vocabulary
  const float *zt, *lse, *entropy, *g, *ge;
  const void* kept;       // kept logits (dist_kept_layout of kept_rows rows), or null: recomputed
  int64_t kept_rows;
  const int32_t* row_of;  // row of the kept logits of each row, or null: the row itself
};

// Kept logits: 16 bits each [rows, ld] (16-byte rows), then the largest of every 32 columns
// [rows, ld_max] in f32.
struct KeptLayout {
  int64_t ld, ld_max;
  size_t max_off, total;
};
KeptLayout dist_kept_layout(int64_t rows, int64_t Vs) {
  KeptLayout K;
  K.ld = (Vs + 7) / 8 * 8;
  K.ld_max = cdiv(Vs, BN) * (BN / 32);
  K.max_off = align_up((size_t)rows * K.ld * 2, 256);
  K.total = K.max_off + (size_t)rows * K.ld_max * sizeof(float);
  return K;
}

// Plan and scratch of lp_dist_bwd: the work counters of every GEMM launch (three per chunk) and the
// row constants, before the layout of lp_bwd. In the workspace, not in the library's rotating
// slots, a counter belongs to the call (or to the captured graph) that zeroes it.
struct DistBwdPlan {
  int cg_dz, cg_dh;
  bool split_dh;  // whether the dH GEMM may split K
  BwdLayout L;
  size_t row_off, dh_off, base;
};
DistBwdPlan dist_bwd_plan(int64_t T, int64_t d, int64_t Vs, int64_t token_chunk, int flags, const DeviceInfo* di) {
  DistBwdPlan P;
  const bool want_dh = !(flags & LP_BWD_NO_DH);
  const int64_t tc = token_chunk > 0 ? std::min<int64_t>(token_chunk, T) : default_token_chunk(T, Vs, d);
  P.cg_dz = cta_group_dist(tc, Vs, d, di, CG_DZ);
  // rows of one M tile waste half of a pair whatever the split of K; and a reduce launch takes
  // about as long as 16 K blocks
  P.split_dh = cdiv(Vs, BK) > 32;
  P.cg_dh = forced_cta_group() == 0 && tc <= 128 ? 1 : cta_group_for(CG_DH);
  if (!P.split_dh) flags |= LP_BWD_NO_DH;  // no room for partials
  P.L = bwd_layout(T, d, Vs, token_chunk, flags, di != nullptr ? workers(di, P.cg_dh) : 148 / P.cg_dh, 128 * P.cg_dh);
  P.row_off = align_up((size_t)std::max<int64_t>(P.L.chunks, 1) * 3 * sizeof(unsigned), 1024);
  P.dh_off = P.row_off + align_up((size_t)T * 3 * sizeof(float), 1024);
  // dH of a chunk in f32, where it is not split
  P.base = P.dh_off + (want_dh && P.L.max_splits <= 1 ? align_up((size_t)P.L.mpad * d * sizeof(float), 1024) : 0);
  return P;
}

int bwd_impl(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs, int64_t v_off,
             const int32_t* y, float softcap, const float* norm, const float* g, void* dH, int64_t ld_dh, void* dW,
             int flags, int64_t token_chunk, void* workspace, size_t workspace_bytes, const MeshSum* ms,
             const DistGrad* dist = nullptr) {
  int rc = check_common(H, T, d, ldh, W, Vs, y);
  if (rc) return rc;
  const bool want_dh = !(flags & LP_BWD_NO_DH), want_dw = !(flags & LP_BWD_NO_DW);
  const bool dh_f32 = flags & LP_BWD_DH_F32, dw_bf16 = flags & LP_BWD_DW_BF16;
  if (want_dh && (dH == nullptr || ld_dh < d || ld_dh % 8 != 0))
    return fail(LP_EINVAL, "dH must be non-null with ld_dh >= d and ld_dh %% 8 == 0");
  if (want_dw && dW == nullptr) return fail(LP_EINVAL, "null dW");
  if (T > 0 && dist == nullptr && (norm == nullptr || g == nullptr)) return fail(LP_EINVAL, "null norm or g");
  DeviceInfo* di = nullptr;
  if ((rc = current_device_info(&di))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (T == 0) {
    // no tokens: dW is zero
    if (want_dw) LP_CUDA_TRY(cudaMemsetAsync(dW, 0, (size_t)Vs * d * (dw_bf16 ? 2 : 4), st));
    return LP_OK;
  }
  DistBwdPlan DP{};
  if (dist != nullptr) DP = dist_bwd_plan(T, d, Vs, token_chunk, flags, di);
  const int cg_dz = dist != nullptr ? DP.cg_dz : cta_group_for(CG_DZ);
  const int cg_dh = dist != nullptr ? DP.cg_dh : cta_group_for(CG_DH);
  const bool split_dh = dist != nullptr ? DP.split_dh : ms == nullptr;
  if (ms != nullptr && want_dh) {
    // chunks start on 256-row boundaries (the row-block counters are per 128 rows)
    if (token_chunk <= 0) token_chunk = default_token_chunk(T, Vs, d);
    if (token_chunk < T) token_chunk = std::max<int64_t>(256, token_chunk / 256 * 256);
  }
  const BwdLayout L =
      dist != nullptr ? DP.L : bwd_layout(T, d, Vs, token_chunk, flags, workers(di, cg_dh), 128 * cg_dh);
  if (workspace == nullptr || workspace_bytes < DP.base + L.total)
    return fail(LP_EWORKSPACE, "%s needs %zu workspace bytes, got %zu", dist != nullptr ? "lp_dist_bwd" : "lp_bwd",
                DP.base + L.total, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 1023) != 0) return fail(LP_EINVAL, "workspace must be 1024-byte aligned");
  unsigned* counters = nullptr;  // the next launch's work counter (dist only)
  float* row_const = nullptr;
  if (dist != nullptr) {
    counters = reinterpret_cast<unsigned*>(workspace);
    row_const = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + DP.row_off);
    if (dist->K == 1) {
      row_const = nullptr;  // the dZ epilogue takes one token per row itself
    } else {
      ProfScope prof(st, "dist_row_const");
      dist_row_const_kernel<<<(unsigned)cdiv(T, 256), 256, 0, st>>>(dist->lse, dist->entropy, y, dist->g, dist->ge,
                                                                    (int)T, dist->K, dist->V, row_const);
      LP_LAUNCH_CHECK("dist_row_const_kernel");
    }
  }
  char* ws = reinterpret_cast<char*>(workspace) + DP.base;
  __nv_bfloat16* dz = reinterpret_cast<__nv_bfloat16*>(ws + L.dz_off);
  float* part = reinterpret_cast<float*>(ws + L.part_off);
  float* dw_acc = (want_dw && dw_bf16 && L.chunks > 1) ? reinterpret_cast<float*>(ws + L.dwacc_off)
                                                        : reinterpret_cast<float*>(dW);
  const bool cap = softcap > 0.f;
  const __nv_bfloat16* Hb = reinterpret_cast<const __nv_bfloat16*>(H);

  for (int64_t c = 0; c < L.chunks; ++c) {
    const int64_t t0 = c * L.tc;
    const int64_t tcur = std::min<int64_t>(L.tc, T - t0);
    const __nv_bfloat16* Hc = Hb + t0 * ldh;

    // 1) recompute logits tile by tile and write dZ (bf16) for this chunk (or take kept logits)
    if (dist == nullptr || dist->kept == nullptr) {
      alignas(64) CUtensorMap ta, tb, to;
      if ((rc = map_bf16(&ta, Hc, d, tcur, ldh, BK, 128, "hidden chunk"))) return rc;
      if ((rc = map_bf16(&tb, W, d, Vs, d, BK, b_box_rows(cg_dz), "embedding"))) return rc;
      if ((rc = map_store_bf16(&to, dz, Vs, tcur, L.ldz, "dZ store"))) return rc;
      GemmParams p{};
      p.s = plan_dz(tcur, Vs, d, workers(di, cg_dz), 128 * cg_dz);
      p.e.softcap = softcap;
      set_hints(p, G_DZ);
      if (dist != nullptr) {
        if (row_const != nullptr) {
          p.e.row_const = row_const + t0;
          p.e.row_ld = T;
        } else {
          p.e.y = y + t0;
          p.e.v_off = v_off;
          p.e.vocab = dist->V;
          p.e.g = dist->g != nullptr ? dist->g + t0 : nullptr;
          p.e.ge = dist->ge != nullptr ? dist->ge + t0 : nullptr;
          p.e.lse = dist->lse + t0;
          p.e.entropy = dist->entropy + t0;
        }
        p.sched = counters++;
        if ((rc = launch_gemm_cap<EPI_DIST_DZ, false, false>(cap, st, ta, tb, to, p, di, "dist_dz_gemm"))) return rc;
      } else {
        p.e.y = y + t0;
        p.e.v_off = v_off;
        p.e.g = g + t0;
        p.e.stats = norm + t0;
        p.e.stats_ld = T;
        if ((rc = launch_gemm_cap<EPI_BWD_DZ, false, false>(cap, st, ta, tb, to, p, di, "bwd_dz_gemm"))) return rc;
      }
    }
    if (dist != nullptr && dist->kept != nullptr) {
      const KeptLayout K = dist_kept_layout(dist->kept_rows, Vs);
      DistDzParams z{};
      // without row_of the kept rows are this call's rows
      const int64_t first = dist->row_of != nullptr ? 0 : t0;
      z.kept = reinterpret_cast<const uint16_t*>(dist->kept) + first * K.ld;
      z.kept_max = reinterpret_cast<const float*>(reinterpret_cast<const char*>(dist->kept) + K.max_off) + first * K.ld_max;
      z.row_of = dist->row_of != nullptr ? dist->row_of + t0 : nullptr;
      z.ldk = K.ld;
      z.ld_max = K.ld_max;
      if (row_const != nullptr) {
        z.row_const = row_const + t0;
        z.row_ld = T;
      } else {
        z.y = y + t0;
        z.zt = dist->zt + t0;
        z.g = dist->g != nullptr ? dist->g + t0 : nullptr;
        z.ge = dist->ge != nullptr ? dist->ge + t0 : nullptr;
        z.lse = dist->lse + t0;
        z.entropy = dist->entropy + t0;
      }
      z.vocab = dist->V;
      z.v_off = v_off;
      z.Vs = Vs;
      z.cap = softcap;
      z.dz = dz;
      z.ldz = L.ldz;
      // enough blocks for every SM, a row each where there are rows enough
      const int64_t row_steps = cdiv(Vs, kDzStep);
      const int64_t per_row = std::max<int64_t>(1, std::min<int64_t>(cdiv(row_steps, 2), cdiv(16 * di->sms, tcur)));
      z.steps = (int)cdiv(row_steps, per_row);
      ProfScope prof(st, "dist_dz");
      for (int64_t r = 0; r < tcur; r += 32768) {  // a grid has at most 65535 rows
        const int64_t rows = std::min<int64_t>(32768, tcur - r);
        DistDzParams zr = z;
        if (z.row_of != nullptr) zr.row_of = z.row_of + r;
        else {
          zr.kept = z.kept + r * K.ld;
          zr.kept_max = z.kept_max + r * K.ld_max;
        }
        if (row_const != nullptr) zr.row_const = z.row_const + r;
        else {
          zr.y = z.y + r;
          zr.zt = z.zt + r;
          zr.g = z.g != nullptr ? z.g + r : nullptr;
          zr.ge = z.ge != nullptr ? z.ge + r : nullptr;
          zr.lse = z.lse + r;
          zr.entropy = z.entropy + r;
        }
        zr.dz = z.dz + r * L.ldz;
        dist_dz_kernel<<<dim3((unsigned)cdiv(row_steps, z.steps), (unsigned)rows), 256, 0, st>>>(zr);
        LP_LAUNCH_CHECK("dist_dz_kernel");
      }
    }
    DistEntries entries{};
    if (dist != nullptr) {
      const int64_t at = t0 * dist->K;
      entries.y = y + at;
      entries.K = dist->K;
      entries.zt = dist->zt + at;
      entries.g = dist->g != nullptr ? dist->g + at : nullptr;
      entries.row_const = row_const != nullptr ? row_const + t0 : nullptr;
      entries.row_ld = T;
      entries.ge = dist->ge != nullptr ? dist->ge + t0 : nullptr;
      entries.lse = dist->lse + t0;
      entries.entropy = dist->entropy + t0;
      entries.v_off = v_off;
      entries.Vs = Vs;
      entries.cap = softcap;
      entries.dz = dz;
      entries.ldz = L.ldz;
    }
    if (dist != nullptr && row_const != nullptr && dist->K > 0) {
      // the given tokens' entries
      ProfScope prof(st, "dist_dz_targets");
      dist_dz_targets_kernel<<<(unsigned)cdiv(tcur * dist->K, 256), 256, 0, st>>>(
          y + t0 * dist->K, dist->zt + t0 * dist->K, dist->g != nullptr ? dist->g + t0 * dist->K : nullptr,
          row_const + t0, T, (int)tcur, dist->K, v_off, Vs, softcap, dz, L.ldz);
      LP_LAUNCH_CHECK("dist_dz_targets_kernel");
    }
    // 2) dH[t0:t0+tcur] = dZ . W
    if (want_dh) {
      alignas(64) CUtensorMap ta, tb, to;
      if ((rc = map_bf16(&ta, dz, Vs, tcur, L.ldz, BK, 128, "dZ as A"))) return rc;
      GemmParams p{};
      p.b_mn3d = mn3d_enabled() && d % 64 == 0;
      if (p.b_mn3d) rc = map_mn3d(&tb, W, d, Vs, d, b_box_rows(cg_dh) / 64, "embedding as MN-major B");
      else rc = map_bf16(&tb, W, d, Vs, d, 64, 64, "embedding as MN-major B");
      if (rc) return rc;
      const int wk = workers(di, cg_dh);
      p.s = plan_gemm(tcur, d, Vs, wk, split_dh, 1, 128 * cg_dh);
      char* dh_c = reinterpret_cast<char*>(dH) + (size_t)t0 * ld_dh * (dh_f32 ? 4 : 2);
      // with given tokens the product stays in f32 until what rounding left of their entries has joined it
      const bool finish = dist != nullptr && dist->K > 0;
      float* dh_part = part;
      if (finish && p.s.k_splits == 1 && L.max_splits <= 1)
        dh_part = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + DP.dh_off);
      if (ms != nullptr) {
        // partial tiles stored (bf16) into this rank's copy, summed across ranks by the
        // reduce items of the same launch
        if ((rc = map_store_bf16(&to, dh_c, d, tcur, ld_dh, "dH partial store", store_box_bytes(cg_dh)))) return rc;
        p.e.store_mode = STORE_BF16;
        p.e.split_rows = 0;
        p.s.red_lag = std::min(p.s.tiles_m, (int)cdiv(3 * (int64_t)wk, p.s.tiles_n) + 2);
        p.s.num_units = p.s.tiles_m * p.s.tiles_n + p.s.tiles_m;
        p.e.sum_mc = reinterpret_cast<__nv_bfloat16*>(reinterpret_cast<char*>(ms->dh_mc) + (size_t)t0 * ld_dh * 2);
        p.e.sum_local = reinterpret_cast<__nv_bfloat16*>(dh_c);
        p.e.sum_ld = ld_dh;
        p.e.cnt_local = ms->cnt_local + t0 / 128;
        p.e.cnt_mc = ms->cnt_mc + t0 / 128;
        p.e.cnt_target = (unsigned)(ms->world * p.s.tiles_n * EPI_WARPS * cg_dh);
        p.e.sum_rank = ms->rank;
        p.e.sum_world = ms->world;
        p.e.peer_limit_ns = ms->limit_ns;
      } else if (p.s.k_splits == 1 && !finish) {
        if (dh_f32) {
          if ((rc = map_store_f32(&to, dh_c, d, tcur, ld_dh, "dH store", store_box_bytes(cg_dh)))) return rc;
          p.e.store_mode = STORE_F32;
        } else {
          if ((rc = map_store_bf16(&to, dh_c, d, tcur, ld_dh, "dH store", store_box_bytes(cg_dh)))) return rc;
          p.e.store_mode = STORE_BF16;
        }
        p.e.split_rows = 0;
      } else {
        if ((rc = map_store_f32(&to, dh_part, d, (uint64_t)p.s.k_splits * L.mpad, d, "dH partials",
                                store_box_bytes(cg_dh))))
          return rc;
        p.e.store_mode = STORE_F32;
        p.e.split_rows = (int)L.mpad;
      }
      set_hints(p, G_DH);
      if (counters != nullptr) p.sched = counters++;
      if ((rc = launch_gemm<EPI_STORE, false, true, false>(st, ta, tb, to, p, di, "bwd_dh_gemm"))) return rc;
      if (finish) {
        ProfScope prof(st, "dist_dh_finish");
        dist_dh_finish_kernel<<<(unsigned)tcur, kDistRowThreads, 0, st>>>(
            dh_part, p.s.k_splits, L.mpad, entries, reinterpret_cast<const __nv_bfloat16*>(W), d, dh_c, ld_dh, !dh_f32);
        LP_LAUNCH_CHECK("dist_dh_finish_kernel");
      } else if (p.s.k_splits > 1) {
        const int64_t total = tcur * (d / 4);
        const unsigned grid = (unsigned)std::min<int64_t>(cdiv(total, 256), (int64_t)di->sms * 8);
        ProfScope prof(st, "splitk_reduce");
        splitk_reduce_kernel<<<grid, 256, 0, st>>>(part, p.s.k_splits, tcur, d, L.mpad, dh_c, ld_dh, dh_f32 ? 0 : 1);
        LP_LAUNCH_CHECK("splitk_reduce_kernel");
      }
    }
    // 3) dW (+)= dZ^T . H_chunk
    if (want_dw) {
      const int cg_dw = cta_group_dw(tcur);
      alignas(64) CUtensorMap ta, tb, to;
      GemmParams p{};
      p.a_mn3d = mn3d_enabled() && Vs % 64 == 0;
      p.b_mn3d = mn3d_enabled() && d % 64 == 0;
      if (p.a_mn3d) rc = map_mn3d(&ta, dz, Vs, tcur, L.ldz, 2, "dZ as MN-major A");
      else rc = map_bf16(&ta, dz, Vs, tcur, L.ldz, 64, 64, "dZ as MN-major A");
      if (rc) return rc;
      if (p.b_mn3d) rc = map_mn3d(&tb, Hc, d, tcur, ldh, b_box_rows(cg_dw) / 64, "hidden as MN-major B");
      else rc = map_bf16(&tb, Hc, d, tcur, ldh, 64, 64, "hidden as MN-major B");
      if (rc) return rc;
      p.s = plan_gemm(Vs, d, tcur, workers(di, cg_dw), false, 1, 128 * cg_dw);
      const bool direct_bf16 = dw_bf16 && L.chunks == 1;
      if (direct_bf16) {
        if ((rc = map_store_bf16(&to, dW, d, Vs, d, "dW store", store_box_bytes(cg_dw)))) return rc;
        p.e.store_mode = STORE_BF16;
      } else {
        if ((rc = map_store_f32(&to, dw_acc, d, Vs, d, "dW store", store_box_bytes(cg_dw)))) return rc;
        p.e.store_mode = c == 0 ? STORE_F32 : STORE_F32_ADD;
      }
      set_hints(p, G_DW);
      if (counters != nullptr) p.sched = counters++;
      if ((rc = launch_gemm<EPI_STORE, true, true, false>(st, ta, tb, to, p, di, "bwd_dw_gemm"))) return rc;
      if (dist != nullptr && dist->K > 0 && L.chunks == 1 && T <= kDistRowThreads && T * T * dist->K <= kDistDwRows) {
        ProfScope prof(st, "dist_dw_rows");
        dist_dw_rows_kernel<<<(unsigned)(T * dist->K), kDistRowThreads, 0, st>>>(entries, (int)T, Hb, ldh, d, dW, dw_bf16);
        LP_LAUNCH_CHECK("dist_dw_rows_kernel");
      }
    }
  }
  if (want_dw && dw_bf16 && L.chunks > 1) {
    const int64_t n = Vs * d;
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(n / 4 + 1, 256), (int64_t)di->sms * 8);
    ProfScope prof(st, "f32_to_bf16");
    f32_to_bf16_kernel<<<grid, 256, 0, st>>>(dw_acc, reinterpret_cast<__nv_bfloat16*>(dW), n);
    LP_LAUNCH_CHECK("f32_to_bf16_kernel");
  }
  return LP_OK;
}

}  // namespace

extern "C" {

int lp_bwd(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs, int64_t v_off,
           const int32_t* y, float softcap, const float* norm, const float* g, void* dH, int64_t ld_dh, void* dW,
           int flags, int64_t token_chunk, void* workspace, size_t workspace_bytes) {
  return bwd_impl(stream, H, T, d, ldh, W, Vs, v_off, y, softcap, norm, g, dH, ld_dh, dW, flags, token_chunk,
                  workspace, workspace_bytes, nullptr);
}

size_t lp_bwd_sum_counters(int64_t T) { return T > 0 ? (size_t)cdiv(T, 128) + 2 : 0; }

int lp_bwd_sum(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs,
               int64_t v_off, const int32_t* y, float softcap, const float* norm, const float* g, void* dH,
               void* dH_multicast, int64_t ld_dh, unsigned* counters, unsigned* counters_multicast, int rank,
               int world, int timeout_ms, void* dW, int flags, int64_t token_chunk, void* workspace,
               size_t workspace_bytes) {
  if (flags & (LP_BWD_DH_F32 | LP_BWD_NO_DH))
    return fail(LP_EINVAL, "lp_bwd_sum sums a bf16 dH: LP_BWD_DH_F32 / LP_BWD_NO_DH do not apply");
  if (dH_multicast == nullptr || counters == nullptr || counters_multicast == nullptr)
    return fail(LP_EINVAL, "null multicast dH or counters");
  if (((reinterpret_cast<uintptr_t>(dH) | reinterpret_cast<uintptr_t>(dH_multicast)) & 15) != 0)
    return fail(LP_EINVAL, "dH and its multicast address must be 16-byte aligned");
  if (world < 1 || rank < 0 || rank >= world) return fail(LP_EINVAL, "bad rank %d / world %d", rank, world);
  if (timeout_ms <= 0) return fail(LP_EINVAL, "timeout_ms must be positive");
  const MeshSum ms{dH_multicast, counters, counters_multicast, rank, world, (unsigned long long)timeout_ms * 1000000ull};
  return bwd_impl(stream, H, T, d, ldh, W, Vs, v_off, y, softcap, norm, g, dH, ld_dh, dW, flags, token_chunk,
                  workspace, workspace_bytes, &ms);
}

int lp_gemm_bf16(void* stream, const void* A, int64_t M, int64_t K, int64_t lda, int a_mn, const void* B, int64_t N,
                 int64_t ldb, int b_mn, float* D, int64_t ldd) {
  if (M <= 0 || N <= 0 || K <= 0) return fail(LP_EINVAL, "bad GEMM sizes");
  if (A == nullptr || B == nullptr || D == nullptr) return fail(LP_EINVAL, "null GEMM operand");
  if (ldd < N || ldd % 4 != 0) return fail(LP_EINVAL, "ldd must be >= N and a multiple of 4");
  if (N % 4 != 0) return fail(LP_EINVAL, "N must be a multiple of 4");
  DeviceInfo* di = nullptr;
  int rc = current_device_info(&di);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  alignas(64) CUtensorMap ta, tb, to;
  // K-major A: [M rows][K], MN-major A: [K rows][M]; likewise B with N.
  if (a_mn) rc = map_bf16(&ta, A, M, K, lda, 64, 64, "A (MN-major)");
  else rc = map_bf16(&ta, A, K, M, lda, BK, 128, "A (K-major)");
  if (rc) return rc;
  const int cg = cta_group_for(CG_HOOK);
  if (b_mn) rc = map_bf16(&tb, B, N, K, ldb, 64, 64, "B (MN-major)");
  else rc = map_bf16(&tb, B, K, N, ldb, BK, b_box_rows(cg), "B (K-major)");
  if (rc) return rc;
  if ((rc = map_store_f32(&to, D, N, M, ldd, "D", store_box_bytes(cg)))) return rc;
  GemmParams p{};
  p.s = plan_gemm(M, N, K, workers(di, cg), false, 0, 128 * cg);
  p.e.store_mode = STORE_F32;
  if (!a_mn && !b_mn) return launch_gemm<EPI_STORE, false, false, false>(st, ta, tb, to, p, di, "gemm");
  if (!a_mn && b_mn) return launch_gemm<EPI_STORE, false, true, false>(st, ta, tb, to, p, di, "gemm");
  if (a_mn && b_mn) return launch_gemm<EPI_STORE, true, true, false>(st, ta, tb, to, p, di, "gemm");
  return launch_gemm<EPI_STORE, true, false, false>(st, ta, tb, to, p, di, "gemm");
}

size_t lp_compact_workspace_bytes(int64_t B, int64_t N) {
  const int64_t slots = std::max<int64_t>(B * N, 1);
  return align_up((size_t)cdiv(slots, kCompactBlock) * 4, 256) * 2;
}

int lp_compact(void* stream, const uint8_t* mask, int64_t B, int64_t N, const void* hidden, int64_t hidden_bstride,
               int64_t hidden_rstride, int64_t row_offset, int64_t d, const int32_t* ids, void* H_out, int32_t* y_out,
               int32_t* idx, int32_t* pos, int32_t* count, void* workspace, size_t workspace_bytes) {
  if (B < 0 || N < 0) return fail(LP_EINVAL, "bad B=%lld N=%lld", (long long)B, (long long)N);
  const int64_t slots = B * N;
  if (slots > ((int64_t)1 << 31) - 1) return fail(LP_EINVAL, "too many slots");
  if (mask == nullptr || idx == nullptr || pos == nullptr || count == nullptr)
    return fail(LP_EINVAL, "null mask / idx / pos / count");
  if (hidden != nullptr) {
    if (d <= 0 || d % 8 != 0) return fail(LP_EINVAL, "d=%lld must be a positive multiple of 8", (long long)d);
    if (H_out == nullptr) return fail(LP_EINVAL, "null H_out");
    if (hidden_rstride % 8 != 0 || hidden_bstride % 8 != 0) return fail(LP_EINVAL, "hidden strides must be multiples of 8");
    if ((reinterpret_cast<uintptr_t>(hidden) & 15) || (reinterpret_cast<uintptr_t>(H_out) & 15))
      return fail(LP_EINVAL, "hidden / H_out must be 16-byte aligned");
    if (y_out != nullptr && ids == nullptr) return fail(LP_EINVAL, "y_out needs ids");
  }
  const size_t need = lp_compact_workspace_bytes(B, N);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(LP_EWORKSPACE, "lp_compact needs %zu workspace bytes, got %zu", need, workspace_bytes);
  DeviceInfo* di = nullptr;
  if (int rc = current_device_info(&di)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (slots == 0) {
    LP_CUDA_TRY(cudaMemsetAsync(count, 0, sizeof(int32_t), st));
    return LP_OK;
  }
  const int nblocks = (int)cdiv(slots, kCompactBlock);
  ProfScope prof(st, "compact");
  int* block_counts = reinterpret_cast<int*>(workspace);
  int* block_offsets = reinterpret_cast<int*>(reinterpret_cast<char*>(workspace) + need / 2);
  compact_count_kernel<<<nblocks, 256, 0, st>>>(mask, slots, block_counts);
  LP_LAUNCH_CHECK("compact_count_kernel");
  compact_scan_kernel<<<1, 1024, 0, st>>>(block_counts, nblocks, block_offsets, count);
  LP_LAUNCH_CHECK("compact_scan_kernel");
  compact_write_kernel<<<nblocks, 256, 0, st>>>(mask, slots, block_offsets, idx, pos);
  LP_LAUNCH_CHECK("compact_write_kernel");
  if (hidden != nullptr) {
    const int64_t warps = std::min<int64_t>(slots, (int64_t)di->sms * 32);
    compact_gather_kernel<<<(unsigned)cdiv(warps * 32, 256), 256, 0, st>>>(
        idx, count, N, reinterpret_cast<const __nv_bfloat16*>(hidden), hidden_bstride, hidden_rstride, row_offset, d,
        ids, reinterpret_cast<__nv_bfloat16*>(H_out), y_out);
    LP_LAUNCH_CHECK("compact_gather_kernel");
  }
  return LP_OK;
}

int lp_scatter_rows(void* stream, const void* src, int64_t src_stride, const int32_t* pos, int64_t slots,
                    int64_t width, int elem_bytes, void* out, int64_t out_stride, int64_t rows_per_group,
                    int64_t group_stride, int out_elem_bytes) {
  if (slots < 0 || width <= 0 || (elem_bytes != 2 && elem_bytes != 4))
    return fail(LP_EINVAL, "bad slots / width / elem_bytes");
  if (out_elem_bytes != elem_bytes && !(elem_bytes == 4 && out_elem_bytes == 2))
    return fail(LP_EINVAL, "out_elem_bytes must equal elem_bytes, or be 2 for f32 -> bf16");
  if (rows_per_group <= 0) return fail(LP_EINVAL, "rows_per_group must be positive");
  if (slots == 0) return LP_OK;
  if (src == nullptr || pos == nullptr || out == nullptr) return fail(LP_EINVAL, "null src / pos / out");
  DeviceInfo* di = nullptr;
  if (int rc = current_device_info(&di)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (out_elem_bytes != elem_bytes) {
    if (width % 8 != 0 || src_stride % 4 != 0 || out_stride % 8 != 0 || group_stride % 8 != 0 ||
        (reinterpret_cast<uintptr_t>(src) & 15) || (reinterpret_cast<uintptr_t>(out) & 15))
      return fail(LP_EINVAL, "f32 -> bf16 scatter needs width % 8 == 0 and 16-byte aligned rows");
    ProfScope prof(st, "scatter_rows");
    const int64_t warps = std::min<int64_t>(slots, 148 * 64);
    scatter_rows_f32_to_bf16_kernel<<<(unsigned)cdiv(warps * 32, 256), 256, 0, st>>>(
        reinterpret_cast<const float*>(src), src_stride, pos, slots, width, reinterpret_cast<__nv_bfloat16*>(out),
        out_stride, rows_per_group, group_stride);
    LP_LAUNCH_CHECK("scatter_rows_f32_to_bf16_kernel");
    return LP_OK;
  }
  const int64_t row_bytes = width * elem_bytes;
  ProfScope prof(st, "scatter_rows");
  const bool vec = row_bytes % 16 == 0 && (src_stride * elem_bytes) % 16 == 0 && (out_stride * elem_bytes) % 16 == 0 &&
                   (group_stride * elem_bytes) % 16 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0 &&
                   (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  if (vec) {
    const int64_t warps = std::min<int64_t>(slots, 148 * 64);
    scatter_rows_vec_kernel<<<(unsigned)cdiv(warps * 32, 256), 256, 0, st>>>(
        reinterpret_cast<const uint8_t*>(src), src_stride * elem_bytes, pos, slots, row_bytes,
        reinterpret_cast<uint8_t*>(out), out_stride * elem_bytes, rows_per_group, group_stride * elem_bytes);
    LP_LAUNCH_CHECK("scatter_rows_vec_kernel");
  } else {
    const int64_t total = slots * width;
    const unsigned grid = (unsigned)std::min<int64_t>(cdiv(total, 256), 148 * 16);
    scatter_rows_elem_kernel<<<grid, 256, 0, st>>>(reinterpret_cast<const uint8_t*>(src), src_stride, pos, slots,
                                                   width, elem_bytes, reinterpret_cast<uint8_t*>(out), out_stride,
                                                   rows_per_group, group_stride);
    LP_LAUNCH_CHECK("scatter_rows_elem_kernel");
  }
  return LP_OK;
}

int lp_peer_barrier(void* stream, const unsigned long long* signal_pads, int rank, int world, int channel,
                    int timeout_ms) {
  if (signal_pads == nullptr) return fail(LP_EINVAL, "null signal_pads");
  if (world < 1 || world > 1024 || rank < 0 || rank >= world) return fail(LP_EINVAL, "bad rank %d / world %d", rank, world);
  if (channel < 0 || timeout_ms <= 0) return fail(LP_EINVAL, "bad channel %d or timeout %d ms", channel, timeout_ms);
  DeviceInfo* di = nullptr;
  if (int rc = current_device_info(&di)) return rc;  // device set-up (host-visible error slot)
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int threads = (world + 31) / 32 * 32;
  ProfScope prof(st, "peer_barrier");
  peer_barrier_kernel<<<1, threads, 0, st>>>(signal_pads, rank, world, channel,
                                             (unsigned long long)timeout_ms * 1000000ull);
  LP_LAUNCH_CHECK("peer_barrier_kernel");
  return LP_OK;
}

}  // extern "C"

// ============================================================================= distribution operators
namespace {

struct DistFwdLayout {
  GemmSched s;
  int cg;
  size_t length_off, part_off, part_a_off, keys_off, total;
};

// Scratch of one launch over T rows as CTA group cg: its work counter, (top) the lengths of the
// embedding's longest rows, the (max, S) and A partials, and (top) the rows' selection keys.
DistFwdLayout dist_fwd_layout(int cg, int64_t T, int64_t Vs, int64_t d, const DeviceInfo* di, size_t key_row_bytes) {
  DistFwdLayout L{};
  L.cg = cg;
  L.s = plan_fwd(T, Vs, d, di != nullptr ? workers(di, cg) : 148 / cg, 128 * cg);
  L.length_off = 256;
  L.part_off = L.length_off +
               align_up(key_row_bytes > 0 ? (size_t)(di != nullptr ? di->sms : 148) * SCAN_WARPS * sizeof(float) : 0, 256);
  L.part_a_off = L.part_off + align_up((size_t)2 * L.s.n_groups * T * sizeof(float2), 256);
  L.keys_off = L.part_a_off + align_up((size_t)2 * L.s.n_groups * T * sizeof(float), 256);
  L.total = L.keys_off + align_up((size_t)T * key_row_bytes, 256);
  return L;
}
DistFwdLayout dist_fwd_layout(int64_t T, int64_t Vs, int64_t d, const DeviceInfo* di) {
  return dist_fwd_layout(cta_group_dist(T, Vs, d, di, CG_FWD), T, Vs, d, di, 0);
}
// Enough for any hidden size, whichever CTA group that leads to.
size_t dist_fwd_bytes(int64_t T, int64_t Vs, const DeviceInfo* di) {
  return std::max(dist_fwd_layout(1, T, Vs, 64, di, 0).total, dist_fwd_layout(2, T, Vs, 64, di, 0).total);
}

// Rows of the hidden operand's box: of a single M tile only the rows there are (in eights, the
// swizzle's period). Loading 128 with all but a few out of bounds took 224 us for one row of the
// 262144 x 2048 head.
uint32_t a_box_rows(const DistFwdLayout& L, int64_t T) {
  return L.cg == 1 && T < 128 ? (uint32_t)align_up((size_t)T, 8) : 128u;
}
uint32_t a_box_bytes(const DistFwdLayout& L, int64_t T) {
  const uint32_t rows = a_box_rows(L, T);
  return rows < 128 ? rows * BK * 2 : 0;
}

// A head that a single M tile streams once leaves the L2 to what is read again: the partials, the
// keys and the next kernel's code.
void dist_hints(GemmParams& p) {
  set_hints(p, G_FWD);
  if (p.s.tiles_m == 1 && p.e.b_l2 == L2_NORMAL) p.e.b_l2 = L2_EVICT_FIRST;
}

int check_dist(const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs, const int32_t* y,
               int64_t K) {
  if (K < 0 || K > LP_DIST_MAX_TOKENS) return fail(LP_EINVAL, "K=%lld tokens per row, at most %d", (long long)K,
                                                    LP_DIST_MAX_TOKENS);
  if (K > 0 && T > 0 && y == nullptr) return fail(LP_EINVAL, "null tokens");
  static const int32_t none = 0;
  return check_common(H, T, d, ldh, W, Vs, K > 0 ? y : &none);
}

// Selection keys of a row: two values per group of 32 or 8 columns, or the f32 logits. Larger groups
// are fewer bytes to write and to search, but two of the about n = k + kTopSpare selected tokens fall into
// one group n^2 / (2 V / group) times, and then its other columns are scored again. A group size is
// taken where that adds at most half as many scores again: V >= 992 n for 32, 56 n for 8.
struct TopKeys {
  int group;   // columns per key
  int64_t ld;  // keys per row in memory
  int n;       // keys per row
  size_t row_bytes;
  int64_t rows;  // rows per launch: their keys stay within 1 GiB
};
TopKeys top_keys(int64_t T, int64_t V, int k) {
  TopKeys K;
  const int64_t n = k + kTopSpare;
  K.group = V >= 992 * n ? 32 : (V >= 56 * n ? 8 : 1);
  K.n = (int)cdiv(V, K.group);
  K.ld = K.group > 1 ? cdiv(V, BN) * (BN / K.group) : (V + 3) / 4 * 4;
  K.row_bytes = (size_t)K.ld * (K.group > 1 ? 2 : 1) * sizeof(float);
  K.rows = std::max<int64_t>(1, std::min<int64_t>(T, (int64_t)(((size_t)1 << 30) / K.row_bytes)));
  return K;
}

// Single CTAs, since only they can take the lengths of the embedding's rows beside the products (pairs
// share their barriers). Pairs would be 0.94 of the time with many rows, but a pass of its own for the
// lengths takes 165 us of the 262144 x 2048 head (512 rows: 528 us as it is, 438 + 165 that way).
DistFwdLayout top_layout(int64_t T, int64_t V, int64_t d, const DeviceInfo* di, size_t key_row_bytes) {
  return dist_fwd_layout(1, T, V, d, di, key_row_bytes);
}

size_t top_workspace(int64_t T, int64_t V, int k, const DeviceInfo* di) {
  const TopKeys K = top_keys(T, V, k);
  size_t need = top_layout(K.rows, V, 64, di, K.row_bytes).total;
  if (T % K.rows != 0) need = std::max(need, top_layout(T % K.rows, V, 64, di, K.row_bytes).total);
  return need;
}

template <int EPI>
int launch_top_gemm(bool cap, cudaStream_t st, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& o,
                    const GemmParams& p, const DeviceInfo* di) {
  return cap ? launch_gemm_cg<1, EPI, false, false, true>(st, a, b, o, p, di, "top_gemm")
             : launch_gemm_cg<1, EPI, false, false, false>(st, a, b, o, p, di, "top_gemm");
}

template <bool SAMPLE, int G>
int launch_top_select(cudaStream_t st, TopParams& P, int64_t rows) {
  const size_t key_bytes = align_up((size_t)P.n_keys * sizeof(uint32_t), 16);
  P.keys_in_smem = key_bytes <= (size_t)kTopKeyBytes;
  const size_t smem = P.keys_in_smem ? key_bytes : 0;
  auto kern = top_select_kernel<SAMPLE, G>;
  static bool configured[kMaxDevices] = {};
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (!configured[dev]) {
    LP_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kTopKeyBytes));
    configured[dev] = true;
  }
  ProfScope prof(st, "top_select");
  kern<<<(unsigned)rows, kTopThreads, smem, st>>>(P);
  LP_LAUNCH_CHECK("top_select_kernel");
  return LP_OK;
}

template <bool SAMPLE>
int launch_top_select(int group, cudaStream_t st, TopParams& P, int64_t rows) {
  return group == 32 ? launch_top_select<SAMPLE, 32>(st, P, rows)
                     : (group == 8 ? launch_top_select<SAMPLE, 8>(st, P, rows) : launch_top_select<SAMPLE, 1>(st, P, rows));
}

// The selection of lp_top and lp_sample_top_k over all rows; `all` holds the outputs and options.
int top_impl(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t V, float softcap,
             bool sample, const TopParams& all, void* workspace, size_t workspace_bytes) {
  DeviceInfo* di = nullptr;
  int rc = current_device_info(&di);
  if (rc) return rc;
  const TopKeys K = top_keys(T, V, all.k);
  const size_t need = top_workspace(T, V, all.k, di);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(LP_EWORKSPACE, "%zu workspace bytes needed, got %zu", need, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return fail(LP_EINVAL, "workspace must be 256-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  for (int64_t t0 = 0; t0 < T; t0 += K.rows) {
    const int64_t n = std::min<int64_t>(K.rows, T - t0);
    const DistFwdLayout L = top_layout(n, V, d, di, K.row_bytes);
    const __nv_bfloat16* Hc = reinterpret_cast<const __nv_bfloat16*>(H) + t0 * ldh;
    alignas(64) CUtensorMap ta, tb, to;
    if ((rc = map_bf16(&ta, Hc, d, n, ldh, BK, a_box_rows(L, n), "hidden"))) return rc;
    if ((rc = map_bf16(&tb, W, d, V, d, BK, b_box_rows(L.cg), "embedding"))) return rc;
    GemmParams p{};
    p.s = L.s;
    p.a_box_bytes = a_box_bytes(L, n);
    p.sched = reinterpret_cast<unsigned*>(ws);
    p.e.softcap = softcap;
    p.e.part = reinterpret_cast<float2*>(ws + L.part_off);
    p.e.part_a = reinterpret_cast<float*>(ws + L.part_a_off);
    p.e.length2 = reinterpret_cast<float*>(ws + L.length_off);
    dist_hints(p);
    if (K.group > 1) {
      p.e.top = reinterpret_cast<float*>(ws + L.keys_off);
      rc = K.group == 32 ? launch_top_gemm<EPI_DIST_TOP32>(softcap > 0.f, st, ta, tb, ta, p, di)
                         : launch_top_gemm<EPI_DIST_TOP8>(softcap > 0.f, st, ta, tb, ta, p, di);
    } else {
      if ((rc = map_store_f32(&to, ws + L.keys_off, V, n, K.ld, "logits store"))) return rc;
      rc = launch_top_gemm<EPI_DIST_LOGITS>(softcap > 0.f, st, ta, tb, to, p, di);
    }
    if (rc) return rc;
    TopParams P = all;
    P.part = p.e.part;
    P.part_a = p.e.part_a;
    P.n_parts = 2 * L.s.n_groups;
    P.length2 = p.e.length2;
    P.n_lengths = std::max(1, std::min(L.s.num_units, workers(di, 1))) * SCAN_WARPS;
    P.T = (int)n;
    P.H = Hc;
    P.ldh = ldh;
    P.W = reinterpret_cast<const __nv_bfloat16*>(W);
    P.d = d;
    P.V = V;
    P.cap = softcap;
    if (K.group > 1) P.groups = p.e.top; else P.logits = reinterpret_cast<const float*>(ws + L.keys_off);
    P.ld_keys = K.ld;
    P.n_keys = K.n;
    if (sample) {
      P.uniform = all.uniform + t0;
      P.sampled = all.sampled + t0;
      P.logps = all.logps + t0;
      rc = launch_top_select<true>(K.group, st, P, n);
    } else {
      P.tokens = all.tokens != nullptr ? all.tokens + t0 : nullptr;
      P.ids = all.ids + t0 * all.k;
      P.logps = all.logps + t0 * all.k;
      P.entropy = all.entropy + t0;
      P.token_logps = all.token_logps != nullptr ? all.token_logps + t0 : nullptr;
      rc = launch_top_select<false>(K.group, st, P, n);
    }
    if (rc) return rc;
  }
  return LP_OK;
}

int check_top(const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t V, int k) {
  if (int rc = check_dist(H, T, d, ldh, W, V, nullptr, 0)) return rc;
  if (k < 1 || k > LP_TOP_MAX || k > V)
    return fail(LP_EINVAL, "k=%d must be between 1 and min(%d, V=%lld)", k, LP_TOP_MAX, (long long)V);
  return LP_OK;
}

}  // namespace

static_assert(kTopMax == LP_TOP_MAX, "LP_TOP_MAX");
static_assert(LP_DIST_MAX_TOKENS <= kDistRowThreads, "a thread for each of a row's tokens");

extern "C" {

size_t lp_dist_fwd_workspace_bytes(int64_t T, int64_t Vs) {
  DeviceInfo* di = nullptr;
  const bool have = current_device_info(&di) == LP_OK;
  if (T <= 0 || Vs <= 0) return 256;
  return dist_fwd_bytes(T, Vs, have ? di : nullptr);
}

size_t lp_dist_kept_bytes(int64_t T, int64_t Vs) {
  return T > 0 && Vs > 0 ? dist_kept_layout(T, Vs).total : 0;
}

int lp_dist_fwd(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs,
                int64_t v_off, const int32_t* y, int64_t K, float softcap, float* stats, float* zt, float* lse,
                float* entropy, float* logp, void* kept, void* workspace, size_t workspace_bytes) {
  int rc = check_dist(H, T, d, ldh, W, Vs, y, K);
  if (rc) return rc;
  if (T == 0) return LP_OK;
  DeviceInfo* di = nullptr;
  if ((rc = current_device_info(&di))) return rc;
  const DistFwdLayout L = dist_fwd_layout(T, Vs, d, di);
  if (workspace == nullptr || workspace_bytes < L.total)
    return fail(LP_EWORKSPACE, "lp_dist_fwd needs %zu workspace bytes, got %zu", L.total, workspace_bytes);
  if ((reinterpret_cast<uintptr_t>(workspace) & 255) != 0) return fail(LP_EINVAL, "workspace must be 256-byte aligned");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  alignas(64) CUtensorMap ta, tb;
  if ((rc = map_bf16(&ta, H, d, T, ldh, BK, a_box_rows(L, T), "hidden"))) return rc;
  if ((rc = map_bf16(&tb, W, d, Vs, d, BK, b_box_rows(L.cg), "embedding"))) return rc;
  GemmParams p{};
  p.s = L.s;
  p.a_box_bytes = a_box_bytes(L, T);
  p.sched = reinterpret_cast<unsigned*>(ws);
  p.e.softcap = softcap;
  p.e.part = reinterpret_cast<float2*>(ws + L.part_off);
  p.e.part_a = reinterpret_cast<float*>(ws + L.part_a_off);
  dist_hints(p);
  if (kept != nullptr) {
    const KeptLayout KL = dist_kept_layout(T, Vs);
    alignas(64) CUtensorMap to;
    if ((rc = map_store_bf16(&to, kept, Vs, T, KL.ld, "kept logits"))) return rc;  // 16-bit elements
    p.e.keep_max = reinterpret_cast<float*>(reinterpret_cast<char*>(kept) + KL.max_off);
    rc = launch_gemm_cap<EPI_DIST_KEEP, false, false>(softcap > 0.f, st, ta, tb, to, p, di, "dist_fwd_gemm");
  } else {
    rc = launch_gemm_cap<EPI_DIST, false, false>(softcap > 0.f, st, ta, tb, ta, p, di, "dist_fwd_gemm");
  }
  if (rc) return rc;
  ProfScope prof(st, "dist_finalize");
  const __nv_bfloat16* Hb = reinterpret_cast<const __nv_bfloat16*>(H);
  const __nv_bfloat16* Wb = reinterpret_cast<const __nv_bfloat16*>(W);
  const int n_parts = 2 * L.s.n_groups;
  // eight rows per block share the 32-byte sectors of the partials; few rows get a block each
  if (T < (int64_t)8 * di->sms)
    dist_finalize_kernel<1><<<(unsigned)T, kDistThreads, 0, st>>>(p.e.part, p.e.part_a, n_parts, (int)T, Hb, ldh, Wb, d,
                                                                  Vs, v_off, y, (int)K, softcap, stats, zt, lse, entropy,
                                                                  logp);
  else
    dist_finalize_kernel<8><<<(unsigned)cdiv(T, 8), kDistThreads, 0, st>>>(p.e.part, p.e.part_a, n_parts, (int)T, Hb, ldh,
                                                                           Wb, d, Vs, v_off, y, (int)K, softcap, stats,
                                                                           zt, lse, entropy, logp);
  LP_LAUNCH_CHECK("dist_finalize_kernel");
  return LP_OK;
}

int lp_dist_combine(void* stream, const float* shard_stats, const float* shard_zt, int P, int64_t T, int64_t K,
                    int64_t V, const int32_t* y, float* lse, float* entropy, float* zt, float* logp) {
  if (P <= 0 || T < 0 || T > (int64_t)1 << 30) return fail(LP_EINVAL, "bad P=%d or T=%lld", P, (long long)T);
  if (K < 0 || K > LP_DIST_MAX_TOKENS) return fail(LP_EINVAL, "K=%lld tokens per row, at most %d", (long long)K,
                                                    LP_DIST_MAX_TOKENS);
  if (T == 0) return LP_OK;
  if (shard_stats == nullptr || lse == nullptr || entropy == nullptr)
    return fail(LP_EINVAL, "null shard_stats, lse or entropy");
  if (K > 0 && (shard_zt == nullptr || y == nullptr || zt == nullptr || logp == nullptr))
    return fail(LP_EINVAL, "null shard_zt, tokens, zt or logp");
  DeviceInfo* di = nullptr;
  if (int rc = current_device_info(&di)) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  ProfScope prof(st, "dist_combine");
  dist_combine_kernel<<<(unsigned)cdiv(T, 128), 128, 0, st>>>(shard_stats, shard_zt, P, (int)T, (int)K, V, y, lse,
                                                              entropy, zt, logp);
  LP_LAUNCH_CHECK("dist_combine_kernel");
  return LP_OK;
}

size_t lp_dist_bwd_workspace_bytes(int64_t T, int64_t d, int64_t Vs, int64_t token_chunk, int flags) {
  if (T <= 0 || Vs <= 0 || d <= 0) return 256;
  DeviceInfo* di = nullptr;
  const bool have = current_device_info(&di) == LP_OK;
  const DistBwdPlan P = dist_bwd_plan(T, d, Vs, token_chunk, flags, have ? di : nullptr);
  return P.base + P.L.total;
}

int lp_dist_bwd(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs,
                int64_t v_off, int64_t V, const int32_t* y, int64_t K, float softcap, const float* zt, const float* lse,
                const float* entropy, const float* g_logp, const float* g_entropy, const void* kept, int64_t kept_rows,
                const int32_t* row_of, void* dH, int64_t ld_dh, void* dW, int flags, int64_t token_chunk,
                void* workspace, size_t workspace_bytes) {
  if (int rc = check_dist(H, T, d, ldh, W, Vs, y, K)) return rc;
  if (v_off < 0 || v_off + Vs > V) return fail(LP_EINVAL, "shard [%lld, %lld) outside the vocabulary of %lld",
                                               (long long)v_off, (long long)(v_off + Vs), (long long)V);
  if (T > 0 && (lse == nullptr || entropy == nullptr || (K > 0 && zt == nullptr)))
    return fail(LP_EINVAL, "null lse, entropy or zt");
  static const int32_t none = 0;
  if (kept != nullptr && ((reinterpret_cast<uintptr_t>(kept) & 15) != 0 || kept_rows < (row_of != nullptr ? 1 : T)))
    return fail(LP_EINVAL, "kept logits must be 16-byte aligned and have a row for each row");
  if (((reinterpret_cast<uintptr_t>(dH) | reinterpret_cast<uintptr_t>(dW)) & 15) != 0)
    return fail(LP_EINVAL, "dH and dW must be 16-byte aligned");
  const DistGrad dg{(int)K, V, zt, lse, entropy, K > 0 ? g_logp : nullptr, g_entropy, kept, kept_rows, row_of};
  return bwd_impl(stream, H, T, d, ldh, W, Vs, v_off, K > 0 ? y : &none, softcap, nullptr, nullptr, dH, ld_dh, dW, flags,
                  token_chunk, workspace, workspace_bytes, nullptr, &dg);
}

size_t lp_dist_rows_workspace_bytes(int64_t T) {
  return align_up((size_t)std::max<int64_t>(T, 1), 256) + lp_compact_workspace_bytes(1, T);
}

int lp_dist_rows(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const int32_t* y, int64_t K,
                 const float* zt, const float* lse, const float* entropy, const float* g_logp, const float* g_entropy,
                 void* H_out, int32_t* y_out, float* zt_out, float* lse_out, float* entropy_out, float* g_logp_out,
                 float* g_entropy_out, int32_t* idx, int32_t* pos, int32_t* count, void* workspace,
                 size_t workspace_bytes) {
  if (T <= 0 || T > (int64_t)1 << 30 || d <= 0 || d % 8 != 0 || ldh < d || ldh % 8 != 0)
    return fail(LP_EINVAL, "bad sizes T=%lld d=%lld ldh=%lld", (long long)T, (long long)d, (long long)ldh);
  if (K < 0 || K > LP_DIST_MAX_TOKENS) return fail(LP_EINVAL, "K=%lld tokens per row, at most %d", (long long)K,
                                                    LP_DIST_MAX_TOKENS);
  if (H == nullptr || lse == nullptr || entropy == nullptr || H_out == nullptr || lse_out == nullptr ||
      entropy_out == nullptr || (K > 0 && (y == nullptr || zt == nullptr || y_out == nullptr || zt_out == nullptr)) ||
      (g_logp != nullptr && g_logp_out == nullptr) || (g_entropy != nullptr && g_entropy_out == nullptr))
    return fail(LP_EINVAL, "null input or output");
  if (((reinterpret_cast<uintptr_t>(H) | reinterpret_cast<uintptr_t>(H_out)) & 15) != 0)
    return fail(LP_EINVAL, "hidden rows must be 16-byte aligned");
  const size_t need = lp_dist_rows_workspace_bytes(T);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(LP_EWORKSPACE, "lp_dist_rows needs %zu workspace bytes, got %zu", need, workspace_bytes);
  DeviceInfo* di = nullptr;
  int rc = current_device_info(&di);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  uint8_t* mask = reinterpret_cast<uint8_t*>(workspace);
  char* rest = reinterpret_cast<char*>(workspace) + align_up((size_t)T, 256);
  ProfScope prof(st, "dist_rows");
  dist_row_mask_kernel<<<(unsigned)cdiv(T, 256), 256, 0, st>>>(K > 0 ? g_logp : nullptr, g_entropy, (int)T, (int)K, mask);
  LP_LAUNCH_CHECK("dist_row_mask_kernel");
  if ((rc = lp_compact(stream, mask, 1, T, nullptr, 0, 0, 0, 0, nullptr, nullptr, nullptr, idx, pos, count, rest,
                       lp_compact_workspace_bytes(1, T))))
    return rc;
  const DistRows from{reinterpret_cast<const __nv_bfloat16*>(H), ldh, y, zt, lse, entropy, g_logp, g_entropy};
  const DistRowsOut to{reinterpret_cast<__nv_bfloat16*>(H_out), y_out, zt_out, lse_out, entropy_out, g_logp_out,
                       g_entropy_out};
  const int64_t warps = std::min<int64_t>(T, (int64_t)di->sms * 32);
  dist_gather_kernel<<<(unsigned)cdiv(warps * 32, 256), 256, 0, st>>>(idx, count, from, to, d, (int)K);
  LP_LAUNCH_CHECK("dist_gather_kernel");
  return LP_OK;
}

size_t lp_top_workspace_bytes(int64_t T, int64_t V, int k) {
  DeviceInfo* di = nullptr;
  const bool have = current_device_info(&di) == LP_OK;
  if (T <= 0 || V <= 0 || k < 1) return 256;
  return top_workspace(T, V, k, have ? di : nullptr);
}

int lp_top(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t V, float softcap,
           int k, const int32_t* tokens, int32_t* ids, float* logps, float* entropy, float* token_logps,
           void* workspace, size_t workspace_bytes) {
  if (int rc = check_top(H, T, d, ldh, W, V, k)) return rc;
  if (T == 0) return LP_OK;
  if (ids == nullptr || logps == nullptr || entropy == nullptr) return fail(LP_EINVAL, "null ids, logps or entropy");
  if (tokens != nullptr && token_logps == nullptr) return fail(LP_EINVAL, "tokens need token_logps");
  TopParams P{};
  P.k = k;
  P.tokens = tokens;
  P.ids = ids;
  P.logps = logps;
  P.entropy = entropy;
  P.token_logps = token_logps;
  return top_impl(stream, H, T, d, ldh, W, V, softcap, false, P, workspace, workspace_bytes);
}

int lp_sample_top_k(void* stream, const void* H, int64_t B, int64_t d, int64_t ldh, const void* W, int64_t V,
                    float softcap, int k, const float* uniform, double temperature, double top_p, int32_t* token,
                    float* logp, void* workspace, size_t workspace_bytes) {
  if (int rc = check_top(H, B, d, ldh, W, V, k)) return rc;
  if (!(temperature > 0.) || temperature > 1.7e308) return fail(LP_EINVAL, "temperature must be finite and positive");
  if (!(top_p > 0. && top_p <= 1.)) return fail(LP_EINVAL, "top_p must be in (0, 1]");
  if (B == 0) return LP_OK;
  if (uniform == nullptr || token == nullptr || logp == nullptr) return fail(LP_EINVAL, "null uniform, token or logp");
  TopParams P{};
  P.k = k;
  P.uniform = uniform;
  P.temperature = temperature;
  P.top_p = top_p;
  P.sampled = token;
  P.logps = logp;
  return top_impl(stream, H, B, d, ldh, W, V, softcap, true, P, workspace, workspace_bytes);
}

}  // extern "C"

// ============================================================================= no-alloc forward
// lp_fwd_noalloc: the forward of lp_fwd for callers that cannot allocate device memory at
// the call site. Its scratch (the per-row partial max / sum of every vocabulary group and
// the owned target logit) lives in one file-scope device array that every GPU which loads
// this library holds until the process exits. Host code must not hand the array's name to
// a kernel (in host code it is only a stand-in symbol): the device address is looked up
// once per device with cudaGetSymbolAddress and cached.
namespace {
constexpr size_t kNoAllocScratchBytes = size_t(LP_NOALLOC_SCRATCH_BYTES);
}  // namespace

static __device__ __align__(256) unsigned char g_lp_noalloc_scratch[kNoAllocScratchBytes];

namespace {

void* g_noalloc_scratch_ptr[kMaxDevices] = {};
std::mutex g_noalloc_mu;

// Device address of the scratch array on the current device (set up on first use there).
int noalloc_scratch(void** out) {
  int dev = 0;
  LP_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= kMaxDevices) return fail(LP_EINVAL, "device ordinal %d out of range", dev);
  std::lock_guard<std::mutex> lk(g_noalloc_mu);
  if (g_noalloc_scratch_ptr[dev] == nullptr) {
    void* p = nullptr;
    const cudaError_t e = cudaGetSymbolAddress(&p, g_lp_noalloc_scratch);
    if (e != cudaSuccess || p == nullptr)
      return fail(LP_ECUDA, "cudaGetSymbolAddress(no-alloc scratch) on device %d: %s", dev, cudaGetErrorString(e));
    g_noalloc_scratch_ptr[dev] = p;
  }
  *out = g_noalloc_scratch_ptr[dev];
  return LP_OK;
}


}  // namespace

extern "C" int lp_fwd_noalloc(void* stream, const void* H, int64_t T, int64_t d, int64_t ldh, const void* W, int64_t Vs,
                              int64_t v_off, const int32_t* y, float softcap, float* stats, float* logp) {
  int rc = check_common(H, T, d, ldh, W, Vs, y);
  if (rc) return rc;
  if (T == 0) return LP_OK;
  if (stats == nullptr) return fail(LP_EINVAL, "null stats");
  DeviceInfo* di = nullptr;
  if ((rc = current_device_info(&di))) return rc;
  // Same tile plan as lp_fwd, with the vocabulary groups widened until the partials fit
  // the fixed scratch; too many tokens for even one group is refused.
  const int cg = cta_group_for(CG_FWD);
  GemmSched s = plan_fwd(T, Vs, d, workers(di, cg), 128 * cg);
  size_t part_bytes = 0;
  const size_t need = widen_fwd_groups(&s, T, kNoAllocScratchBytes, &part_bytes);
  if (need > kNoAllocScratchBytes)
    return fail(LP_EINVAL,
                "lp_fwd_noalloc: T=%lld tokens need %zu scratch bytes, above its fixed limit of %zu bytes "
                "(LP_NOALLOC_SCRATCH_BYTES); use lp_fwd with a workspace",
                (long long)T, need, kNoAllocScratchBytes);
  void* scratch = nullptr;
  if ((rc = noalloc_scratch(&scratch))) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  float2* part = reinterpret_cast<float2*>(scratch);
  float* tgt = reinterpret_cast<float*>(reinterpret_cast<char*>(scratch) + part_bytes);

  alignas(64) CUtensorMap ta, tb;
  if ((rc = map_bf16(&ta, H, d, T, ldh, BK, 128, "hidden"))) return rc;
  if ((rc = map_bf16(&tb, W, d, Vs, d, BK, b_box_rows(cg), "embedding"))) return rc;
  GemmParams p{};
  p.s = s;
  p.e.y = y;
  p.e.v_off = v_off;
  p.e.softcap = softcap;
  p.e.part = part;
  p.e.tgt = tgt;
  set_hints(p, G_FWD);
  if ((rc = launch_gemm_cap<EPI_FWD_LSE, false, false>(softcap > 0.f, st, ta, tb, ta, p, di, "fwd_lse_gemm"))) return rc;
  ProfScope prof(st, "fwd_finalize");
  fwd_finalize_kernel<<<(unsigned)cdiv(T, 256), 256, 0, st>>>(part, 2 * s.n_groups, (int)T, tgt, y, v_off, Vs, stats,
                                                              logp);
  LP_LAUNCH_CHECK("fwd_finalize_kernel");
  return LP_OK;
}
