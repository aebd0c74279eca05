// Shared by the decode operators (kv_cache.cu, tree_attn.cu, verify.cu): argument checks on the host, lookups on the device.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/pcp_b200.h"
#include "decode_index.h"

namespace pcpb {
namespace {

inline int op_fail(char* err, size_t cap, int code, const char* fmt, ...) {
  if (err && cap) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, cap, fmt, ap);
    va_end(ap);
  }
  return code;
}

// Driver entry point of the pointer query, resolved at run time (no link-time dependency on libcuda): one call for both attributes takes
// a third of cudaPointerGetAttributes, and a small operator has a dozen pointers.
typedef CUresult (*PointerQueryFn)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
inline PointerQueryFn pointer_query() {
  static PointerQueryFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    return cudaGetDriverEntryPoint("cuPointerGetAttributes", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess ? (PointerQueryFn)p : nullptr;
  }();
  return fn;
}
// Multiprocessors of a device, asked for once.
inline int sm_count(int dev) {
  static int known[64] = {};
  if (dev < 0 || dev >= 64) return 148;
  if (!known[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) { cudaGetLastError(); return 148; }
    known[dev] = n;
  }
  return known[dev];
}

// The device all pointers of a call live on becomes the current one for the call.
struct OpDevice {
  char* err;
  size_t cap;
  int dev = -1, prev = -1, rc = PCPB_OK;
  OpDevice(char* e, size_t c) : err(e), cap(c) {}
  // `what` names the argument in the message; NULL is accepted (optional arguments)
  void on(const void* p, const char* what) {
    if (!p || rc) return;
    const PointerQueryFn query = pointer_query();
    unsigned type = 0;
    int where = -1;
    CUpointer_attribute which[2] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
    void* out[2] = {&type, &where};
    const CUresult e = query ? query(2, which, out, (CUdeviceptr)p) : CUDA_ERROR_NOT_INITIALIZED;
    if (e != CUDA_SUCCESS) rc = op_fail(err, cap, PCPB_E_CUDA, "%s: no CUDA device, or the driver refused the address (%d)", what, (int)e);
    else if (type != CU_MEMORYTYPE_DEVICE && type != CU_MEMORYTYPE_UNIFIED) rc = op_fail(err, cap, PCPB_E_INVALID, "%s is not device memory", what);
    else if (dev < 0) dev = where;
    else if (where != dev) rc = op_fail(err, cap, PCPB_E_INVALID, "%s lives on device %d, the call's other arguments on device %d", what, where, dev);
  }
  int enter() {
    if (rc) return rc;
    if (cudaGetDevice(&prev) != cudaSuccess) { prev = -1; return rc = op_fail(err, cap, PCPB_E_CUDA, "no current CUDA device"); }
    if (dev < 0) dev = prev;
    if (dev == prev) prev = -1;
    else if (cudaSetDevice(dev) != cudaSuccess) return rc = op_fail(err, cap, PCPB_E_CUDA, "cannot select device %d", dev);
    return PCPB_OK;
  }
  int done(cudaError_t e) {
    return e == cudaSuccess ? PCPB_OK : op_fail(err, cap, PCPB_E_CUDA, "launch failed: %s", cudaGetErrorString(e));
  }
  ~OpDevice() { if (prev >= 0) cudaSetDevice(prev); }
};

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Checks a cache description and fills in its default strides.
inline int check_cache(const pcpb_kv_cache* c, pcpb_kv_cache* out, char* err, size_t cap) {
  if (!c) return op_fail(err, cap, PCPB_E_INVALID, "null cache");
  *out = *c;
  pcpb_kv_cache& o = *out;
  if (o.dtype != PCPB_BF16 && o.dtype != PCPB_I8 && o.dtype != PCPB_E4M3) return op_fail(err, cap, PCPB_E_INVALID, "cache dtype must be bf16, i8 or e4m3");
  if (o.head_dim != 32 && o.head_dim != 64 && o.head_dim != 128) return op_fail(err, cap, PCPB_E_INVALID, "head_dim must be 32, 64 or 128");
  if (o.n_kv_head < 1 || o.n_kv_head > 1024 || o.page_tokens < 1 || o.n_pages < 1 || o.batch < 1 || o.max_pages < 1)
    return op_fail(err, cap, PCPB_E_INVALID, "bad cache geometry");
  if ((long long)o.max_pages * o.page_tokens > 0x7fff0000ll) return op_fail(err, cap, PCPB_E_TOO_LARGE, "more than 2^31 positions a sequence");
  const long long rows = (long long)o.n_kv_head * o.page_tokens;
  if (!o.page_stride) o.page_stride = rows * o.head_dim;
  if (!o.scale_stride) o.scale_stride = rows;
  if (o.page_stride < rows * o.head_dim || o.scale_stride < rows) return op_fail(err, cap, PCPB_E_INVALID, "pages overlap (page_stride or scale_stride too small)");
  const bool codes = o.dtype != PCPB_BF16;
  if (o.page_stride % (codes ? 16 : 8)) return op_fail(err, cap, PCPB_E_INVALID, "pages must start on 16-byte boundaries");
  if (!o.k || !o.v || !o.block_table) return op_fail(err, cap, PCPB_E_INVALID, "null pages or block table");
  if (codes && (!o.k_scale || !o.v_scale)) return op_fail(err, cap, PCPB_E_INVALID, "an 8-bit cache needs k_scale and v_scale");
  if (!aligned16(o.k) || !aligned16(o.v)) return op_fail(err, cap, PCPB_E_INVALID, "pages must start on 16-byte boundaries");
  return PCPB_OK;
}
inline void on_cache(OpDevice& d, const pcpb_kv_cache& c) {
  d.on(c.k, "cache.k"); d.on(c.v, "cache.v"); d.on(c.block_table, "block_table");
  if (c.dtype != PCPB_BF16) { d.on(c.k_scale, "k_scale"); d.on(c.v_scale, "v_scale"); }
}
// Rows [row][head][i] of element size es: a row of a head starts on a 16-byte boundary
inline bool rows_aligned(const void* p, long long row, long long head, int es) {
  const int n = 16 / es;
  return aligned16(p) && row % n == 0 && head % n == 0;
}

__device__ __forceinline__ void op_note(int32_t* status, int bit) {
  if (status && !(*(volatile int32_t*)status & bit)) atomicOr(status, bit);
}
// The sequence b with cu[b] <= e < cu[b + 1], by the whole warp (32-ary search, one round for up to 32 sequences); cu need
// not be sorted for the search to stay inside [0, batch).
__device__ __forceinline__ int warp_find_seq(const int32_t* __restrict__ cu, int batch, int e) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = batch;
  while (n > 1) {
    const int step = (n + 31) / 32, at = (lane + 1) * step;     // is the boundary before lo + at at or below e?
    const bool below = at < n && __ldg(cu + lo + at) <= e;
    const int cnt = __popc(__ballot_sync(0xffffffffu, below));
    lo += cnt * step;
    n = min(step, n - cnt * step);
  }
  return lo;
}
// Physical page of position pos of sequence b, or -1 (outside the table or the cache)
__device__ __forceinline__ int page_of(const pcpb_kv_cache& c, int b, int lp) {
  if (lp < 0 || lp >= c.max_pages) return -1;
  return clip_page(__ldg(c.block_table + (size_t)b * c.max_pages + lp), c.n_pages);
}

}  // namespace
}  // namespace pcpb
