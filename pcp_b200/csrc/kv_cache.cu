// A paged KV cache in 8 bits: rows quantised as they are written, and read back.
//
//   a = max(amax |x| / Q, 2^-126),  c = round(x / a),  value a c        Q = 448 (e4m3), 127 (signed integers)
//
// One row of a head has one scale.  Both divisions are f32 divisions rounded to nearest, so that codes and scales are the same
// bits wherever they are computed.  The scale's floor keeps it a normal number: rows of zeros get codes 0 and no division by zero,
// and rows below 2^-126 Q lose precision instead of overflowing their codes.
// Bound: HBM.  A row is read once (16-byte loads, HD / 8 lanes a row, the row's largest magnitude by shuffles) and its codes are
// written once.
#include <cuda_fp8.h>

#include "common.cuh"
#include "decode_ops.h"

namespace pcpb {
namespace {

struct KvArgs {
  pcpb_kv_cache c;
  pcpb_kv_rows r;
  int32_t* status;
};

template <int CODE> struct CodeMax { static constexpr float v = CODE == PCPB_I8 ? 127.f : 448.f; };

// Eight values to eight codes (two 32-bit words).
template <int CODE> __device__ __forceinline__ uint2 encode8(const float (&f)[8], float a) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (CODE == PCPB_E4M3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[4 * h], a), __fdiv_rn(f[4 * h + 1], a)), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(f[4 * h + 2], a), __fdiv_rn(f[4 * h + 3], a)), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | (hi << 16);
    } else {
      w[h] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[h] |= (uint32_t)(__float2int_rn(__fdiv_rn(f[4 * h + i], a)) & 0xFF) << (8 * i);
    }
  }
  return make_uint2(w[0], w[1]);
}
template <int CODE> __device__ __forceinline__ void decode8(uint2 w, float (&f)[8]) {
  const uint32_t ws[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t b = (ws[i >> 2] >> (8 * (i & 3))) & 0xFF;
    if (CODE == PCPB_E4M3) f[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
    else f[i] = (float)(int)(int8_t)b;
  }
}

// Where an entry's rows are: false when the entry is left out.  Called by whole warps.
struct Entry { int page, off, row; };
__device__ __forceinline__ bool find_entry(const KvArgs& A, int e, Entry* out) {
  const int b = warp_find_seq(A.r.cu_rows, A.c.batch, e);
  const int lo = A.r.cu_rows[b], hi = A.r.cu_rows[b + 1];
  if (e < lo || e >= hi) return false;
  const int row = A.r.index ? A.r.index[e] : e;
  if (row < 0) return false;
  const long long pos = (long long)A.r.pos0[b] + (e - lo);
  if (row >= A.r.n_rows || pos < 0 || pos >= (long long)A.c.max_pages * A.c.page_tokens) { op_note(A.status, PCPB_OPS_BAD_LENGTH); return false; }
  out->row = row;
  out->page = page_of(A.c, b, (int)pos / A.c.page_tokens);
  out->off = (int)pos % A.c.page_tokens;
  if (out->page < 0) op_note(A.status, PCPB_OPS_BAD_PAGE);
  return true;
}

// One block per entry: groups of HD / 8 lanes take the rows (k heads, then v heads) in turn.
template <int HD, int CODE, typename S> __global__ void __launch_bounds__(256) k_kv_write(KvArgs A) {
  constexpr int L = HD / 8;                                     // lanes of a row
  Entry en;
  if (!find_entry(A, (int)blockIdx.x, &en) || en.page < 0) return;
  const int lane = threadIdx.x % L, Hkv = A.c.n_kv_head;
  for (int u0 = 0; u0 < 2 * Hkv; u0 += blockDim.x / L) {
    const int u = u0 + threadIdx.x / L;
    const bool on = u < 2 * Hkv, isv = u >= Hkv;
    const int h = isv ? u - Hkv : u;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on) ld8<S>((const S*)(isv ? A.r.v : A.r.k) + (isv ? en.row * A.r.v_row + h * A.r.v_head : en.row * A.r.k_row + h * A.r.k_head) + lane * 8, f);
    const size_t at = page_row(en.page, A.c.page_stride, h, A.c.page_tokens, en.off, HD) + lane * 8;
    if (CODE == PCPB_BF16) {
      if (on) st8<bf16>((bf16*)(isv ? A.c.v : A.c.k) + at, f);
      continue;
    }
    uint32_t m = 0;                                             // magnitudes as bit patterns: NaN sorts above every number
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const bool finite = m < 0x7F800000u;
    const float a = finite ? fmaxf(__fdiv_rn(__uint_as_float(m), CodeMax<CODE>::v), 1.17549435e-38f) : __uint_as_float(0x7FC00000u);
    if (!on) continue;
    const uint2 w = finite ? encode8<CODE == PCPB_BF16 ? PCPB_I8 : CODE>(f, a) : make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>((uint8_t*)(isv ? A.c.v : A.c.k) + at) = w;
    if (lane == 0) (isv ? A.c.v_scale : A.c.k_scale)[page_row(en.page, A.c.scale_stride, h, A.c.page_tokens, en.off, 1)] = a;
  }
}

template <int HD, int CODE, typename S> __global__ void __launch_bounds__(256) k_kv_read(KvArgs A) {
  constexpr int L = HD / 8;
  Entry en;
  if (!find_entry(A, (int)blockIdx.x, &en)) return;
  const int lane = threadIdx.x % L, Hkv = A.c.n_kv_head;
  for (int u = threadIdx.x / L; u < 2 * Hkv; u += blockDim.x / L) {
    const bool isv = u >= Hkv;
    const int h = isv ? u - Hkv : u;
    float f[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (en.page >= 0) {
      const size_t at = page_row(en.page, A.c.page_stride, h, A.c.page_tokens, en.off, HD) + lane * 8;
      if (CODE == PCPB_BF16) {
        ld8<bf16>((const bf16*)(isv ? A.c.v : A.c.k) + at, f);
      } else {
        const float a = (isv ? A.c.v_scale : A.c.k_scale)[page_row(en.page, A.c.scale_stride, h, A.c.page_tokens, en.off, 1)];
        decode8<CODE>(*reinterpret_cast<const uint2*>((const uint8_t*)(isv ? A.c.v : A.c.k) + at), f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] *= a;
      }
    }
    st8<S>((S*)(isv ? A.r.v : A.r.k) + (isv ? en.row * A.r.v_row + h * A.r.v_head : en.row * A.r.k_row + h * A.r.k_head) + lane * 8, f);
  }
}

template <int HD, int CODE, typename S> void launch(bool write, cudaStream_t st, const KvArgs& A) {
  const int rows = 2 * A.c.n_kv_head * (HD / 8);
  const int threads = rows >= 256 ? 256 : (rows + 31) / 32 * 32;
  if (write) k_kv_write<HD, CODE, S><<<A.r.n_entries, threads, 0, st>>>(A);
  else k_kv_read<HD, CODE, S><<<A.r.n_entries, threads, 0, st>>>(A);
}
template <int HD, typename S> void by_code(bool write, cudaStream_t st, const KvArgs& A) {
  if (A.c.dtype == PCPB_BF16) launch<HD, PCPB_BF16, S>(write, st, A);
  else if (A.c.dtype == PCPB_I8) launch<HD, PCPB_I8, S>(write, st, A);
  else launch<HD, PCPB_E4M3, S>(write, st, A);
}
template <typename S> void by_width(bool write, cudaStream_t st, const KvArgs& A) {
  if (A.c.head_dim == 128) by_code<128, S>(write, st, A);
  else if (A.c.head_dim == 64) by_code<64, S>(write, st, A);
  else by_code<32, S>(write, st, A);
}

int kv_rows_call(bool write, void* stream, const pcpb_kv_cache* cache, const pcpb_kv_rows* rows, int32_t* status, char* err, size_t cap) {
  if (err && cap) err[0] = 0;
  KvArgs A;
  const int rc = check_cache(cache, &A.c, err, cap);
  if (rc) return rc;
  if (!rows) return op_fail(err, cap, PCPB_E_INVALID, "null rows");
  A.r = *rows; A.status = status;
  const pcpb_kv_rows& r = A.r;
  if (r.dtype != PCPB_BF16 && r.dtype != PCPB_F32) return op_fail(err, cap, PCPB_E_INVALID, "rows must be bf16 or f32");
  if (r.n_rows < 0 || r.n_entries < 0) return op_fail(err, cap, PCPB_E_INVALID, "negative row or entry count");
  if (r.n_entries == 0 || r.n_rows == 0) return PCPB_OK;
  if (!r.k || !r.v || !r.cu_rows || !r.pos0) return op_fail(err, cap, PCPB_E_INVALID, "null rows, cu_rows or pos0");
  const int es = r.dtype == PCPB_BF16 ? 2 : 4;
  if (!rows_aligned(r.k, r.k_row, r.k_head, es) || !rows_aligned(r.v, r.v_row, r.v_head, es))
    return op_fail(err, cap, PCPB_E_INVALID, "rows of k and v must start on 16-byte boundaries");
  OpDevice d(err, cap);
  on_cache(d, A.c);
  d.on(r.k, "k"); d.on(r.v, "v"); d.on(r.cu_rows, "cu_rows"); d.on(r.pos0, "pos0"); d.on(r.index, "index"); d.on(status, "status");
  if (d.enter()) return d.rc;
  if (es == 2) by_width<bf16>(write, (cudaStream_t)stream, A);
  else by_width<float>(write, (cudaStream_t)stream, A);
  return d.done(cudaGetLastError());
}

}  // namespace
}  // namespace pcpb

using namespace pcpb;

extern "C" int pcpb_op_kv_write(void* stream, const pcpb_kv_cache* cache, const pcpb_kv_rows* rows, int32_t* status, char* err, size_t err_cap) {
  return kv_rows_call(true, stream, cache, rows, status, err, err_cap);
}
extern "C" int pcpb_op_kv_read(void* stream, const pcpb_kv_cache* cache, const pcpb_kv_rows* rows, int32_t* status, char* err, size_t err_cap) {
  return kv_rows_call(false, stream, cache, rows, status, err, err_cap);
}
