// A paged KV cache in 8 bits: rows quantised as they are written, and read back.
//
//   a = max(amax |x| / Q, 2^-126),  c = round(x / a),  value a c        Q = 448 (e4m3), 127 (signed integers)
//
// One row of a head has one scale.  Both divisions are f32 divisions rounded to nearest, so that codes and scales are the same
// bits wherever they are computed.  The scale's floor keeps it a normal number: rows of zeros get codes 0 and no division by zero,
// and rows below 2^-126 Q lose precision instead of overflowing their codes.
// A row is read once (16-byte loads, HD / 8 lanes a row, the row's largest magnitude by shuffles) and its codes are written once.
// Bound: for few rows latency (5 us a call), for many HBM by intent and issue slots in fact: 16 prompts of up to 2048 (bf16, 8 heads x 128)
// into i8 take 53 us to write (0.71 instructions a cycle, DRAM 28 %) and 40 to read back (DRAM 29 %).
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

// x / a rounded to nearest, from the correctly rounded reciprocal r of a: one product and one correction (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990, theorem on the last step of a division).  The remainder, a
// multiple of 2^-46 times the powers of two of quotient and divisor, must not fall below the smallest number, 2^-149: callers keep to
// a >= 2^-80, where it does so only for quotients below 2^-23, which become code 0.
__device__ __forceinline__ float quotient(float x, float a, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, a, x), r, q);
}
// Eight values to eight codes (two 32-bit words).
template <int CODE> __device__ __forceinline__ uint2 encode8(const float (&f)[8], float a) {
  float y[8];
  if (a >= 8.28e-25f) {
    const float r = __frcp_rn(a);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = quotient(f[i], a, r);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __fdiv_rn(f[i], a);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (CODE == PCPB_E4M3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * h], y[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * h + 2], y[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
      w[h] = lo | (hi << 16);
    } else {
      // |y| <= 127 (1 + 2^-23): adding 1.5 2^23 rounds to the nearest integer, ties to even, and leaves it in the low byte
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(y[4 * h + i] + 12582912.f);
      w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
  return make_uint2(w[0], w[1]);
}
template <int CODE> __device__ __forceinline__ void decode8(uint2 w, float (&f)[8]) {
  const uint32_t ws[2] = {w.x, w.y};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (CODE == PCPB_E4M3) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const __half2_raw p = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((ws[h] >> (16 * i)) & 0xFFFF), __NV_E4M3);
        const float2 q = __half22float2(__half2(p));
        f[4 * h + 2 * i] = q.x; f[4 * h + 2 * i + 1] = q.y;
      }
    } else {
      // the code plus 128 in the low byte of 2^23's bit pattern is the float 2^23 + 128 + code
      const uint32_t u = ws[h] ^ 0x80808080u;
      f[4 * h] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650)) - 8388736.f;
      f[4 * h + 1] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7651)) - 8388736.f;
      f[4 * h + 2] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7652)) - 8388736.f;
      f[4 * h + 3] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7653)) - 8388736.f;
    }
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

// Eight values as they lie in memory
template <typename S> struct Raw8;
template <> struct Raw8<bf16> { uint4 w; };
template <> struct Raw8<float> { uint4 w, w2; };
__device__ __forceinline__ void ld_raw(Raw8<bf16>& r, const bf16* p) { r.w = __ldg(reinterpret_cast<const uint4*>(p)); }
__device__ __forceinline__ void ld_raw(Raw8<float>& r, const float* p) { r.w = __ldg(reinterpret_cast<const uint4*>(p)); r.w2 = __ldg(reinterpret_cast<const uint4*>(p) + 1); }
__device__ __forceinline__ void to_floats(const Raw8<bf16>& r, float (&f)[8]) {
  const uint32_t w[4] = {r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = bf_lo(w[i]); f[2 * i + 1] = bf_hi(w[i]); }
}
__device__ __forceinline__ void to_floats(const Raw8<float>& r, float (&f)[8]) {
  const uint32_t w[8] = {r.w.x, r.w.y, r.w.z, r.w.w, r.w2.x, r.w2.y, r.w2.z, r.w2.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
}

// A block takes E entries: their places are found by a warp each, then groups of HD / 8 lanes take the rows (k heads, then v heads) in turn,
// one row of every entry in flight.  E = 1 for few entries (as many blocks as there are entries; up to 2048 there is no difference), more for
// many (8192 entries written into e4m3 and read back: 31 us against 33): with one entry a block the
// lookups, three loads deep, stood between a block's start and its rows (16 prompts of up to 2048 into i8, 8 heads x 128: 82 us, now 53).
template <int E> __device__ __forceinline__ void find_entries(const KvArgs& A, Entry (&en)[E], bool (&on)[E]) {
  if constexpr (E == 1) {
    on[0] = find_entry(A, (int)blockIdx.x, &en[0]);
  } else {
    __shared__ Entry found[E];
    __shared__ int ok[E];
    const int w = threadIdx.x >> 5;
    for (int k = w; k < E; k += blockDim.x >> 5) {
      const int e = (int)blockIdx.x * E + k;
      Entry x{-1, 0, 0};
      const bool have = e < A.r.n_entries && find_entry(A, e, &x);
      if ((threadIdx.x & 31) == 0) { found[k] = x; ok[k] = have; }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < E; ++k) { en[k] = found[k]; on[k] = ok[k]; }
  }
}

template <int HD, int CODE, typename S, int E> __global__ void __launch_bounds__(256) k_kv_write(const __grid_constant__ KvArgs A) {
  constexpr int L = HD / 8;                                     // lanes of a row
  Entry en[E];
  bool on[E];
  find_entries<E>(A, en, on);
  const int lane = threadIdx.x % L, Hkv = A.c.n_kv_head;
  for (int u0 = 0; u0 < 2 * Hkv; u0 += blockDim.x / L) {        // whole warps stay together: the groups of a warp exchange their maxima
    const int u = u0 + threadIdx.x / L;
    const bool isv = u >= Hkv;
    const int h = isv ? u - Hkv : u;
    const S* src = (const S*)(isv ? A.r.v : A.r.k) + (long long)h * (isv ? A.r.v_head : A.r.k_head) + lane * 8;
    const long long row = isv ? A.r.v_row : A.r.k_row;
    Raw8<S> x[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
      x[k] = {};
      if (on[k] && en[k].page >= 0 && u < 2 * Hkv) ld_raw(x[k], src + en[k].row * row);
    }
#pragma unroll
    for (int k = 0; k < E; ++k) {
      float f[8];
      to_floats(x[k], f);
      const bool mine = on[k] && en[k].page >= 0 && u < 2 * Hkv;
      const long long at = mine ? page_row(en[k].page, A.c.page_stride, h, A.c.page_tokens, en[k].off, HD) + lane * 8 : 0;
      if (CODE == PCPB_BF16) {
        if (mine) st8<bf16>((bf16*)(isv ? A.c.v : A.c.k) + at, f);
        continue;
      }
      uint32_t m = 0;                                           // magnitudes as bit patterns: NaN sorts above every number
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const bool finite = m < 0x7F800000u;
      const float a = finite ? fmaxf(__fdiv_rn(__uint_as_float(m), CodeMax<CODE>::v), 1.17549435e-38f) : __uint_as_float(0x7FC00000u);
      if (!mine) continue;
      const uint2 w = finite ? encode8<CODE == PCPB_BF16 ? PCPB_I8 : CODE>(f, a) : make_uint2(0u, 0u);
      *reinterpret_cast<uint2*>((uint8_t*)(isv ? A.c.v : A.c.k) + at) = w;
      if (lane == 0) (isv ? A.c.v_scale : A.c.k_scale)[page_row(en[k].page, A.c.scale_stride, h, A.c.page_tokens, en[k].off, 1)] = a;
    }
  }
}

// 16 bytes of codes (or of bf16) a lane and entry: with 8 a lane, not enough was in flight.  More entries a block cost the registers, and with
// them the blocks an SM, that this kernel lives on (E = 8: 79 us where E = 1 took 53).
template <int HD, int CODE, typename S, int E> __global__ void __launch_bounds__(256, 5) k_kv_read(const __grid_constant__ KvArgs A) {
  constexpr int W = CODE == PCPB_BF16 ? 8 : 16, L = HD / W;     // elements a lane, lanes a row
  Entry en[E];
  bool on[E];
  find_entries<E>(A, en, on);
  const int lane = threadIdx.x % L, Hkv = A.c.n_kv_head;
  for (int u = threadIdx.x / L; u < 2 * Hkv; u += blockDim.x / L) {
    const bool isv = u >= Hkv;
    const int h = isv ? u - Hkv : u;
    const uint8_t* const pages = (const uint8_t*)(isv ? A.c.v : A.c.k);
    const float* const scales = isv ? A.c.v_scale : A.c.k_scale;
    uint4 w[E];
    float a[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
      w[k] = make_uint4(0u, 0u, 0u, 0u); a[k] = 0.f;
      if (!on[k] || en[k].page < 0) continue;
      w[k] = __ldg(reinterpret_cast<const uint4*>(pages + (page_row(en[k].page, A.c.page_stride, h, A.c.page_tokens, en[k].off, HD) + lane * W) * (16 / W)));
      if (CODE != PCPB_BF16) a[k] = __ldg(scales + page_row(en[k].page, A.c.scale_stride, h, A.c.page_tokens, en[k].off, 1));
    }
#pragma unroll
    for (int k = 0; k < E; ++k) {
      if (!on[k]) continue;
      S* dst = (S*)(isv ? A.r.v : A.r.k) + (isv ? en[k].row * A.r.v_row + h * A.r.v_head : en[k].row * A.r.k_row + h * A.r.k_head) + lane * W;
      float f[8];
      if (CODE == PCPB_BF16) {
        to_floats(Raw8<bf16>{w[k]}, f);
        st8<S>(dst, f);
      } else {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          decode8<CODE>(half ? make_uint2(w[k].z, w[k].w) : make_uint2(w[k].x, w[k].y), f);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] *= a[k];
          st8<S>(dst + 8 * half, f);
        }
      }
    }
  }
}

template <int HD, int CODE, typename S> void launch(bool write, cudaStream_t st, const KvArgs& A) {
  const int lanes = HD / (!write && CODE != PCPB_BF16 ? 16 : 8), rows = 2 * A.c.n_kv_head * lanes, n = A.r.n_entries;
  const int threads = rows >= 256 ? 256 : (rows + 31) / 32 * 32;
  if (n <= 1024) {
    if (write) k_kv_write<HD, CODE, S, 1><<<n, threads, 0, st>>>(A);
    else k_kv_read<HD, CODE, S, 1><<<n, threads, 0, st>>>(A);
  } else {
    if (write) k_kv_write<HD, CODE, S, 4><<<(n + 3) / 4, threads, 0, st>>>(A);
    else k_kv_read<HD, CODE, S, 2><<<(n + 1) / 2, threads, 0, st>>>(A);
  }
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
