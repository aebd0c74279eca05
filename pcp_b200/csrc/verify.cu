// Verification of drafted tokens: the walk from node 0 of a sequence's tree along the children that are taken, and the last token.
//
//   p_i = exp((z_i - max z) / T) / S;  child (t, u) taken if u q_t D < max(p_t - a q_t, 0)
//   after a refusal a += D, D = sum_i max(p_i - a q_i, 0): with r_0 = p and r_{k+1} = max(r_k - q, 0) / Z_k one finds by induction
//   r_k = max(p - a_k q, 0) / D_k with a_{k+1} = a_k + D_k, so the k-th residual needs p, q and two numbers.
//
// Only the rows of the nodes on the accepted path are read.  Sums are 64-bit: a decision that hangs on the last bits of a probability then
// comes out as the definition's.
#include <math.h>

#include "common.cuh"
#include "decode_ops.h"

namespace pcpb {
namespace {

constexpr int VT = 1024;

struct VerifyArgs {
  pcpb_verify v;
  int32_t* status;
};

__device__ __forceinline__ double block_sum_d(double x, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  double s = 0.0;
  for (int i = 0; i < VT / 32; ++i) s += red[i];
  return s;
}

// Weight of index i in the distribution that is left: row z, draft row q, a, and the refused tokens
template <typename T> struct Row {
  const T* z;
  const float* q;
  double zmax, invT, invS, a;
  __device__ __forceinline__ double p(int i) const {
    const double x = (double)to_f<T>(z[i]);
    return x == x ? exp((x - zmax) * invT) * invS : 0.0;
  }
  __device__ __forceinline__ double w(int i) const {
    if (!q) return p(i);
    const double r = p(i) - a * (double)q[i];
    return r > 0.0 ? r : 0.0;
  }
};

template <typename T> __global__ void __launch_bounds__(VT) k_verify(const __grid_constant__ VerifyArgs A) {
  __shared__ double red[VT / 32];
  __shared__ float bv[VT / 32];
  __shared__ int bi[VT / 32];
  __shared__ int16_t par[PCPB_TREE_MAX_NODES];
  __shared__ int refused[PCPB_TREE_MAX_NODES];
  __shared__ int pick;
  const pcpb_verify& v = A.v;
  const int b = blockIdx.x, tid = threadIdx.x, V = v.vocab;
  const SeqLen s = clip_seq(v.cu_nodes[b], v.cu_nodes[b + 1], 0, v.n_rows, v.max_nodes, 0);
  if (s.bad) op_note(A.status, PCPB_OPS_BAD_LENGTH);
  const int lo = s.n0, n = s.n;
  for (int i = tid; i < n; i += VT) {
    int bad = 0;
    par[i] = (int16_t)clip_parent(v.parent ? v.parent[lo + i] : i - 1, i, &bad);
    if (bad) op_note(A.status, PCPB_OPS_BAD_TREE);
  }
  for (int i = tid; i < v.max_out; i += VT) { v.tokens_out[(size_t)b * v.max_out + i] = 0; v.path_out[(size_t)b * v.max_out + i] = -1; }
  __syncthreads();
  const bool greedy = v.temperature < 1e-6;
  int node = 0, level = 0;
  while (n > 0 && level < v.max_out) {
    Row<T> row;
    row.z = (const T*)v.logits + (size_t)(lo + node) * v.logits_row;
    row.q = v.draft_probs && !greedy ? v.draft_probs + (size_t)(lo + node) * v.draft_row : nullptr;
    // first maximum
    float best = -INFINITY;
    int at = 0x7fffffff;
    for (int i = tid; i < V; i += VT) { const float x = to_f<T>(row.z[i]); if (x > best) { best = x; at = i; } }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int oi = __shfl_xor_sync(0xffffffffu, at, o);
      if (ov > best || (ov == best && oi < at)) { best = ov; at = oi; }
    }
    __syncthreads();
    if ((tid & 31) == 0) { bv[tid >> 5] = best; bi[tid >> 5] = at; }
    __syncthreads();
    best = bv[0]; at = bi[0];
    for (int k = 1; k < VT / 32; ++k) if (bv[k] > best || (bv[k] == best && bi[k] < at)) { best = bv[k]; at = bi[k]; }
    const bool choice = isfinite(best);
    int taken = -1, nref = 0;
    long long last = choice ? at : -1;
    if (!choice && tid == 0) op_note(A.status, PCPB_OPS_NO_CHOICE);
    if (choice && !greedy) {
      row.zmax = best; row.invT = 1.0 / v.temperature; row.a = 0.0; row.invS = 1.0;
      double s = 0.0;
      for (int i = tid; i < V; i += VT) s += row.p(i);
      row.invS = 1.0 / block_sum_d(s, red);
    }
    double D = 1.0;
    if (choice && level + 1 < v.max_out)
      for (int c = node + 1; c < n && taken < 0; ++c) {
        if (par[c] != node) continue;
        const long long t = v.token[lo + c];
        if (t < 0 || t >= V) { if (tid == 0) op_note(A.status, PCPB_OPS_NO_CHOICE); continue; }
        if (greedy) { if (t == at) taken = c; continue; }
        bool gone = false;
        for (int k = 0; k < nref; ++k) gone |= refused[k] == (int)t;
        const double w = gone ? 0.0 : row.w((int)t);
        if ((double)v.u_accept[lo + c] * (row.q ? (double)row.q[t] : 1.0) * D < w) { taken = c; continue; }
        if (row.q) {
          const double a0 = row.a;
          row.a += D;
          double s = 0.0;
          for (int i = tid; i < V; i += VT) s += row.w(i);
          s = block_sum_d(s, red);
          if (s > 0.0) D = s; else row.a = a0;
        } else if (!gone && D - w > 0.0) {
          D -= w;
          __syncthreads();
          if (tid == 0) refused[nref] = (int)t;
          ++nref;
          __syncthreads();
        }
      }
    if (choice && taken < 0 && !greedy) {                       // the last token
      const int per = (V + VT - 1) / VT, i0 = min(V, tid * per), i1 = min(V, i0 + per);
      auto weight = [&](int i) { for (int k = 0; k < nref; ++k) if (refused[k] == i) return 0.0; return row.w(i); };
      double s = 0.0;
      int lastpos = -1;
      for (int i = i0; i < i1; ++i) { const double w = weight(i); s += w; if (w > 0.0) lastpos = i; }
      double inc = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(0xffffffffu, inc, o); if ((tid & 31) >= o) inc += y; }
      __syncthreads();
      if ((tid & 31) == 31) red[tid >> 5] = inc;
      if (tid == 0) pick = -1;
      __syncthreads();
      double before = 0.0, total = 0.0;
      for (int k = 0; k < VT / 32; ++k) { if (k < (tid >> 5)) before += red[k]; total += red[k]; }
      const double goal = (double)v.u_sample[b] * total, excl = before + inc - s;
      if (lastpos >= 0 && excl <= goal) {                       // the last such chunk holds the index (or rounding put it just before)
        double run = excl;
        int hit = lastpos;
        for (int i = i0; i < i1; ++i) { run += weight(i); if (run > goal) { hit = i; break; } }
        atomicMax(&pick, hit);
      }
      __syncthreads();
      last = pick;
    }
    if (tid == 0) {
      v.path_out[(size_t)b * v.max_out + level] = lo + node;
      v.tokens_out[(size_t)b * v.max_out + level] = taken >= 0 ? v.token[lo + taken] : last;
    }
    ++level;
    if (taken < 0) break;
    node = taken;
    __syncthreads();
  }
  if (tid == 0) v.n_out[b] = level;
}

}  // namespace
}  // namespace pcpb

using namespace pcpb;

extern "C" int pcpb_op_verify_drafts(void* stream, const pcpb_verify* args, int32_t* status, char* err, size_t cap) {
  if (err && cap) err[0] = 0;
  if (!args) return op_fail(err, cap, PCPB_E_INVALID, "null arguments");
  VerifyArgs A;
  A.v = *args; A.status = status;
  const pcpb_verify& v = A.v;
  if (v.dtype != PCPB_BF16 && v.dtype != PCPB_F32) return op_fail(err, cap, PCPB_E_INVALID, "logits must be bf16 or f32");
  if (v.vocab < 1 || v.n_rows < 0 || v.batch < 0 || v.max_out < 1 || v.max_nodes < 1) return op_fail(err, cap, PCPB_E_INVALID, "bad sizes");
  if (v.max_nodes > PCPB_TREE_MAX_NODES) return op_fail(err, cap, PCPB_E_TOO_LARGE, "at most %d nodes a sequence", PCPB_TREE_MAX_NODES);
  if (!(v.temperature >= 0.0) || v.temperature > 1e30) return op_fail(err, cap, PCPB_E_INVALID, "temperature must be a finite number >= 0");
  if (v.batch == 0) return PCPB_OK;
  if ((v.n_rows && (!v.logits || !v.token)) || !v.cu_nodes || !v.tokens_out || !v.path_out || !v.n_out) return op_fail(err, cap, PCPB_E_INVALID, "null argument");
  if (v.n_rows && v.temperature >= 1e-6 && (!v.u_accept || !v.u_sample)) return op_fail(err, cap, PCPB_E_INVALID, "sampling needs u_accept and u_sample");
  if (v.logits_row < v.vocab || (v.draft_probs && v.draft_row < v.vocab)) return op_fail(err, cap, PCPB_E_INVALID, "rows overlap (row stride below vocab)");
  OpDevice d(err, cap);
  d.on(v.logits, "logits"); d.on(v.draft_probs, "draft_probs"); d.on(v.cu_nodes, "cu_nodes"); d.on(v.parent, "parent"); d.on(v.token, "token");
  d.on(v.u_accept, "u_accept"); d.on(v.u_sample, "u_sample"); d.on(v.tokens_out, "tokens_out"); d.on(v.path_out, "path_out"); d.on(v.n_out, "n_out");
  d.on(status, "status");
  if (d.enter()) return d.rc;
  if (v.dtype == PCPB_BF16) k_verify<bf16><<<v.batch, VT, 0, (cudaStream_t)stream>>>(A);
  else k_verify<float><<<v.batch, VT, 0, (cudaStream_t)stream>>>(A);
  return d.done(cudaGetLastError());
}
