// Verification of drafted tokens: the walk from node 0 of a sequence's tree along the children that are taken, and the last token.
//
//   p_i = exp((z_i - max z) / T) / S;  child (t, u) taken if u q_t D < max(p_t - a q_t, 0)
//   after a refusal a += D, D = sum_i max(p_i - a q_i, 0): with r_0 = p and r_{k+1} = max(r_k - q, 0) / Z_k one finds by induction
//   r_k = max(p - a_k q, 0) / D_k with a_{k+1} = a_k + D_k, so the k-th residual needs p, q and two numbers.
//
// Bound: latency.  Only the rows of the nodes on the accepted path have to be read, one after the other, so a step's time is that of one row
// (304 KB at 151936 words): a cluster of up to 16 blocks takes a sequence, every warp a contiguous segment of the row.  Per step the warps'
// maxima and sums go to all blocks of the cluster through distributed shared memory, and after ONE cluster barrier every thread
// makes the same decision from the same numbers; buffers alternate, so the next exchange needs no second barrier.  32 trees of 24 tokens at
// 151936 words: 65 to 72 us over several runs (one block a sequence: 519).  Rows of short chains (AHEAD_N) are read before the walk, four at a time, and a step is a decision only: 16 chains of 8 at 65536 f32 words take 52 to 59 us.
//
// Precision.  Sums of a step are f32.  S is off (relative) by at most 2^-22 of exp2, three roundings of its argument, whose weighted mean
// is at most log2 V (3 ln 2 log2(V) 2^-24 = 2.1e-6), as much again and 2^-22 for each of the dozen joins of parts, and the
// additions of a thread's V / 4096 terms: below 8e-6 + V / 4096 2^-24.  A decision within twice that is made again with a 64-bit S; the
// residuals and the running sum for the last token are 64-bit throughout.  So the result is that of 64-bit arithmetic.
#include <cooperative_groups.h>
#include <math.h>

#include "common.cuh"
#include "decode_ops.h"

namespace pcpb {
namespace {

namespace cg = cooperative_groups;

constexpr int VW = 8, VT = 32 * (VW + 1);          // warps that read rows, threads of a block: one more warp looks after the children
constexpr int MAX_CL = 16;                         // blocks of a cluster
constexpr int MAX_N = PCPB_TREE_MAX_NODES;
constexpr int KEEP = 10;                           // a lane's first pieces of the last token's row, whose sums are kept for the search
constexpr int AHEAD_N = 8;                         // most nodes whose rows are all read ahead of the walk
// Reading every row before the walk pays where most of them will be walked anyway.  Ahead / one after the other: 1 chain of 6 at 50304 words 15 /
// 21 us, 32 chains of 8 at 50304 45 / 48, 16 of 8 at 65536 (f32, drafter) 52 / 54; but 1 tree of 24 at 151936 68 / 36, 16 at 65536 68 / 43.
constexpr double AHEAD_BYTES = 64e6;

struct VerifyArgs {
  pcpb_verify v;
  int32_t* status;
  int ahead;                                       // read every node's row first, walk afterwards
};

struct Stat { float m, s; int at; };               // maximum, sum of exp2((z - m) c), first index of the maximum
__device__ __forceinline__ float fast_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool GREEDY> __device__ __forceinline__ void stat_join(Stat& a, const Stat& b, float c) {
  if (GREEDY) {
    if (b.m > a.m || (b.m == a.m && b.at < a.at)) a = b;
  } else {
    const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
    a.s = a.s * fast_ex2((a.m - ref) * c) + b.s * fast_ex2((b.m - ref) * c);
    a.m = m;
  }
}

// A row of logits as 16-byte pieces: piece j holds the elements [j E - shift, (j + 1) E - shift) of the row; the first and the last may be short.
template <typename T> struct Pieces {
  static constexpr int E = 16 / sizeof(T);
  const T* z;
  int V, shift, n;
  __device__ __forceinline__ Pieces(const T* row, int vocab) : z(row), V(vocab) {
    shift = (int)(((uintptr_t)row & 15) / sizeof(T));
    n = (V + shift + E - 1) / E;
  }
  __device__ __forceinline__ int first(int j) const { return j * E - shift; }
  __device__ __forceinline__ bool inside(int j) const { return j < n && first(j) >= 0 && first(j) + E <= V; }
  __device__ __forceinline__ uint4 raw(int j) const { return inside(j) ? __ldg(reinterpret_cast<const uint4*>(z + first(j))) : make_uint4(0u, 0u, 0u, 0u); }
  // values of piece j from its raw bits, -inf where there is no element or a NaN
  __device__ __forceinline__ void values(int j, const uint4& w, float (&f)[E]) const {
    if (inside(j)) {
      const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (sizeof(T) == 2) { f[(2 * i) % E] = bf_lo(r[i]); f[(2 * i + 1) % E] = bf_hi(r[i]); }
        else f[i] = __uint_as_float(r[i]);
      }
    } else {
      const int i0 = first(j);
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = j < n && i0 + i >= 0 && i0 + i < V ? to_f<T>(z[i0 + i]) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = fmaxf(f[i], -INFINITY);
  }
  __device__ __forceinline__ void load(int j, float (&f)[E]) const { values(j, raw(j), f); }
};

// Maxima and sums of R rows' shares [j0, j1) of pieces, by a warp (a lane's own part; joined by the caller): U pieces of every row in flight per
// lane.  The pieces stay as raw bits until they are used, which keeps enough blocks on an SM.
template <typename T, bool GREEDY, int R, int U> __device__ __forceinline__ void scan(const Pieces<T> (&P)[R], const int (&j0)[R], const int (&j1)[R], float c, Stat (&a)[R]) {
  constexpr int E = Pieces<T>::E;
  int most = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) { a[r] = Stat{-INFINITY, 0.f, 0x7fffffff}; most = max(most, j1[r] - j0[r]); }
  for (int d = threadIdx.x & 31; d - (int)(threadIdx.x & 31) < most; d += 32 * U) {
    uint4 w[R][U];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int u = 0; u < U; ++u) w[r][u] = j0[r] + d + 32 * u < j1[r] ? P[r].raw(j0[r] + d + 32 * u) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float m = a[r].m;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = j0[r] + d + 32 * u;
        if (j >= j1[r]) break;
        float f[E];
        P[r].values(j, w[r][u], f);
        if (GREEDY) {
#pragma unroll
          for (int i = 0; i < E; ++i) { if (f[i] > m) a[r].at = P[r].first(j) + i; m = fmaxf(m, f[i]); }          // ascending: the first index of the maximum
        } else {
          float top = f[0];
#pragma unroll
          for (int i = 1; i < E; ++i) top = fmaxf(top, f[i]);
          if (top > m) { a[r].s *= fast_ex2((m - top) * c); m = top; }           // (a sum over nothing is 0, whatever the factor; -inf - x is -inf)
          if (m > -INFINITY) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) s += fast_ex2((f[i] - m) * c);
            a[r].s += s;
          }
        }
      }
      a[r].m = m;
    }
  }
}
template <bool GREEDY> __device__ __forceinline__ Stat warp_join(Stat a, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat b;
    b.m = __shfl_xor_sync(0xffffffffu, a.m, o); b.s = __shfl_xor_sync(0xffffffffu, a.s, o); b.at = __shfl_xor_sync(0xffffffffu, a.at, o);
    stat_join<GREEDY>(a, b, c);
  }
  // lane 0's: the lanes' sums may differ in the last bit, and every thread of the cluster has to decide from the same numbers
  a.m = __shfl_sync(0xffffffffu, a.m, 0); a.s = __shfl_sync(0xffffffffu, a.s, 0); a.at = __shfl_sync(0xffffffffu, a.at, 0);
  return a;
}

// 2^y for -1000 < y <= 0, off by at most 3e-13: y = n + f with |f| <= 1/2, Taylor's series of e^(f ln 2) to the tenth power (the next term is
// below (ln 2 / 2)^11 / 11! = 2.2e-13), and n added to the exponent.  14 operations in 64 bits; the library's exp takes about three
// times as many, and 64-bit operations are what the last token's row is bound by.
__device__ __forceinline__ double pow2_neg(double y) {
  const double t = y + 6755399441055744.0, f = y - (t - 6755399441055744.0);
  const int n = __double2loint(t);
  constexpr double L = 0.69314718055994530942, L2 = L * L, L4 = L2 * L2;
  const double f2 = f * f, f4 = f2 * f2;
  const double p0 = fma(f, L, 1.0), p1 = fma(f, L2 * L / 6.0, L2 / 2.0), p2 = fma(f, L4 * L / 120.0, L4 / 24.0), p3 = fma(f, L4 * L2 * L / 5040.0, L4 * L2 / 720.0),
               p4 = fma(f, L4 * L4 * L / 362880.0, L4 * L4 / 40320.0);
  const double q0 = fma(f2, p1, p0), q1 = fma(f2, p3, p2), q2 = fma(f2, L4 * L4 * L2 / 3628800.0, p4);
  const double r = fma(f4, fma(f4, q2, q1), q0);
  return __hiloint2double(__double2hiint(r) + (n << 20), __double2loint(r));
}

struct Shared {
  Stat stat[2][MAX_CL * VW];                       // one exchange: an entry from every warp of the cluster
  double sum[2][MAX_CL * VW];
  Stat ahead[AHEAD_N][MAX_CL];                     // AHEAD: an entry of every block for every row
  Stat mine[AHEAD_N][VW];
  long long token[MAX_N];
  float u[MAX_N];
  int16_t par[MAX_N];
  int16_t kid[MAX_N];                              // the current node's children in index order, and what a decision needs of them
  float kz[MAX_N], kq[MAX_N];
  uint8_t gone[MAX_N];                             // the child's token has no weight left
  int nkid;
  int refused[MAX_N];                              // those tokens, for the last token's sum
  double kept[VW][KEEP][32];
};

// What is left of a row's distribution: weights max(e_i - aS q_i, 0) with e_i = exp((z_i - max) / T), the refused tokens' weights 0.
template <typename T> struct Left {
  Pieces<T> P;
  const float* q;
  double zmax, log2T, aS;                           // log2T: log2(e) / T
  int nref;                                        // refused tokens: those of the first nref children with gone[] set
  __device__ __forceinline__ double weight(float z, int i, const Shared& sh) const {
    if (z == -INFINITY) return 0.0;
    const double y = ((double)z - zmax) * log2T;
    double w = y > -1000.0 ? pow2_neg(y) : exp2(y);
    if (q) { w -= aS * (double)__ldg(q + i); return w > 0.0 ? w : 0.0; }
    return w;
  }
  // weights of piece j from its raw bits
  __device__ __forceinline__ void weights(int j, const uint4& raw, const Shared& sh, double (&w)[Pieces<T>::E]) const {
    constexpr int E = Pieces<T>::E;
    float f[E];
    P.values(j, raw, f);
    const int i0 = P.first(j);
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = weight(f[i], i0 + i, sh);
#pragma unroll 1
    for (int k = 0; k < nref; ++k) {
      const unsigned d = (unsigned)(sh.refused[k] - i0);
      if (d < (unsigned)E)
#pragma unroll
        for (int i = 0; i < E; ++i) if (i == (int)d) w[i] = 0.0;
    }
  }
};

template <typename T, bool GREEDY> __global__ void __launch_bounds__(VT) k_verify(const __grid_constant__ VerifyArgs A) {
  extern __shared__ __align__(16) uint8_t verify_smem[];
  Shared& sh = *reinterpret_cast<Shared*>(verify_smem);
  cg::cluster_group cl = cg::this_cluster();
  cl.barrier_arrive();                                          // waited for before the first write into another block
  const pcpb_verify& v = A.v;
  const int CL = (int)cl.num_blocks(), rank = (int)cl.block_rank(), b = (int)blockIdx.x / CL;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = v.vocab;
  const SeqLen s = clip_seq(v.cu_nodes[b], v.cu_nodes[b + 1], 0, v.n_rows, v.max_nodes, 0);
  if (s.bad) op_note(A.status, PCPB_OPS_BAD_LENGTH);
  const int lo = s.n0, n = s.n;
  const bool writer = rank == 0 && tid == 0;
  const float c = GREEDY ? 1.f : (float)(1.4426950408889634 / v.temperature);
  for (int i = tid; i < n; i += VT) {
    int bad = 0;
    sh.par[i] = (int16_t)clip_parent(v.parent ? v.parent[lo + i] : i - 1, i, &bad);
    if (bad) op_note(A.status, PCPB_OPS_BAD_TREE);
    sh.token[i] = v.token[lo + i];
    sh.u[i] = GREEDY ? 0.f : v.u_accept[lo + i];
  }
  if (rank == 0)
    for (int i = tid; i < v.max_out; i += VT) { v.tokens_out[(size_t)b * v.max_out + i] = 0; v.path_out[(size_t)b * v.max_out + i] = -1; }
  // the warp's share of a row's n pieces
  auto share = [&](int pieces, int* j0, int* j1) {
    const int parts = CL * VW, per = (pieces + parts - 1) / parts, w = rank * VW + warp;
    *j0 = min(pieces, w * per); *j1 = warp < VW ? min(pieces, *j0 + per) : *j0;
  };
  const double slack = 1.6e-5 + V * (1.0 / 4096 / 8388608);
  int turn = 0;                                                 // buffer of the next exchange
  // an f64 value of every warp -> the sum over all, in warp order; the values stay in sh.sum[*which]
  auto exchange = [&](double x, int* which) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    if (warp < VW && lane < CL) *cl.map_shared_rank(&sh.sum[turn][rank * VW + warp], lane) = x;
    cl.sync();
    double t = 0.0;
    for (int i = lane; i < CL * VW; i += 32) t += sh.sum[turn][i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    *which = turn;
    turn ^= 1;
    return t;
  };
  const bool ahead = A.ahead && n <= AHEAD_N;
  __syncthreads();
  cl.barrier_wait();
  if (ahead && n > 0) {
    constexpr int R = 4;                                        // rows in flight
    if (warp < VW)
      for (int i = 0; i < n; i += R) {
        const T* base = (const T*)v.logits + (size_t)lo * v.logits_row;
        const Pieces<T> P[R] = {Pieces<T>(base + (size_t)i * v.logits_row, V), Pieces<T>(base + (size_t)min(i + 1, n - 1) * v.logits_row, V),
                                Pieces<T>(base + (size_t)min(i + 2, n - 1) * v.logits_row, V), Pieces<T>(base + (size_t)min(i + 3, n - 1) * v.logits_row, V)};
        int j0[R], j1[R];
        Stat a[R];
#pragma unroll
        for (int r = 0; r < R; ++r) { share(P[r].n, &j0[r], &j1[r]); if (i + r >= n) j1[r] = j0[r]; }
        scan<T, GREEDY, R, 2>(P, j0, j1, c, a);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          a[r] = warp_join<GREEDY>(a[r], c);
          if (lane == 0 && i + r < n) sh.mine[i + r][warp] = a[r];
        }
      }
    __syncthreads();
    for (int i = tid; i < n; i += VT) {
      Stat a = sh.mine[i][0];
      for (int w = 1; w < VW; ++w) stat_join<GREEDY>(a, sh.mine[i][w], c);
      for (int r = 0; r < CL; ++r) *cl.map_shared_rank(&sh.ahead[i][rank], r) = a;
    }
    cl.sync();
  }
  int node = 0, level = 0;
  while (n > 0 && level < v.max_out) {
    const T* zrow = (const T*)v.logits + (size_t)(lo + node) * v.logits_row;
    const float* qrow = !GREEDY && v.draft_probs ? v.draft_probs + (size_t)(lo + node) * v.draft_row : nullptr;
    const Pieces<T> P(zrow, V);
    int j0, j1;
    share(P.n, &j0, &j1);
    if (warp == VW) {                                           // children, while the other warps read the row
      int cnt = 0;
      if (level + 1 < v.max_out)
        for (int base = node + 1; base < n; base += 32) {
          const int i = base + lane;
          const bool is = i < n && sh.par[i] == node;
          const bool in = is && sh.token[i] >= 0 && sh.token[i] < V;
          if (is && !in) op_note(A.status, PCPB_OPS_NO_CHOICE);
          const uint32_t bal = __ballot_sync(0xffffffffu, in);
          if (in) {
            const int k = cnt + __popc(bal & ((1u << lane) - 1));
            sh.kid[k] = (int16_t)i;
            sh.gone[k] = 0;
            if (!GREEDY) { sh.kz[k] = to_f<T>(zrow[sh.token[i]]); sh.kq[k] = qrow ? qrow[sh.token[i]] : 1.f; }
          }
          cnt += __popc(bal);
        }
      if (lane == 0) sh.nkid = cnt;
    }
    Stat st;
    if (ahead) {
      __syncthreads();
      st = Stat{-INFINITY, 0.f, 0x7fffffff};
      if (lane < CL) st = sh.ahead[node][lane];
      st = warp_join<GREEDY>(st, c);
    } else {
      Stat a{-INFINITY, 0.f, 0x7fffffff};
      if (warp < VW) {
        const Pieces<T> rows[1] = {P};
        const int f0[1] = {j0}, f1[1] = {j1};
        Stat one[1];
        scan<T, GREEDY, 1, 5>(rows, f0, f1, c, one);
        a = warp_join<GREEDY>(one[0], c);
      }
      if (warp < VW && lane < CL) *cl.map_shared_rank(&sh.stat[turn][rank * VW + warp], lane) = a;
      cl.sync();
      st = Stat{-INFINITY, 0.f, 0x7fffffff};
      for (int i = lane; i < CL * VW; i += 32) stat_join<GREEDY>(st, sh.stat[turn][i], c);
      st = warp_join<GREEDY>(st, c);
      turn ^= 1;
    }
    const bool choice = isfinite(st.m);
    if (!choice && writer) op_note(A.status, PCPB_OPS_NO_CHOICE);
    int taken = -1;
    const int nkid = choice ? sh.nkid : 0;
    if (GREEDY) {
      for (int k = lane; k < nkid + lane; k += 32) {            // the first child with the winning token
        const uint32_t hit = __ballot_sync(0xffffffffu, k < nkid && sh.token[sh.kid[k < nkid ? k : 0]] == st.at);
        if (hit) { taken = sh.kid[k - lane + __ffs(hit) - 1]; break; }
      }
    }
    Left<T> left{P, qrow, (double)st.m, GREEDY ? 1.0 : 1.4426950408889634074 / v.temperature, 0.0, 0};
    double S = (double)st.s, a = 0.0, a0 = 0.0, D = 1.0;
    bool sure = false;                                          // S is a 64-bit sum
    int which;
    auto sum_left = [&]() {                                     // sum of the weights that are left
      double x = 0.0;
      left.aS = a * S;
      uint4 w0 = make_uint4(0u, 0u, 0u, 0u), w1 = w0;           // two pieces at a time, the next two on their way
      if (j0 + lane < j1) w0 = P.raw(j0 + lane);
      if (j0 + lane + 32 < j1) w1 = P.raw(j0 + lane + 32);
#pragma unroll 1
      for (int j = j0 + lane, q = 0; j < j1; j += 64, q += 2) {
        const uint4 c0 = w0, c1 = w1;
        if (j + 64 < j1) w0 = P.raw(j + 64);
        if (j + 96 < j1) w1 = P.raw(j + 96);
        double u[Pieces<T>::E], y[Pieces<T>::E];
        left.weights(j, c0, sh, u);
        if (j + 32 < j1) left.weights(j + 32, c1, sh, y);
        else
#pragma unroll
          for (int i = 0; i < Pieces<T>::E; ++i) y[i] = 0.0;
#pragma unroll
        for (int i = Pieces<T>::E / 2; i > 0; i >>= 1)
#pragma unroll
          for (int k = 0; k < i; ++k) { u[k] += u[k + i]; y[k] += y[k + i]; }
        if (q < KEEP) { sh.kept[warp][q][lane] = u[0]; sh.kept[warp][q + 1][lane] = y[0]; }
        x += u[0] + y[0];
      }
      return exchange(x, &which);
    };
    auto make_sure = [&]() {
      const float* q = left.q;
      left.q = nullptr; left.nref = 0;
      S = sum_left();
      left.q = q;
      sure = true;
    };
    if (!GREEDY && choice) {
      double e32 = 0.0;                                         // lane l: exp of child (k & ~31) + l
      for (int k = 0; k < nkid && taken < 0; ++k) {
        if ((k & 31) == 0) e32 = k + lane < nkid && sh.kz[k + lane] > -INFINITY ? exp2(((double)sh.kz[k + lane] - left.zmax) * left.log2T) : 0.0;
        const double u = sh.u[sh.kid[k]], qt = sh.kq[k], e = __shfl_sync(0xffffffffu, e32, k & 31);
        bool again = false;                                     // an earlier sibling with this token was refused: nothing is left of it
        if (!qrow) for (int i = lane; i < k + lane; i += 32) again |= __any_sync(0xffffffffu, i < k && sh.gone[i < k ? i : 0] && sh.token[sh.kid[i < k ? i : 0]] == sh.token[sh.kid[k]]);
        auto weight = [&]() { const double w = e / S - a * qt; return qrow ? (w > 0.0 ? w : 0.0) : again ? 0.0 : e / S; };
        double w = weight();
        if (!sure && (fabs(u * qt * D - w) <= slack * (u * qt + e / S) || (!qrow && D - w < 1e-4))) {
          const double S0 = S;
          make_sure();
          w = weight();
          if (!qrow) D = 1.0 - (1.0 - D) * (S0 / S);
        }
        if (u * qt * D < w) { taken = sh.kid[k]; break; }
        if (qrow) {
          a0 = a;
          a += D;
          if (k + 1 < nkid) {                                   // (after the last child the sum below does this)
            if (!sure) { make_sure(); }
            const double d = sum_left() / S;
            if (d > 0.0) D = d; else a = a0;
          }
        } else if (!again && D - w > 0.0) {
          D -= w;
          __syncwarp();
          sh.gone[k] = 1;                                       // every thread of the cluster writes the same into its block's copy
          __syncwarp();
        }
      }
    }
    if (taken < 0 && !GREEDY && choice) {                       // the last token
      if (qrow && !sure && a > 0.0) make_sure();
      __syncthreads();
      int nref = 0;
      if (!qrow)
        for (int k = 0; k < nkid; ++k)
          if (sh.gone[k]) { if (tid == 0) sh.refused[nref] = (int)sh.token[sh.kid[k]]; ++nref; }
      __syncthreads();
      left.nref = nref;
      double total = sum_left();
      if (!(total > 0.0) && (a > 0.0 || left.nref)) { a = a0; left.nref = 0; total = sum_left(); }
      // the last segment that begins at or before the goal and is not empty
      const double goal = (double)v.u_sample[b] * total;
      constexpr int PER = MAX_CL * VW / 32;
      double part[PER], inc = 0.0, before = 0.0;
      int seg = -1;
#pragma unroll
      for (int i = 0; i < PER; ++i) { part[i] = lane * PER + i < CL * VW ? sh.sum[which][lane * PER + i] : 0.0; inc += part[i]; }
      double run = inc;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(0xffffffffu, run, o); if (lane >= o) run += y; }
      run -= inc;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (part[i] > 0.0 && run <= goal) { seg = lane * PER + i; before = run; }
        run += part[i];
      }
      seg = __reduce_max_sync(0xffffffffu, seg);
      before = __shfl_sync(0xffffffffu, before, max(seg, 0) / PER);
      if (seg == rank * VW + warp) {                            // that warp looks for the index
        // the last piece that begins at or before the goal and is not empty, then the index in it
        int piece = -1;
        double at = before, begin = before;
        for (int base = j0, q = 0; base < j1; base += 32, ++q) {
          const int j = base + lane;
          double x = 0.0;
          if (j < j1) {
            if (q < KEEP) {
              x = sh.kept[warp][q][lane];
            } else {
              double w[Pieces<T>::E];
              left.weights(j, P.raw(j), sh, w);
#pragma unroll
              for (int i = 0; i < Pieces<T>::E; ++i) x += w[i];
            }
          }
          double inc = x;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) { const double y = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += y; }
          const double start = at + inc - x;
          const uint32_t here = __ballot_sync(0xffffffffu, x > 0.0 && start <= goal);
          if (here) { const int src = 31 - __clz(here); piece = base + src; begin = __shfl_sync(0xffffffffu, start, src); }
          at += __shfl_sync(0xffffffffu, inc, 31);
        }
        int hit = -1, lastpos = -1;
        if (piece >= 0) {
          double w[Pieces<T>::E], r = begin;
          left.weights(piece, P.raw(piece), sh, w);
#pragma unroll
          for (int i = 0; i < Pieces<T>::E; ++i) {
            r += w[i];
            if (w[i] > 0.0) { lastpos = P.first(piece) + i; if (hit < 0 && r > goal) hit = lastpos; }
          }
        }
        if (lane == 0) v.tokens_out[(size_t)b * v.max_out + level] = hit >= 0 ? hit : lastpos;
      }
      if (seg < 0 && writer) v.tokens_out[(size_t)b * v.max_out + level] = -1;
    }
    if (writer) {
      v.path_out[(size_t)b * v.max_out + level] = lo + node;
      if (taken >= 0) v.tokens_out[(size_t)b * v.max_out + level] = sh.token[taken];
      else if (GREEDY || !choice) v.tokens_out[(size_t)b * v.max_out + level] = choice ? st.at : -1;
    }
    ++level;
    if (taken < 0) break;
    node = taken;
    __syncthreads();                                            // the children's arrays are used again
  }
  if (writer) v.n_out[b] = level;
  cl.sync();                                                    // no block leaves while another may still write into its shared memory
}

template <typename T, bool GREEDY> cudaError_t launch(cudaStream_t st, const VerifyArgs& A) {
  // Blocks of a cluster: 512 pieces of 16 bytes a block (two rounds of its 256 reading threads), not more than 16, and no more than can be
  // resident together: two blocks an SM, and 16 only where one an SM will do, because a cluster lies within a group of 16 to 18 SMs.  With 16
  // blocks for each of 32 sequences (16 sequences) a third of the clusters began when others had ended: 81 us against 70 (65 against 50).
  const long long pieces = ((long long)A.v.vocab * (long long)sizeof(T) + 15) / 16;
  int cl = 1;
  while (cl < MAX_CL && pieces > cl * 512ll && (cl < 2 || 2ll * cl * A.v.batch <= (cl < 8 ? 2 * 148 : 148))) cl *= 2;
  static bool done[64] = {};                       // attributes of the kernel on a device, set once
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64 || !done[dev])) {
    e = cudaFuncSetAttribute(k_verify<T, GREEDY>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(k_verify<T, GREEDY>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Shared));
    if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  }
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)A.v.batch * cl); cfg.blockDim = dim3(VT); cfg.dynamicSmemBytes = sizeof(Shared); cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cl; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_verify<T, GREEDY>, A);
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
  const bool greedy = v.temperature < 1e-6, half = v.dtype == PCPB_BF16;
  A.ahead = v.max_nodes <= AHEAD_N && (double)v.n_rows * v.vocab * (half ? 2 : 4) <= AHEAD_BYTES;
  cudaStream_t st = (cudaStream_t)stream;
  return d.done(half ? (greedy ? launch<bf16, true>(st, A) : launch<bf16, false>(st, A)) : (greedy ? launch<float, true>(st, A) : launch<float, false>(st, A)));
}
