// Attention of the nodes of drafted trees over a paged cache in bf16 or 8 bits.
//
//   out_i = sum_j w_ij v_j,  w_ij = exp2(z_ij - m_i) / l_i,  z_ij = scale log2(e) a_j (q_i . c_j),  m_i = max_j z_ij,  l_i = sum_j exp2(z_ij - m_i)
//
// in one pass over the keys with the running maximum and sum of a row (a_j: the key's scale, c_j its codes; values enter as
// (w_ij b_j) d_j with b_j their scale).  Where a row's keys are split, the parts (O, m, l) are joined by
//   m = max m_s,  l = sum exp2(m_s - m) l_s,  O = sum exp2(m_s - m) O_s.
//
// Work.  The rows of one item are those of a sequence's nodes and of the query heads of one kv head, node-major (row = node G + head),
// in tiles of ROWS; its keys are the cached positions, then the nodes, in tiles of TILE.  All tiles of all items are laid end
// to end, and block c of the grid takes the c-th equal share of them (or one whole item: make_plan): ragged contexts balance, and one
// long context spreads over the whole GPU.  Lengths are read on the device, so the grid does not depend on them.  An item that lies in one block is
// finished there; the parts of the others go to the workspace (a block has at most two of them: the item it begins in and the
// one it ends in) and k_tree_join adds them up in block order, so results do not depend on timing.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "decode_ops.h"
#include "tc_common.cuh"

namespace pcpb {
namespace {

constexpr int TILE = 128;            // keys of a scheduling step
constexpr int MAX_NODES = PCPB_TREE_MAX_NODES, MAX_BATCH = PCPB_TREE_MAX_BATCH;
constexpr int SLACK_FEW = 2, SLACK_MANY = 6;      // make_plan: what a segment and the join cost, in tiles of either kernel
constexpr float LN2 = 0.69314718055994531f, LOG2E = 1.4426950408889634f;

struct AttnArgs {
  pcpb_kv_cache c;
  pcpb_tree_attn a;
  int32_t* status;
  int G;                             // query heads of a kv head
  long long* plan;                   // workspace: [batch + 2] first tile of every sequence, all tiles, pitch
  float* part_ml;                    // [blocks][2][ROWS][2] maximum and sum
  float* part_o;                     // [blocks][2][ROWS][HD]
};

// Programmatic dependent launch: the join's blocks may be set up while the attention kernel drains; they wait for its results themselves.
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Pairs of f32 in one 64-bit register: one instruction for both.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pk2(float a, float b) { f32x2 d; asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b)); return d; }
__device__ __forceinline__ void un2(f32x2 a, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) { f32x2 d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) { f32x2 d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) { f32x2 d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ float max3(float a, float b, float c) { float d; asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c)); return d; }
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t bsub2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void mma16816_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four codes in a word -> two pairs of bf16 (exact: both code types have fewer significant bits than bf16).
//   e4m3: sign and the seven other bits move to the bf16 fields of the same name; the exponent's bias then differs by
//         127 - 7 = 120, which one product with 2^120 repairs, for subnormal codes as well.
//   i8:   with c7 the sign bit and c the other seven, 0x4300 + c is 128 + c and 0x4300 + (c7 << 7) is 128 or 256; the code is their difference.
template <int CODE> __device__ __forceinline__ void widen4(uint32_t w, uint32_t& p01, uint32_t& p23) {
  if (CODE == PCPB_E4M3) {
    const uint32_t hi = (w & 0x80808080u) | ((w >> 4) & 0x07070707u), lo = (w << 4) & 0xF0F0F0F0u;    // the high and the low bytes of the four
    p01 = bmul2(__byte_perm(lo, hi, 0x5140), 0x7B807B80u);
    p23 = bmul2(__byte_perm(lo, hi, 0x7362), 0x7B807B80u);
  } else {
    const uint32_t t0 = __byte_perm(w, 0, 0x4140), t1 = __byte_perm(w, 0, 0x4342);
    p01 = bsub2((t0 & 0x007F007Fu) | 0x43004300u, (t0 & 0x00800080u) | 0x43004300u);
    p23 = bsub2((t1 & 0x007F007Fu) | 0x43004300u, (t1 & 0x00800080u) | 0x43004300u);
  }
}

// Four codes in a word -> two pairs of f16 (exact as well), which takes fewer operations: e4m3 has an instruction, and with u = code + 128 in
// the low byte of 1024's bit pattern an i8 code is (1024 + u) - 1152.  Keys are widened this way, against q in f16; values are not, because
// the weights they meet (times the values' scales) need bf16's range.
template <int CODE> __device__ __forceinline__ void widen4_f16(uint32_t w, uint32_t& p01, uint32_t& p23) {
  if (CODE == PCPB_E4M3) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(p01), "=r"(p23) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p01) : "r"(__byte_perm(u, 0x64646464u, 0x4140)), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(p23) : "r"(__byte_perm(u, 0x64646464u, 0x4342)), "r"(0x64806480u));
  }
}
// Rows of bf16 become f16 times a power of two that puts the row's largest magnitude into [2^15, 2^16): exact for elements down to 2^-29 of it,
// and off by at most 2^-40 of it below.  exp15: 15 - exponent of the largest magnitude (bit pattern `top` of its bf16); rows with an
// infinity or a NaN are not scaled (their scores are not numbers either way).
__device__ __forceinline__ int exp15(uint32_t top) {
  const int e = (int)(top >> 7) - 127;
  return e > 127 ? 0 : 15 - max(e, -100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }       // -126 <= e <= 127
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t w, float f) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(bf_hi(w) * f), "f"(bf_lo(w) * f));
  return d;
}
__device__ __forceinline__ uint32_t top_abs2(uint32_t m, uint32_t w) { return max(m, max(w & 0x7FFFu, (w >> 16) & 0x7FFFu)); }

// Clipped lengths of sequence b.
typedef SeqLen Seq;
__device__ __forceinline__ Seq seq_of(const AttnArgs& A, int b) {
  const Seq s = clip_seq(A.a.cu_nodes[b], A.a.cu_nodes[b + 1], A.a.ctx_len[b], A.a.n_rows, A.a.max_nodes, A.c.max_pages * A.c.page_tokens);
  if (s.bad) op_note(A.status, PCPB_OPS_BAD_LENGTH);
  return s;
}
__device__ __forceinline__ int tiles_of(int x) { return (x + TILE - 1) / TILE; }

// plan[b] = first tile of sequence b, plan[batch] = all tiles, plan[batch + 1] = pitch; by the whole block, into shared memory.
// pitch > 0: every block takes one whole item, whose tiles are counted as `pitch` of them (the longest item's).  That is the better cut where
// there are no more items than blocks and the longest is at most `slack` tiles above the equal share, because a second segment of a block
// (rows of q, outputs, filling the pipeline) and the join cost about that many.  24 drafts on 16 sequences of 2048 (bf16): 49 us cut
// into equal shares, 43 with whole items; chains of 130 on 8 sequences of 1000, 16 heads x 64: 58 and 47.
template <int ROWS> __device__ void make_plan(const AttnArgs& A, long long* plan, int slack) {
  __shared__ long long wsum[32], wtiles[32];
  __shared__ int witems[32], wmost[32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long tiles = 0;
  int items = 0, most = 0;
  for (int b = threadIdx.x; b < A.c.batch; b += blockDim.x) {
    const Seq s = seq_of(A, b);
    const int T = tiles_of(s.ctx) + tiles_of(s.n), n = (s.n * A.G + ROWS - 1) / ROWS * A.c.n_kv_head;
    tiles += (long long)n * T;
    items += n;
    if (n) most = max(most, T);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    items += __shfl_xor_sync(0xffffffffu, items, o);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
  }
  if (lane == 0) { wtiles[w] = tiles; witems[w] = items; wmost[w] = most; }
  __syncthreads();
  tiles = 0; items = 0; most = 0;
  for (int i = 0; i < nw; ++i) { tiles += wtiles[i]; items += witems[i]; most = max(most, wmost[i]); }
  const int pitch = items <= (int)gridDim.x && most <= tile_share(tiles, gridDim.x) + slack ? most : 0;
  long long base = 0;
  for (int b0 = 0; b0 < A.c.batch; b0 += blockDim.x) {
    const int b = b0 + threadIdx.x;
    long long x = 0;
    if (b < A.c.batch) {
      const Seq s = seq_of(A, b);
      x = (long long)((s.n * A.G + ROWS - 1) / ROWS) * A.c.n_kv_head * (pitch ? pitch : tiles_of(s.ctx) + tiles_of(s.n));
    }
    long long inc = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += y; }
    if (lane == 31) wsum[w] = inc;
    __syncthreads();
    long long before = base, all = base;
    for (int i = 0; i < nw; ++i) { if (i < w) before += wsum[i]; all += wsum[i]; }
    if (b < A.c.batch) plan[b] = before + inc - x;
    base = all;
    __syncthreads();
  }
  if (threadIdx.x == 0) { plan[A.c.batch] = base; plan[A.c.batch + 1] = pitch; }
  __syncthreads();
}
// Tiles of a block's share
__device__ __forceinline__ long long share_of(const long long* plan, int batch, int blocks) {
  return plan[batch + 1] ? plan[batch + 1] : tile_share(plan[batch], blocks);
}
// The sequence tile t belongs to: plan[b] <= t < plan[b + 1]
__device__ __forceinline__ int seq_at(const long long* plan, int batch, long long t) {
  int lo = 0, hi = batch;                                       // plan[lo] <= t < plan[hi]
  while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (plan[mid] <= t) lo = mid; else hi = mid; }
  return lo;
}

// ---- the kernel for few rows: 8 a tile, mma.sync ---------------------------------------------------------------------
// The warps of a block share the 8 rows and split the keys in units of 16: no barrier until the item ends.  Keys and values are the 16-row
// operands of mma.sync m16n8k16 (S^T = K Q^T, O^T = V^T P^T), the rows of q its 8 columns.  A lane's 16-byte pieces of keys and values are
// what it needs as fragments: which of the head_dim elements meet in one k16 step does not matter as long as q is read with the
// same assignment, and which output columns a lane holds does not matter as long as they are stored where they belong; so no element
// changes lanes, and a lane reads back from shared memory only what it copied there itself.  Values are paired by position with
// byte permutes, the weights change from accumulator to operand with movmatrix.
// Bound: the widening of 8-bit codes (16 sequences of 8192 e4m3 positions, 32 q / 8 kv heads x 128: 64 us, DRAM 41 %, ALU pipe 48 %); HBM
// for bf16.  Every warp keeps a ring of units in flight with cp.async (130 to 200 KB an SM); the block-table entries are read one unit
// ahead of that.  With 16 rows a tile, keys as the other operand and loads straight into registers the same case took 131 us, with the
// ring 101, with 8 rows a tile and sixteen warps 76, with the keys in f16 68.
constexpr int RW = 8;                // rows of a tile

template <int HD, int CODE> struct Frag {
  static constexpr int ES = CODE == PCPB_BF16 ? 2 : 1;
  static constexpr int WARPS = CODE == PCPB_BF16 ? 8 : 16;
  static constexpr int KB = HD * ES / 4 < 16 ? HD * ES / 4 : 16, KE = KB / ES, KC = HD / (4 * KE);   // bytes, elements of a lane's key piece; pieces a row
  static constexpr int VB = HD * ES / 8 < 16 ? HD * ES / 8 : 16, VE = VB / ES, VC = HD / (8 * VE);
};
template <int BYTES> __device__ __forceinline__ void ld_bytes(const void* p, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 16) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
  else if constexpr (BYTES == 8) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
  else w[0] = *reinterpret_cast<const uint32_t*>(p);
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {     // an 8 x 8 tile of 16-bit values, a row in four lanes
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// m, l, zs: rows 2 qd, 2 qd + 1 (l: this lane's share); o[t][k]: row 2 qd + (k & 1), column out_col(t, g, k >> 1)
template <int HD> struct RowState {
  uint32_t q[HD / 16][2];
  float o[HD / 16][4], m[2], l[2], zs[2];                        // zs: factor of a row's scores
};
template <int HD, int CODE> __device__ __forceinline__ int out_col(int t, int g, int i) {
  typedef Frag<HD, CODE> F;
  return (t / (F::VE / 2)) * 8 * F::VE + g * F::VE + t % (F::VE / 2) * 2 + i;
}

// q fragments of rows row0 .. row0 + 7 (row g in the lanes 4 g ..) in the element order of Frag<HD, CODE>
template <int HD, int CODE> __device__ __forceinline__ void load_q(const AttnArgs& A, const Seq& s, int kvh, int row0, RowState<HD>& R) {
  typedef Frag<HD, CODE> F;
  const int lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3, r = row0 + g;
  const bf16* p = (const bf16*)A.a.q + (long long)(s.n0 + r / A.G) * A.a.q_row + (long long)(kvh * A.G + r % A.G) * A.a.q_head;
#pragma unroll
  for (int st = 0; st < HD / 16; ++st) {
    const int e = 4 * F::KE * (st / (F::KE / 4)) + F::KE * qd + 4 * (st % (F::KE / 4));
    const uint2 v = r < s.n * A.G ? *reinterpret_cast<const uint2*>(p + e) : make_uint2(0u, 0u);
    R.q[st][0] = v.x; R.q[st][1] = v.y;
  }
  R.zs[0] = R.zs[1] = A.a.scale * LOG2E;
  if (CODE != PCPB_BF16) {                                      // q in f16, scaled by a power of two per row
    uint32_t top = 0;
#pragma unroll
    for (int st = 0; st < HD / 16; ++st) top = top_abs2(top_abs2(top, R.q[st][0]), R.q[st][1]);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = exp15(top);
#pragma unroll
    for (int st = 0; st < HD / 16; ++st) { R.q[st][0] = bf16x2_to_f16x2(R.q[st][0], pow2(e)); R.q[st][1] = bf16x2_to_f16x2(R.q[st][1], pow2(e)); }
#pragma unroll
    for (int j = 0; j < 2; ++j) R.zs[j] *= pow2(-__shfl_sync(0xffffffffu, e, 4 * (2 * qd + j)));
  }
}

// One unit of 16 keys.  load_k(j, c, w), load_v(j, c, w): this lane's pieces of its rows of keys (positions g, g + 8 of the unit) and values
// (2 qd, 2 qd + 1, 8 + 2 qd, 9 + 2 qd); zeros where there is no row.  ks, vs: scales of the positions g and g + 8.  keep: bit 2 i + j: may
// row 2 qd + j attend position g + 8 i; zero: the same for slots that count as a zero key and value.
// The reference maximum of a row moves only when a score passes it by 2^8, so that the outputs are rarely rescaled.
// TREE: rows attend different keys of the unit.  A weight of 0 does not keep an infinity or a NaN of another branch's value out of the
// matrix product, so a unit with such a value adds its products one by one (vrow: the rows of the values), attended ones only.
template <int HD, int CODE, bool TREE, typename LK, typename LV>
__device__ __forceinline__ void unit(RowState<HD>& R, const LK& load_k, const LV& load_v, const uint8_t* const (&vrow)[4], const float (&ks)[2],
                                     const float (&vs)[2], uint32_t keep, uint32_t zero) {
  typedef Frag<HD, CODE> F;
  const int lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
  float s[4] = {0.f, 0.f, 0.f, 0.f};                            // s[2 i + j]: position g + 8 i, row 2 qd + j
#pragma unroll
  for (int c = 0; c < F::KC; ++c) {
    uint32_t k0[F::KB / 4], k1[F::KB / 4];
    load_k(0, c, k0);
    load_k(1, c, k1);
#pragma unroll
    for (int sub = 0; sub < F::KE / 4; ++sub) {
      const int st = c * (F::KE / 4) + sub;
      uint32_t a[4];
      if (CODE == PCPB_BF16) { a[0] = k0[(2 * sub) % (F::KB / 4)]; a[2] = k0[(2 * sub + 1) % (F::KB / 4)]; a[1] = k1[(2 * sub) % (F::KB / 4)]; a[3] = k1[(2 * sub + 1) % (F::KB / 4)]; }
      else { widen4_f16<CODE>(k0[sub % (F::KB / 4)], a[0], a[2]); widen4_f16<CODE>(k1[sub % (F::KB / 4)], a[1], a[3]); }
      if (CODE == PCPB_BF16) mma16816(s, a, R.q[st][0], R.q[st][1]);
      else mma16816_f16(s, a, R.q[st][0], R.q[st][1]);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      s[2 * i + j] *= R.zs[j] * ks[i];
      if (TREE && (zero >> (2 * i + j)) & 1u) s[2 * i + j] = 0.f;
      if (!((keep >> (2 * i + j)) & 1u)) s[2 * i + j] = -INFINITY;
    }
  float top[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
  if (__any_sync(0xffffffffu, top[0] > R.m[0] + 8.f || top[1] > R.m[1] + 8.f || (R.m[0] == -INFINITY && top[0] > -INFINITY) || (R.m[1] == -INFINITY && top[1] > -INFINITY))) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) top[j] = fmaxf(top[j], __shfl_xor_sync(0xffffffffu, top[j], o));
      const float m = R.m[j], to = fmaxf(m, top[j]), corr = m == -INFINITY ? 1.f : ex2(m - to);      // (nothing but zeros so far: any factor will do)
      R.m[j] = to;
      R.l[j] *= corr;
#pragma unroll
      for (int t = 0; t < HD / 16; ++t) { R.o[t][j] *= corr; R.o[t][2 + j] *= corr; }
    }
  }
  float w[4];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const float ref = R.m[j] == -INFINITY ? 0.f : R.m[j];       // a row that has seen nothing yet: every weight is 0
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float e = ex2(s[2 * i + j] - ref);
      R.l[j] += e;
      w[2 * i + j] = TREE && (zero >> (2 * i + j)) & 1u ? 0.f : CODE == PCPB_BF16 ? e : e * vs[i];
    }
  }
  const uint32_t b0 = transpose8(pack2(w[0], w[1])), b1 = transpose8(pack2(w[2], w[3]));
  uint32_t vw[4][F::VC][F::VB / 4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int c = 0; c < F::VC; ++c) load_v(j, c, vw[j][c]);
  if (TREE) {
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int c = 0; c < F::VC; ++c)
#pragma unroll
        for (int i = 0; i < F::VB / 4; ++i) odd |= (vw[j][c][i] & 0x7F80u) == 0x7F80u || (vw[j][c][i] & 0x7F800000u) == 0x7F800000u;
    if (__any_sync(0xffffffffu, odd)) {
#pragma unroll 1
      for (int pos = 0; pos < 16; ++pos) {                      // its weights are with the lanes 4 (pos & 7) + qd, its value's row with the lanes whose qd is x
        const int src = (pos & 7) * 4 + qd, x = (pos & 7) >> 1;
        const uint8_t* row = (pos & 8) ? ((pos & 1) ? vrow[3] : vrow[2]) : ((pos & 1) ? vrow[1] : vrow[0]);
        const bf16* v = (const bf16*)__shfl_sync(0xffffffffu, (unsigned long long)row, x);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float wt = __shfl_sync(0xffffffffu, bf16_round((pos & 8) ? w[2 + j] : w[j]), src);
          const uint32_t on = __shfl_sync(0xffffffffu, keep & ~zero, src) >> (((pos & 8) ? 2 : 0) + j) & 1u;
          if (!on) continue;
#pragma unroll
          for (int t = 0; t < HD / 16; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) R.o[t][2 * i + j] += wt * to_f(v[out_col<HD, CODE>(t, g, i)]);
        }
      }
      return;
    }
  }
#pragma unroll
  for (int c = 0; c < F::VC; ++c)
#pragma unroll
    for (int i = 0; i < F::VB / 4; ++i) {
      if (CODE == PCPB_BF16) {
        const uint32_t a[4] = {__byte_perm(vw[0][c][i], vw[1][c][i], 0x5410), __byte_perm(vw[0][c][i], vw[1][c][i], 0x7632),
                               __byte_perm(vw[2][c][i], vw[3][c][i], 0x5410), __byte_perm(vw[2][c][i], vw[3][c][i], 0x7632)};
        mma16816(R.o[c * (F::VE / 2) + i], a, b0, b1);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t a[4];
          widen4<CODE>(__byte_perm(vw[0][c][i], vw[1][c][i], h ? 0x7362 : 0x5140), a[0], a[1]);
          widen4<CODE>(__byte_perm(vw[2][c][i], vw[3][c][i], h ? 0x7362 : 0x5140), a[2], a[3]);
          mma16816(R.o[c * (F::VE / 2) + 2 * i + h], a, b0, b1);
        }
      }
    }
}

// Ancestors-or-self of the nodes of a tile's rows, 256 bits a row, in shared memory
__device__ void make_ancestors(const AttnArgs& A, const Seq& s, int row0, int rows_tile, int16_t* par, uint32_t (*anc)[MAX_NODES / 32]) {
  for (int i = threadIdx.x; i < s.n; i += blockDim.x) {
    int bad = 0;
    par[i] = (int16_t)clip_parent(A.a.parent ? A.a.parent[s.n0 + i] : i - 1, i, &bad);
    if (bad) op_note(A.status, PCPB_OPS_BAD_TREE);
  }
  __syncthreads();
  for (int r = threadIdx.x; r < rows_tile; r += blockDim.x) {
    uint32_t w[MAX_NODES / 32] = {};
    int i = (row0 + r) / A.G;
    if (i < s.n)
      while (i >= 0) {                                          // parents come before their children: at most n steps
#pragma unroll
        for (int k = 0; k < MAX_NODES / 32; ++k) w[k] |= (i >> 5) == k ? 1u << (i & 31) : 0u;
        i = par[i];
      }
#pragma unroll
    for (int k = 0; k < MAX_NODES / 32; ++k) anc[r][k] = w[k];
  }
  __syncthreads();
}

template <int BYTES> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool on) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(on ? BYTES : 0), "n"(BYTES) : "memory");
}
// A warp's ring: stages of one unit (keys, values, 16 key scales, 16 value scales, the valid positions); the same memory holds the warp's part
// of the outputs when the item ends.
template <int HD, int CODE> struct Ring {
  typedef Frag<HD, CODE> F;
  static constexpr int K_BYTES = 16 * HD * F::ES, STAGE = 2 * K_BYTES + 144;
  static constexpr int FIT = 204000 / F::WARPS / STAGE, NST = FIT < 6 ? FIT : 6;
  static constexpr int OUT = RW * HD * 4, BYTES = NST * STAGE > OUT ? NST * STAGE : OUT;
};

template <int HD, int CODE> __global__ void __launch_bounds__(Frag<HD, CODE>::WARPS * 32, 1) k_tree_rows(const __grid_constant__ AttnArgs A) {
  typedef Frag<HD, CODE> F;
  typedef Ring<HD, CODE> G;
  constexpr int WARPS = F::WARPS;
  extern __shared__ __align__(16) uint8_t smem[];
  long long* plan = reinterpret_cast<long long*>(smem);                       // [batch + 2]
  uint8_t* rings = smem + ((A.c.batch + 2) * 8 + 15) / 16 * 16;
  __shared__ float mml[WARPS][RW][2];
  __shared__ int16_t par[MAX_NODES];
  __shared__ uint32_t anc[RW][MAX_NODES / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, qd = lane & 3;
  uint8_t* const ring = rings + warp * G::BYTES;
  float* const mine = reinterpret_cast<float*>(ring);           // [RW][HD]
  const uint32_t ring_s = smem_u32(ring);
  pdl_launch_dependents();
  make_plan<RW>(A, plan, SLACK_FEW);
  const long long total = plan[A.c.batch], per = share_of(plan, A.c.batch, gridDim.x);
  if (blockIdx.x == 0) for (int b = threadIdx.x; b < A.c.batch + 2; b += blockDim.x) A.plan[b] = plan[b];
  const long long w0 = per * blockIdx.x, w1 = min(total, w0 + per);
  for (long long w = w0; w < w1;) {
    const int b = seq_at(plan, A.c.batch, w);
    const Seq s = seq_of(A, b);
    const int ct = tiles_of(s.ctx), T = ct + tiles_of(s.n), RT = (s.n * A.G + RW - 1) / RW;
    const int pitch = (int)plan[A.c.batch + 1], P = pitch ? pitch : T;
    const long long at = w - plan[b], item = at < 0x7fffffffll ? (long long)((unsigned)at / (unsigned)P) : at / P;
    const int t0 = (int)(at - item * P), t1 = (int)min((long long)T, t0 + (w1 - w));
    const int kvh = (int)item / RT, row0 = ((int)item - kvh * RT) * RW, rows = s.n * A.G;
    RowState<HD> R;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) R.o[t][0] = R.o[t][1] = R.o[t][2] = R.o[t][3] = 0.f;
    R.m[0] = R.m[1] = -INFINITY; R.l[0] = R.l[1] = 0.f;
    // the nodes' own keys (bf16)
    if (t1 > ct) {
      make_ancestors(A, s, row0, RW, par, anc);
      load_q<HD, PCPB_BF16>(A, s, kvh, row0, R);
      const int lo = max(t0 - ct, 0) * TILE, end = min(s.n, (t1 - ct) * TILE);
      const float one[2] = {1.f, 1.f};
      typedef Frag<HD, PCPB_BF16> B;
      for (int u = lo + warp * 16; u < end; u += WARPS * 16) {
        const uint8_t *krow[2], *vrow[4];
        uint32_t keep = 0, zero = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int at = u + 8 * i + g;
          krow[i] = at < end ? (const uint8_t*)((const bf16*)A.a.k + (long long)(s.n0 + at) * A.a.k_row + (long long)kvh * A.a.k_head) : nullptr;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int r = 2 * qd + j;
            if (at < end && ((anc[r][(at >> 5) & 7] >> (at & 31)) & 1u)) keep |= 1u << (2 * i + j);
            if (A.a.null_self && at == (row0 + r) / A.G) zero |= 1u << (2 * i + j);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = u + 8 * (j >> 1) + 2 * qd + (j & 1);
          vrow[j] = i < end ? (const uint8_t*)((const bf16*)A.a.v + (long long)(s.n0 + i) * A.a.v_row + (long long)kvh * A.a.v_head) : nullptr;
        }
        auto zeros = [](uint32_t* w, int n) { for (int i = 0; i < n; ++i) w[i] = 0u; };
        auto load_k = [&](int j, int c, uint32_t (&w)[B::KB / 4]) { zeros(w, B::KB / 4); if (krow[j]) ld_bytes<B::KB>(krow[j] + (4 * B::KE * c + B::KE * qd) * 2, w); };
        auto load_v = [&](int j, int c, uint32_t (&w)[B::VB / 4]) { zeros(w, B::VB / 4); if (vrow[j]) ld_bytes<B::VB>(vrow[j] + (8 * B::VE * c + B::VE * g) * 2, w); };
        unit<HD, PCPB_BF16, true>(R, load_k, load_v, vrow, one, one, keep, zero);
      }
      if (CODE != PCPB_BF16) {                                  // from a lane's columns of the bf16 form to those of the codes' form
#pragma unroll
        for (int t = 0; t < HD / 16; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) mine[(2 * qd + (k & 1)) * HD + out_col<HD, PCPB_BF16>(t, g, k >> 1)] = R.o[t][k];
        __syncwarp();
#pragma unroll
        for (int t = 0; t < HD / 16; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) R.o[t][k] = mine[(2 * qd + (k & 1)) * HD + out_col<HD, CODE>(t, g, k >> 1)];
        __syncwarp();
      }
    }
    // cached keys [t0 TILE, t1 TILE)
    if (t0 < ct) {
      const int end = min(s.ctx, t1 * TILE), first = t0 * TILE + warp * 16;
      const int nu = first < end ? (end - first + WARPS * 16 - 1) / (WARPS * 16) : 0;      // this warp's units
      struct Entry { int raw, in; };
      auto look = [&](int k) {                                  // lanes l and l + 16 look up position l of unit k
        Entry e{-1, -1};
        const int pos = first + k * (WARPS * 16) + (lane & 15);
        if (k < nu && pos < end) {
          const int lp = pos / A.c.page_tokens;
          e.in = pos - lp * A.c.page_tokens;
          e.raw = __ldg(A.c.block_table + (size_t)b * A.c.max_pages + lp);           // lp < max_pages: ctx is clipped to the table
        }
        return e;
      };
      auto issue = [&](int k, const Entry& e) {
        const int page = clip_page(e.raw, A.c.n_pages);
        if (e.in >= 0 && page < 0) op_note(A.status, PCPB_OPS_BAD_PAGE);
        const long long off = page < 0 ? -1 : page_row(page, A.c.page_stride, kvh, A.c.page_tokens, e.in, HD) * F::ES;
        const uint32_t st = ring_s + (k % G::NST) * G::STAGE;
        const uint32_t valid = __ballot_sync(0xffffffffu, off >= 0) & 0xFFFFu;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const long long o = __shfl_sync(0xffffffffu, off, 8 * j + g);
#pragma unroll
          for (int c = 0; c < F::KC; ++c)
            cp_async<F::KB>(st + ((j * F::KC + c) * 32 + lane) * F::KB, (const uint8_t*)A.c.k + (o < 0 ? 0 : o + (4 * F::KE * c + F::KE * qd) * F::ES), o >= 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const long long o = __shfl_sync(0xffffffffu, off, 8 * (j >> 1) + 2 * qd + (j & 1));
#pragma unroll
          for (int c = 0; c < F::VC; ++c)
            cp_async<F::VB>(st + G::K_BYTES + ((j * F::VC + c) * 32 + lane) * F::VB, (const uint8_t*)A.c.v + (o < 0 ? 0 : o + (8 * F::VE * c + F::VE * g) * F::ES), o >= 0);
        }
        if (CODE != PCPB_BF16)
          cp_async<4>(st + 2 * G::K_BYTES + lane * 4,
                      (lane < 16 ? A.c.k_scale : A.c.v_scale) + (page < 0 ? 0 : page_row(page, A.c.scale_stride, kvh, A.c.page_tokens, e.in, 1)), page >= 0);
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + (k % G::NST) * G::STAGE + 2 * G::K_BYTES + 128) = valid;
      };
      Entry pre[G::NST];
#pragma unroll
      for (int k = 0; k < G::NST; ++k) pre[k] = look(k);
#pragma unroll
      for (int k = 0; k < G::NST - 1; ++k) {
        if (k < nu) issue(k, pre[k]);
        asm volatile("cp.async.commit_group;" ::: "memory");
      }
      Entry next = pre[G::NST - 1];
      load_q<HD, CODE>(A, s, kvh, row0, R);
#pragma unroll 1
      for (int k = 0; k < nu; ++k) {
        if (k + G::NST - 1 < nu) issue(k + G::NST - 1, next);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next = look(k + G::NST);
        asm volatile("cp.async.wait_group %0;" ::"n"(G::NST - 1) : "memory");
        __syncwarp();
        const uint8_t* st = ring + (k % G::NST) * G::STAGE;
        const float* sc = reinterpret_cast<const float*>(st + 2 * G::K_BYTES);
        const uint32_t valid = *reinterpret_cast<const uint32_t*>(sc + 32);
        float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
        uint32_t keep = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          keep |= ((valid >> (g + 8 * i)) & 1u) * (3u << (2 * i));
          if (CODE != PCPB_BF16) { ks[i] = sc[g + 8 * i]; vs[i] = sc[16 + g + 8 * i]; }
        }
        auto load_k = [&](int j, int c, uint32_t (&w)[F::KB / 4]) { ld_bytes<F::KB>(st + ((j * F::KC + c) * 32 + lane) * F::KB, w); };
        auto load_v = [&](int j, int c, uint32_t (&w)[F::VB / 4]) { ld_bytes<F::VB>(st + G::K_BYTES + ((j * F::VC + c) * 32 + lane) * F::VB, w); };
        const uint8_t* const no_rows[4] = {};
        unit<HD, CODE, false>(R, load_k, load_v, no_rows, ks, vs, keep, 0u);
        __syncwarp();                                           // scales and valid positions are read by other lanes than wrote them
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
    }
    // the warps' parts -> the tile's rows
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float l = R.l[j];
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (g == 0) { mml[warp][2 * qd + j][0] = R.m[j]; mml[warp][2 * qd + j][1] = l; }
    }
#pragma unroll
    for (int t = 0; t < HD / 16; ++t)
#pragma unroll
      for (int k = 0; k < 4; ++k) mine[(2 * qd + (k & 1)) * HD + out_col<HD, CODE>(t, g, k >> 1)] = R.o[t][k];
    __syncthreads();
    const bool whole = t0 == 0 && t1 == T;
    const size_t slot = (size_t)blockIdx.x * 2 + (w == w0 ? 0 : 1);
    for (int i = threadIdx.x; i < RW * (HD / 4); i += blockDim.x) {
      const int r = i / (HD / 4), c = i % (HD / 4) * 4;
      if (row0 + r >= rows) continue;
      float m = -INFINITY;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) m = fmaxf(m, mml[k][r][0]);
      const float ref = m == -INFINITY ? 0.f : m;
      float l = 0.f, o[4] = {};
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float f = ex2(mml[k][r][0] - ref);
        const float4 v = *reinterpret_cast<const float4*>(rings + k * G::BYTES + (r * HD + c) * 4);
        l += f * mml[k][r][1];
        o[0] += f * v.x; o[1] += f * v.y; o[2] += f * v.z; o[3] += f * v.w;
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int node = (row0 + r) / A.G, h = kvh * A.G + (row0 + r) % A.G;
        bf16* dst = (bf16*)A.a.out + (long long)(s.n0 + node) * A.a.out_row + (long long)h * A.a.out_head + c;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv));
        if (A.a.lse && c == 0) A.a.lse[(size_t)(s.n0 + node) * A.a.n_head + h] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
      } else {
        *reinterpret_cast<float4*>(A.part_o + (slot * RW + r) * HD + c) = make_float4(o[0], o[1], o[2], o[3]);
        if (c == 0) { A.part_ml[(slot * RW + r) * 2] = m; A.part_ml[(slot * RW + r) * 2 + 1] = l; }
      }
    }
    __syncthreads();
    w = pitch ? w1 : w + (t1 - t0);
  }
}

// Adds up the parts of the items that were split.  grid = (batch, n_kv_head * most row tiles, ROWS / 16): a block joins 16 rows, a thread
// four columns of one or more of them.
template <int HD, int ROWS> __global__ void __launch_bounds__(256) k_tree_join(const __grid_constant__ AttnArgs A, int blocks) {
  const int b = blockIdx.x;
  const Seq s = seq_of(A, b);
  const int rows = s.n * A.G, RT = (rows + ROWS - 1) / ROWS, T = tiles_of(s.ctx) + tiles_of(s.n);
  const int item = blockIdx.y;
  pdl_wait();                                                   // in every block: whatever comes after this kernel comes after the attention too
  if (item >= RT * A.c.n_kv_head) return;
  const int kvh = item / RT, row0 = item % RT * ROWS, r0 = blockIdx.z * 16;
  if (row0 + r0 >= rows) return;
  if (A.plan[A.c.batch + 1]) return;                            // whole items: nothing was split
  const Parts P = parts_of(A.plan[b] + (long long)item * T, T, tile_share(A.plan[A.c.batch], blocks));
  if (P.c0 == P.c1) return;
  for (int i = threadIdx.x; i < 16 * (HD / 4); i += blockDim.x) {
    const int r = r0 + i / (HD / 4), c = i % (HD / 4) * 4;
    if (r >= ROWS || row0 + r >= rows) continue;
    float m = -INFINITY, l = 0.f, o[4] = {};
    for (int k0 = P.c0; k0 <= P.c1; k0 += 4) {                  // four parts in flight, taken in block order
      float2 q[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        q[k] = make_float2(-INFINITY, 0.f);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k0 + k <= P.c1) {
          const size_t at = (size_t)part_slot(P, k0 + k) * ROWS + r;
          q[k] = *reinterpret_cast<const float2*>(A.part_ml + at * 2);
          v[k] = *reinterpret_cast<const float4*>(A.part_o + at * HD + c);
        }
      }
      const float top = fmaxf(fmaxf(fmaxf(q[0].x, q[1].x), fmaxf(q[2].x, q[3].x)), m), ref = top == -INFINITY ? 0.f : top;
      const float f0 = ex2(m - ref);
      m = top;
      l *= f0; o[0] *= f0; o[1] *= f0; o[2] *= f0; o[3] *= f0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = ex2(q[k].x - ref);
        l += f * q[k].y;
        o[0] += f * v[k].x; o[1] += f * v[k].y; o[2] += f * v[k].z; o[3] += f * v[k].w;
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int node = (row0 + r) / A.G, h = kvh * A.G + (row0 + r) % A.G;
    bf16* dst = (bf16*)A.a.out + (long long)(s.n0 + node) * A.a.out_row + (long long)h * A.a.out_head + c;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv));
    if (A.a.lse && c == 0) A.a.lse[(size_t)(s.n0 + node) * A.a.n_head + h] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
  }
}

// ---- the kernel for many rows: tcgen05.mma ---------------------------------------------------------------------------
// An item is up to 256 rows (two tiles of 128) of one kv head.  Two streams of score and output tiles are in flight in tensor memory, so that
// the products of one run while the other's softmax does: with more than 128 rows the streams are the two row tiles, which share
// every tile of keys; with fewer both streams have the same rows and take the tiles of keys in turn, and are joined at the end.
//   loaders (4 warps for keys, 4 for values)   find the rows of a tile's 128 positions in the block table, two tiles ahead, and bring them into
//                       128-byte-swizzled shared memory.  8-bit codes are widened on the way (keys to f16, values to bf16); a thread
//                       holds its pieces of the next tile in registers meanwhile.  The key loaders also describe the tile (scales,
//                       valid positions) in a ring.
//   softmax (2 x 4)     a thread owns a row: scores from tensor memory, running maximum and sum, weights as bf16 over the scores.  The first
//                       warp of each stream also issues its products when the four warps' weights are there: O += P V (P in tensor
//                       memory, V as the MN-major operand), then S = Q K^T of the stream's next tile; it would only wait for them
//                       otherwise, and a warp of its own for it would cost the loaders the registers that hold their codes.
// The reference maximum of a row moves only when a score passes it by 2^8 (weights up to 256 cost nothing: bf16 keeps its relative
// precision), so the output is rescaled in few tiles.
// Loops over a tile's columns are not unrolled further than 32: with everything unrolled the roles' code did not fit the instruction
// caches (a third of the stalls were missing instructions).
// Bound: the softmax warps' issue latency.  64 drafts on 4 sequences of 40960 i8 positions, 32 q / 8 kv heads x 128: 280 us (500 TFLOP/s,
// tensor pipe 23 %; with one group of loaders and a warp of its own for the products 551); 24 drafts on 16 x 2048 in bf16: 43 us.
// Every wait is bounded.  A wait that runs out marks the block as failed and sets PCPB_OPS_STUCK; from there on waits return at once and all
// warps run their loops to the end (the same barriers, valid addresses, wrong numbers), so that nothing hangs.
constexpr int TR = 256;              // rows of an item
constexpr int TC_THREADS = 512;      // 128 registers a thread
constexpr int INFO = 4;              // tile descriptions in flight

template <int HD> struct TcCfg {
  static constexpr int TILE_BYTES = 128 * HD * 2;
  static constexpr int OFF_K = 2 * TILE_BYTES, OFF_V = OFF_K + 2 * TILE_BYTES, OFF_INFO = OFF_V + 2 * TILE_BYTES;
  static constexpr int INFO_BYTES = 2 * 128 * 4 + 16;                     // key scales, value scales, valid positions (a word for 32)
  static constexpr int OFF_ROW = OFF_INFO + INFO * INFO_BYTES;            // [2 loader groups][3][128] byte offsets of rows
  static constexpr int OFF_ML = OFF_ROW + 6 * 128 * 8;                    // [2][128][2] maxima and sums of the streams
  static constexpr int OFF_PAR = OFF_ML + 2 * 128 * 2 * 4;                // parents
  static constexpr int OFF_ANC = OFF_PAR + MAX_NODES * 2;                 // [MAX_NODES / 32][256] ancestors-or-self of the rows' nodes
  static constexpr int OFF_QF = OFF_ANC + MAX_NODES / 32 * 256 * 4;       // [256] factors of the rows of q
  static constexpr int OFF_BAR = OFF_QF + 256 * 4;
  static constexpr int OFF_PLAN = OFF_BAR + 256;
  static constexpr int BYTES = OFF_PLAN + (MAX_BATCH + 2) * 8 + 1024;
  static_assert(BYTES <= 232448, "shared memory");
};

__device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n) : "memory");
}
__device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, int* fail) {
  if (!mbar_try(bar, parity) && !*(volatile int*)fail) mbar_wait(bar, parity, fail, 1);
  __syncwarp();                                                 // what follows is for whole warps
}
__device__ __forceinline__ void cp_async16z(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
// Byte offset of 16-byte piece c of row r in a 128-row tile of 64-column halves, 128-byte swizzle
__device__ __forceinline__ uint32_t sw_off(int r, int c) { return (uint32_t)((c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4)); }
__device__ __forceinline__ void st_shared16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// The blocks' segments: a run of tiles [t0, t1) of one item
struct Seg { int b, kvh, row0, rows, t0, t1, ct, T; Seq s; long long next; };       // next: where the block goes on
__device__ __forceinline__ Seg seg_at(const AttnArgs& A, const long long* plan, long long w, long long w1) {
  Seg g;
  g.b = seq_at(plan, A.c.batch, w);
  g.s = seq_of(A, g.b);
  g.ct = tiles_of(g.s.ctx); g.T = g.ct + tiles_of(g.s.n);
  const int all = g.s.n * A.G, RT = (all + TR - 1) / TR;
  const long long at = w - plan[g.b];
  const int pitch = (int)plan[A.c.batch + 1], P = pitch ? pitch : g.T;
  const long long item = at < 0x7fffffffll ? (long long)((unsigned)at / (unsigned)P) : at / P;
  g.t0 = (int)(at - item * P);
  g.t1 = (int)min((long long)g.T, g.t0 + (w1 - w));
  g.next = pitch ? w1 : w + (g.t1 - g.t0);
  g.kvh = (int)item / RT; g.row0 = ((int)item - g.kvh * RT) * TR;          // items of a sequence: kv heads x row tiles, an int
  g.rows = min(TR, all - g.row0);
  return g;
}

template <int HD, int CODE> __global__ void __launch_bounds__(TC_THREADS, 1) k_tree_tc(const __grid_constant__ AttnArgs A) {
  using Cfg = TcCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t sQ = base, sK = base + Cfg::OFF_K, sV = base + Cfg::OFF_V, sBar = base + Cfg::OFF_BAR;
  long long* plan = reinterpret_cast<long long*>(gen + Cfg::OFF_PLAN);
  __shared__ int fail;
  __shared__ uint32_t tmem_slot, odd[4][MAX_NODES / 32];        // odd: nodes of a segment whose values hold an infinity or a NaN (the loaders are at most two segments ahead)
  auto kfull = [&](int i) { return sBar + 8u * i; };
  auto kempty = [&](int i) { return sBar + 16u + 8u * i; };
  auto vfull = [&](int i) { return sBar + 32u + 8u * i; };
  auto vempty = [&](int i) { return sBar + 48u + 8u * i; };
  auto sfull = [&](int x) { return sBar + 64u + 8u * x; };
  auto pfull = [&](int x) { return sBar + 80u + 8u * x; };
  auto pvdone = [&](int x) { return sBar + 96u + 8u * x; };
  auto ifull = [&](int i) { return sBar + 128u + 8u * i; };
  auto iempty = [&](int i) { return sBar + 160u + 8u * i; };
  const uint32_t qfull = sBar + 192u, odone = sBar + 200u;

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    fail = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(kfull(i), 128); mbar_init(kempty(i), 2); mbar_init(vfull(i), 128); mbar_init(vempty(i), 2);
      mbar_init(sfull(i), 1); mbar_init(pfull(i), 4); mbar_init(pvdone(i), 1);
    }
    for (int i = 0; i < INFO; ++i) { mbar_init(ifull(i), 128); mbar_init(iempty(i), 8); }
    mbar_init(qfull, 256); mbar_init(odone, 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  make_plan<TR>(A, plan, SLACK_MANY);                                       // (its barriers also publish the setup above)
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *(volatile uint32_t*)&tmem_slot;
  const long long total = plan[A.c.batch], per = share_of(plan, A.c.batch, gridDim.x);
  if (blockIdx.x == 0) for (int b = threadIdx.x; b < A.c.batch + 2; b += blockDim.x) A.plan[b] = plan[b];
  const long long w0 = per * blockIdx.x, w1 = min(total, w0 + per);
  auto s_col = [&](int x) { return tmem + 128u * x; };
  auto o_col = [&](int x) { return tmem + 256u + 128u * x; };

  if (warp >= 8) {
    // =========================== loaders ===========================
    const bool vals = warp >= 12;                               // this group's operand
    const int t = threadIdx.x & 127, bar = vals ? 3 : 2;
    constexpr int ES = CODE == PCPB_BF16 ? 2 : 1, PIECES = HD * ES / 16, NP = PIECES;          // 16-byte pieces of a row = pieces of a thread per tile
    constexpr int PB = HD / 8;                                  // pieces of a node's row (bf16)
    long long* rowoff = reinterpret_cast<long long*>(gen + Cfg::OFF_ROW) + (vals ? 384 : 0);
    const uint8_t* const pages = (const uint8_t*)(vals ? A.c.v : A.c.k);
    const bf16* const nodes = (const bf16*)(vals ? A.a.v : A.a.k);
    const long long node_row = vals ? A.a.v_row : A.a.k_row, node_head = vals ? A.a.v_head : A.a.k_head;
    const uint32_t full0 = vals ? vfull(0) : kfull(0), empty0 = vals ? vempty(0) : kempty(0), dst0 = vals ? sV : sK;
    int gi = 0, seg = 0;                                        // tiles so far (ring positions), segments
    uint32_t pending = 0;                                       // cp.async path: barrier of the tile that is in flight
    auto flush = [&]() {
      if (pending) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async_smem();
        mbar_arrive(pending);
        pending = 0;
      }
    };
    auto wait_empty = [&](uint32_t bar, uint32_t parity) {
      if (!mbar_try(bar, parity)) {
        flush();                                                // what the consumers may need to free the place
        if (!*(volatile int*)&fail) mbar_wait(bar, parity, &fail, 1);
      }
      __syncwarp();
    };
    for (long long w = w0; w < w1; ++seg) {
      const Seg g = seg_at(A, plan, w, w1);
      const int nt = g.t1 - g.t0;
      // Position t of a cached tile, in three steps a tile apart, so that no load is waited for: the block-table entry, then the row's
      // place and its scales, then both are used.
      struct Entry { int raw, in; };
      struct Found { long long off; float ks, vs; };
      auto look = [&](int tile) {
        const int pos = tile * TILE + t;
        Entry e{-1, -1};
        if (tile < min(g.ct, g.t1) && pos < g.s.ctx) {
          const int lp = pos / A.c.page_tokens;
          e.in = pos - lp * A.c.page_tokens;
          e.raw = __ldg(A.c.block_table + (size_t)g.b * A.c.max_pages + lp);       // lp < max_pages: ctx is clipped to the table
        }
        return e;
      };
      auto find = [&](const Entry& e) {
        Found f{-1, 1.f, 1.f};
        const int page = clip_page(e.raw, A.c.n_pages);
        if (e.in >= 0 && page < 0) op_note(A.status, PCPB_OPS_BAD_PAGE);
        if (page >= 0) {
          f.off = page_row(page, A.c.page_stride, g.kvh, A.c.page_tokens, e.in, HD) * ES;
          if (CODE != PCPB_BF16 && !vals) {
            const long long so = page_row(page, A.c.scale_stride, g.kvh, A.c.page_tokens, e.in, 1);
            f.ks = __ldg(A.c.k_scale + so); f.vs = __ldg(A.c.v_scale + so);
          }
        }
        return f;
      };
      auto piece = [&](int k, int slot) {                       // piece k of this thread of a cached tile
        const int idx = t + 128 * k, row = idx / PIECES, c = idx % PIECES;
        const long long o = rowoff[slot * 128 + row];
        return o < 0 ? make_uint4(0u, 0u, 0u, 0u) : __ldg(reinterpret_cast<const uint4*>(pages + o + c * 16));
      };
      uint4 cur[CODE == PCPB_BF16 ? 1 : NP];
      Entry e1 = look(g.t0), e2 = look(g.t0 + 1);
      Found f0 = find(e1), f1 = find(e2);                       // of this tile and the next
      e2 = look(g.t0 + 2);
      // Three places of row offsets: at tile i a thread writes those of tile i + 1, while others may still be reading tile i - 1's (they are
      // only known to have passed tile i - 1's barrier).
      int slot = gi % 3;
      rowoff[slot * 128 + t] = f0.off;
      bar_sync(bar, 128);
      if (CODE != PCPB_BF16 && g.t0 < g.ct) {
#pragma unroll
        for (int k = 0; k < NP; ++k) cur[k] = piece(k, slot);
      }
#pragma unroll 1
      for (int i = 0; i < nt; ++i, ++gi) {
        const int tile = g.t0 + i, st = gi & 1, in = gi % INFO;
        const bool cached = tile < g.ct;
        float* info = nullptr;
        if (!vals) {                                            // description of the tile
          wait_empty(iempty(in), ((gi / INFO) & 1) ^ 1);
          info = reinterpret_cast<float*>(gen + Cfg::OFF_INFO + in * Cfg::INFO_BYTES);
          info[128 + t] = f0.vs;
          const uint32_t valid = __ballot_sync(0xffffffffu, f0.off >= 0);
          if (lane == 0) reinterpret_cast<uint32_t*>(info)[256 + (t >> 5)] = valid;
          if (cached || CODE == PCPB_BF16) {                    // (the nodes' key factors are known when their rows are there)
            const float factor = f0.ks * (fabsf(A.a.scale) * LOG2E);
            info[t] = factor < 1.17549435e-38f ? 1.17549435e-38f : factor;           // (a NaN stays)
            mbar_arrive(ifull(in));
          }
        }
        // the next tile's rows
        const int slot1 = slot == 2 ? 0 : slot + 1;
        if (i + 1 < nt) rowoff[slot1 * 128 + t] = f1.off;
        bar_sync(bar, 128);
        const uint32_t dst = dst0 + st * Cfg::TILE_BYTES, full = full0 + 8u * st;
        wait_empty(empty0 + 8u * st, ((gi >> 1) & 1) ^ 1);
        if (CODE == PCPB_BF16 && cached) {
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            const int idx = t + 128 * k, row = idx / PIECES, c = idx % PIECES;
            const long long o = rowoff[slot * 128 + row];
            cp_async16z(dst + sw_off(row, c), pages + (o < 0 ? 0 : o + c * 16), o >= 0);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          if (pending) {
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            fence_proxy_async_smem();
            mbar_arrive(pending);
          }
          pending = full;
        } else if (cached) {
          const bool more = i + 1 < nt && tile + 1 < g.ct;
          auto fill = [&](auto is_values) {
#pragma unroll
          for (int k = 0; k < NP; ++k) {
            const int idx = t + 128 * k, row = idx / PIECES, c = idx % PIECES;
            uint32_t p[8];
            constexpr int CC = CODE == PCPB_BF16 ? PCPB_I8 : CODE;
            const uint4 r = cur[CODE == PCPB_BF16 ? 0 : k];
            if constexpr (decltype(is_values)::value) { widen4<CC>(r.x, p[0], p[1]); widen4<CC>(r.y, p[2], p[3]); widen4<CC>(r.z, p[4], p[5]); widen4<CC>(r.w, p[6], p[7]); }
            else { widen4_f16<CC>(r.x, p[0], p[1]); widen4_f16<CC>(r.y, p[2], p[3]); widen4_f16<CC>(r.z, p[4], p[5]); widen4_f16<CC>(r.w, p[6], p[7]); }
            const int flip = (c >> 2) & 1;                      // pieces of the second half go the other way round: other banks than the first half's
            st_shared16(dst + sw_off(row, 2 * c + flip), p[flip ? 4 : 0], p[flip ? 5 : 1], p[flip ? 6 : 2], p[flip ? 7 : 3]);
            st_shared16(dst + sw_off(row, 2 * c + 1 - flip), p[flip ? 0 : 4], p[flip ? 1 : 5], p[flip ? 2 : 6], p[flip ? 3 : 7]);
          }
          };
          if (vals) fill(std::true_type()); else fill(std::false_type());
          fence_proxy_async_smem();
          mbar_arrive(full);
          // All of the next tile's loads together, after the last use of this one's: loads that are issued between uses of earlier ones share
          // their scoreboards, and every use then waits for the newest load (1000 cycles a piece).
          if (more) {
#pragma unroll
            for (int k = 0; k < NP; ++k) cur[CODE == PCPB_BF16 ? 0 : k] = piece(k, slot1);
          }
        } else {
          // rows of the nodes (bf16); values that are not numbers are left out and their nodes marked
          const int n0 = (tile - g.ct) * TILE;
          flush();
          if (vals && tile == max(g.ct, g.t0)) {
            if (t < MAX_NODES / 32) odd[seg & 3][t] = 0u;
            bar_sync(bar, 128);
          }
#pragma unroll 1
          for (int base = 0; base < PB; base += 8) {            // eight pieces in flight
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int idx = t + 128 * (base + k), node = n0 + idx / PB;
              v[k] = make_uint4(0u, 0u, 0u, 0u);
              if (node < g.s.n) v[k] = *reinterpret_cast<const uint4*>(nodes + (long long)(g.s.n0 + node) * node_row + (long long)g.kvh * node_head + idx % PB * 8);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int idx = t + 128 * (base + k), row = idx / PB, node = n0 + row;
              uint32_t q[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
              if (vals) {
                bool bad = false;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  if ((q[j] & 0x7F80u) == 0x7F80u) { q[j] &= 0xFFFF0000u; bad = true; }
                  if ((q[j] & 0x7F800000u) == 0x7F800000u) { q[j] &= 0x0000FFFFu; bad = true; }
                }
                if (bad) atomicOr(&odd[seg & 3][(node >> 5) & 7], 1u << (node & 31));
              } else if (CODE != PCPB_BF16) {                   // keys in f16, scaled by a power of two per row; PB lanes hold a row
                uint32_t top = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) top = top_abs2(top, q[j]);
#pragma unroll
                for (int o = PB / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                const int e = exp15(top);
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = bf16x2_to_f16x2(q[j], pow2(e));
                if (idx % PB == 0) info[row] = fmaxf(pow2(-e) * (fabsf(A.a.scale) * LOG2E), 1.17549435e-38f);
              }
              st_shared16(dst + sw_off(row, idx % PB), q[0], q[1], q[2], q[3]);
            }
          }
          if (!vals && CODE != PCPB_BF16) mbar_arrive(ifull(in));
          fence_proxy_async_smem();
          mbar_arrive(full);
        }
        f0 = f1; f1 = find(e2); e2 = look(tile + 3);
        slot = slot1;
      }
      w = g.next;
    }
    flush();
  } else {
    // =========================== softmax ===========================
    const int x = warp >> 2, q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t lane_off = (uint32_t)(q4 * 32) << 16;
    // a negative scale changes the sign of q instead; a positive factor at least, so that a masked score stays -inf
    const float zscale = fmaxf(fabsf(A.a.scale) * LOG2E, 1.17549435e-38f);
    const uint32_t qsign = A.a.scale < 0.f ? 0x80008000u : 0u;
    constexpr uint32_t KT = CODE == PCPB_BF16 ? 1u : 0u;        // type of both operands of the scores: bf16, or f16 for codes
    constexpr uint32_t ID_S = (1u << 4) | (KT << 7) | (KT << 10) | ((uint32_t)(128 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    constexpr uint32_t ID_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    const bool issuer = q4 == 0;
    int gi = 0, seg = 0, sn = 0;                                // tiles, segments; score tiles of this stream so far
    int16_t* par = reinterpret_cast<int16_t*>(gen + Cfg::OFF_PAR);
    float* ml = reinterpret_cast<float*>(gen + Cfg::OFF_ML);
    float* qfac = reinterpret_cast<float*>(gen + Cfg::OFF_QF);
    uint32_t* anc = reinterpret_cast<uint32_t*>(gen + Cfg::OFF_ANC) + threadIdx.x;       // this thread's row: word k at anc[256 k]
    for (long long w = w0; w < w1; ++seg) {
      const Seg g = seg_at(A, plan, w, w1);
      const int nt = g.t1 - g.t0;
      const bool pair = g.rows > 128;
      const int tr = pair ? x * 128 + r : r;                    // row of the item
      const bool live = tr < g.rows, warp_live = (pair ? x * 128 : 0) + q4 * 32 < g.rows;
      const int node = (g.row0 + tr) / A.G, head = g.kvh * A.G + (g.row0 + tr) % A.G;
      const bool has_tree = g.t1 > g.ct;
      if (has_tree && threadIdx.x < g.s.n) {                    // at most 256 nodes, as many threads
        int bad = 0;
        par[threadIdx.x] = (int16_t)clip_parent(A.a.parent ? A.a.parent[g.s.n0 + threadIdx.x] : (int)threadIdx.x - 1, threadIdx.x, &bad);
        if (bad) op_note(A.status, PCPB_OPS_BAD_TREE);
      }
      {
        // rows of q: HD / 8 lanes a row, eight rows of a thread in flight; rows of both tiles, or all 256 threads on the one tile
        constexpr int PQ = HD / 8, RP = 256 / PQ;               // rows of a pass
        const int c = threadIdx.x % PQ, passes = (pair ? 256 : 128) / RP;
#pragma unroll 1
        for (int p0 = 0; p0 < passes; p0 += 4) {
          uint4 v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int qr = (p0 + k) * RP + (int)threadIdx.x / PQ, qn = (g.row0 + qr) / A.G, qh = g.kvh * A.G + (g.row0 + qr) - qn * A.G;
            v[k] = qr < g.rows ? *reinterpret_cast<const uint4*>((const bf16*)A.a.q + (long long)(g.s.n0 + qn) * A.a.q_row + (long long)qh * A.a.q_head + c * 8) : make_uint4(0u, 0u, 0u, 0u);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int qr = (p0 + k) * RP + (int)threadIdx.x / PQ;
            uint4 y = make_uint4(v[k].x ^ qsign, v[k].y ^ qsign, v[k].z ^ qsign, v[k].w ^ qsign);
            if (CODE != PCPB_BF16) {                            // q in f16, scaled by a power of two per row
              uint32_t top = top_abs2(top_abs2(top_abs2(top_abs2(0u, y.x), y.y), y.z), y.w);
#pragma unroll
              for (int o = PQ / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
              const int e = exp15(top);
              const float up = pow2(e);
              y = make_uint4(bf16x2_to_f16x2(y.x, up), bf16x2_to_f16x2(y.y, up), bf16x2_to_f16x2(y.z, up), bf16x2_to_f16x2(y.w, up));
              if (c == 0) qfac[qr] = pow2(-e);
            }
            st_shared16(sQ + (qr >> 7) * Cfg::TILE_BYTES + sw_off(qr & 127, c), y.x, y.y, y.z, y.w);
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(qfull);
      }
      // products of tile i of the segment; a ring place is free when both streams' products (one stream: its own, twice) are done
      auto issue_qk = [&](int i) {
        const int at = gi + i, st = at & 1;
        wait(kfull(st), (at >> 1) & 1, &fail);
        tc_fence_after();
        const uint32_t a = sQ + (pair ? x * Cfg::TILE_BYTES : 0), b = sK + st * Cfg::TILE_BYTES;
#pragma unroll
        for (int k = 0; k < HD / 16; ++k) {
          const uint32_t o = (uint32_t)(k >> 2) * 16384u + (uint32_t)(k & 3) * 32u;
          mma_bf16_elect(s_col(x), make_desc(a + o, 16, 1024), make_desc(b + o, 16, 1024), ID_S, k > 0);
        }
        mma_commit_elect(sfull(x));
        mma_commit_elect(kempty(st));
        if (!pair) mma_commit_elect(kempty(st));
      };
      auto issue_pv = [&](int i, bool first) {
        const int at = gi + i, st = at & 1;
        wait(vfull(st), (at >> 1) & 1, &fail);
        tc_fence_after();
        const uint32_t b = sV + st * Cfg::TILE_BYTES;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          mma_bf16_ts_elect(o_col(x), s_col(x) + 8u * k, make_desc(b + k * 2048u, 16384, 1024), ID_O, !first || k > 0);
        mma_commit_elect(pvdone(x));
        mma_commit_elect(vempty(st));
        if (!pair) mma_commit_elect(vempty(st));
      };
      const int step = pair ? 1 : 2;
      if (issuer) {
        wait(qfull, seg & 1, &fail);
        if ((pair ? 0 : x) < nt) issue_qk(pair ? 0 : x);
      }
      if (has_tree) {
        bar_sync(1, 256);
#pragma unroll 1
        for (int k = 0; k < MAX_NODES / 32; ++k) anc[256 * k] = 0u;
#pragma unroll 1
        for (int i = live ? node : -1; i >= 0; i = par[i]) anc[256 * (i >> 5)] |= 1u << (i & 31);
      }
      // factor of the row's scores (codes: the keys' factors hold the scale); the first score tile comes after every thread's part of q
      float rowf = zscale;
      float mref = -INFINITY;
      f32x2 l2 = pk2(0.f, 0.f);
      int done = 0;                                             // tiles of this stream in this segment
      for (int i = pair ? 0 : x; i < nt; i += step, ++done, ++sn) {
        const int in = (gi + i) % INFO;
        const float* info = reinterpret_cast<const float*>(gen + Cfg::OFF_INFO + in * Cfg::INFO_BYTES);
        const int tile = g.t0 + i;
        const bool tree = tile >= g.ct;
        wait(ifull(in), ((gi + i) / INFO) & 1, &fail);
        const uint4 valid = *reinterpret_cast<const uint4*>(info + 256);
        wait(sfull(x), sn & 1, &fail);
        tc_fence_after();
        if (CODE != PCPB_BF16) rowf = qfac[tr];
        if (warp_live) {
          // The reference maximum moves (rarely): outputs, sums and the tile's weights so far (columns below 32 c) are scaled down.
          auto raise = [&](float top, int c) {
            const bool up = top > mref + 8.f || (mref == -INFINITY && top > -INFINITY);
            const float to = up ? top : mref, corr = up && mref > -INFINITY ? ex2(mref - to) : 1.f;
            if (done > 0) {
              wait(pvdone(x), (sn - 1) & 1, &fail);
              tc_fence_after();
#pragma unroll 1
              for (int k = 0; k < HD; k += 16) {
                uint32_t u[16];
                tmem_ld16(o_col(x) + lane_off + k, u);
#pragma unroll
                for (int j = 0; j < 16; ++j) u[j] = __float_as_uint(__uint_as_float(u[j]) * corr);
                tmem_st16(o_col(x) + lane_off + k, u);
              }
            }
#pragma unroll 1
            for (int k = 0; k < c; ++k) {
              uint32_t u[16];
              tmem_ld16(s_col(x) + lane_off + 16u * k, u);
#pragma unroll
              for (int j = 0; j < 16; ++j) u[j] = pack2(bf_lo(u[j]) * corr, bf_hi(u[j]) * corr);
              tmem_st16(s_col(x) + lane_off + 16u * k, u);
            }
            tmem_st_wait();
            l2 = mul2(l2, pk2(corr, corr));
            mref = to;
          };
          // 32 columns at a time.  The weights are formed with the
          // reference maximum as it stands, and once more in the rare case that it has to move.
          auto chunk = [&](uint32_t (&v)[32], int c, int own) {
            float z[32], top;
            uint32_t p[16];
            f32x2 sum;
            const ulonglong2* k4 = reinterpret_cast<const ulonglong2*>(info + 32 * c);
            const ulonglong2* v4 = reinterpret_cast<const ulonglong2*>(info + 128 + 32 * c);
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
              if (CODE != PCPB_BF16) {
                const ulonglong2 f = k4[j / 4];
                un2(mul2(pk2(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), f.x), z[j], z[j + 1]);
                un2(mul2(pk2(__uint_as_float(v[j + 2]), __uint_as_float(v[j + 3])), f.y), z[j + 2], z[j + 3]);
              } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) z[j + k] = __uint_as_float(v[j + k]);
              }
            }
            for (;;) {
              const float ref = mref == -INFINITY ? 0.f : mref;
              const f32x2 nref = pk2(-ref, -ref), zs = pk2(rowf, rowf);
              f32x2 s0 = pk2(0.f, 0.f), s1 = s0;
              float m0 = z[0], m1 = z[1];
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                f32x2 d0 = pk2(z[j], z[j + 1]), d1 = pk2(z[j + 2], z[j + 3]);
                d0 = fma2(d0, zs, nref);
                d1 = fma2(d1, zs, nref);
                float e0, e1, e2, e3;
                un2(d0, e0, e1); un2(d1, e2, e3);
                m0 = max3(m0, z[j], z[j + 1]); m1 = max3(m1, z[j + 2], z[j + 3]);
                e0 = ex2(e0); e1 = ex2(e1); e2 = ex2(e2); e3 = ex2(e3);
                d0 = pk2(e0, e1); d1 = pk2(e2, e3);
                s0 = add2(s0, d0); s1 = add2(s1, d1);
                if (CODE != PCPB_BF16) {
                  const ulonglong2 y = v4[j / 4];
                  un2(mul2(d0, y.x), e0, e1); un2(mul2(d1, y.y), e2, e3);
                }
                p[j / 2] = pack2(e0, e1); p[j / 2 + 1] = pack2(e2, e3);
              }
              top = fmaxf(m0, m1) * rowf;
              sum = add2(s0, s1);
              if (!__any_sync(0xffffffffu, top > mref + 8.f || (mref == -INFINITY && top > -INFINITY))) break;
              raise(top, c);
            }
            l2 = add2(l2, sum);
            if (own >= 0) {                                     // counted above, but its value is a zero
#pragma unroll
              for (int j = 0; j < 16; ++j) p[j] &= own == 2 * j ? 0xFFFF0000u : own == 2 * j + 1 ? 0x0000FFFFu : 0xFFFFFFFFu;
            }
            tmem_st16(s_col(x) + lane_off + 16u * c, p);
          };
          const int own = tree && A.a.null_self ? node - (tile - g.ct) * TILE : -1;       // a column that counts as a zero key and value
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            uint32_t v[32];
            tmem_ld32(s_col(x) + lane_off + 32u * c, v);
            const uint32_t word = tree ? anc[256 * ((tile - g.ct) * (TILE / 32) + c)] : c == 0 ? valid.x : c == 1 ? valid.y : c == 2 ? valid.z : valid.w;
            const int mine = own >= 32 * c && own < 32 * c + 32 ? own - 32 * c : -1;
            if (!__all_sync(0xffffffffu, word == 0xffffffffu && mine < 0)) {
#pragma unroll
              for (int j = 0; j < 32; ++j) v[j] = j == mine ? 0u : (word >> j) & 1u ? v[j] : 0xFF800000u;
            }
            chunk(v, c, mine);
          }
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(pfull(x));
          mbar_arrive_n(iempty(in), pair ? 1u : 2u);
        }
        if (issuer) {
          wait(pfull(x), sn & 1, &fail);
          tc_fence_after();
          issue_pv(i, done == 0);
          if (i + step < nt) issue_qk(i + step);
        }
      }
      if (issuer) mma_commit_elect(odone);
      float l, lo;
      un2(l2, l, lo);
      l += lo;
      // the segment's end: outputs of both streams are complete
      wait(odone, seg & 1, &fail);
      tc_fence_after();
      if (!pair) {
        ml[(x * 128 + r) * 2] = mref; ml[(x * 128 + r) * 2 + 1] = l;
        bar_sync(1, 256);
      }
      if (warp_live) {
        float f0 = 1.f, f1 = 0.f;
        __syncwarp();
        const bool two = !pair && nt > 1;                       // the second stream had tiles
        if (!pair) {
          const float m0 = ml[r * 2], l0 = ml[r * 2 + 1], m1 = two ? ml[(128 + r) * 2] : -INFINITY, l1 = two ? ml[(128 + r) * 2 + 1] : 0.f;
          mref = fmaxf(m0, m1);
          const float ref = mref == -INFINITY ? 0.f : mref;
          f0 = ex2(m0 - ref); f1 = ex2(m1 - ref);
          l = f0 * l0 + f1 * l1;
        }
        const bool whole = g.t0 == 0 && g.t1 == g.T;
        const float inv = whole ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
        const size_t slot = (size_t)blockIdx.x * 2 + (w == w0 ? 0 : 1);
        bf16* dst = (bf16*)A.a.out + (long long)(g.s.n0 + node) * A.a.out_row + (long long)head * A.a.out_head;
        float* part = A.part_o + (slot * TR + tr) * HD;
        bool strange = false;
        if (has_tree) {
#pragma unroll 1
          for (int k = 0; k < MAX_NODES / 32; ++k) strange |= (anc[256 * k] & odd[seg & 3][k]) != 0u;
        }
        // columns: with two row tiles all of the row's; else the warps of the two groups take half of them each
        const int c0 = pair ? 0 : x * (HD / 32), c1 = pair ? HD / 16 : c0 + HD / 32;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
          uint32_t v[16], u[16];
          __syncwarp();
          tmem_ld16_issue(o_col(pair ? x : 0) + lane_off + 16u * c, v);
          if (two) tmem_ld16_issue(o_col(1) + lane_off + 16u * c, u);
          tmem_ld_wait16(v);
          if (two) tmem_ld_wait16(u);
          float o[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            o[j] = __uint_as_float(v[j]) * f0;
            if (two) o[j] = fmaf(__uint_as_float(u[j]), f1, o[j]);
          }
          if (strange)                                          // infinities and NaN of the values this row does attend
            for (int i = max(0, g.t0 - g.ct) * TILE; i < min(g.s.n, (g.t1 - g.ct) * TILE); ++i) {
              if (!(((anc[256 * (i >> 5)] & odd[seg & 3][i >> 5]) >> (i & 31)) & 1u) || (A.a.null_self && i == node)) continue;
              const bf16* vr = (const bf16*)A.a.v + (long long)(g.s.n0 + i) * A.a.v_row + (long long)g.kvh * A.a.v_head + 16 * c;
#pragma unroll
              for (int j = 0; j < 16; ++j) { const float y = to_f(vr[j]); if (!isfinite(y)) o[j] += y; }
            }
          if (live && whole) {
            uint32_t p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = pack2(o[2 * j] * inv, o[2 * j + 1] * inv);
            *reinterpret_cast<uint4*>(dst + 16 * c) = make_uint4(p[0], p[1], p[2], p[3]);
            *reinterpret_cast<uint4*>(dst + 16 * c + 8) = make_uint4(p[4], p[5], p[6], p[7]);
          } else if (live) {
#pragma unroll
            for (int j = 0; j < 16; j += 4) *reinterpret_cast<float4*>(part + 16 * c + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
        if (live && (pair || x == 0)) {
          if (whole) { if (A.a.lse) A.a.lse[(size_t)(g.s.n0 + node) * A.a.n_head + head] = l == 0.f ? -INFINITY : mref * LN2 + logf(l); }
          else { A.part_ml[(slot * TR + tr) * 2] = mref; A.part_ml[(slot * TR + tr) * 2 + 1] = l; }
        }
      }
      tc_fence_before();
      __syncwarp();
      bar_sync(1, 256);                                         // the outputs, ml, par and q are used again
      tc_fence_after();
      gi += nt;
      w = g.next;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0 && fail) op_note(A.status, PCPB_OPS_STUCK);
  if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// ---- host -----------------------------------------------------------------------------------------------------------
// The attribute of a kernel on the current device, set once.
template <typename K> cudaError_t allow_smem(K kern, bool (&done)[64], size_t bytes) {
  int dev = -1;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 0 && dev < 64 && done[dev]) return cudaSuccess;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}
struct Layout { size_t plan, ml, o, bytes; };
Layout layout(const pcpb_kv_cache& c, int blocks, int rows_tile) {
  Layout L;
  auto up = [](size_t x) { return (x + 255) / 256 * 256; };
  L.plan = 0;
  L.ml = up((size_t)(c.batch + 2) * 8);
  L.o = L.ml + up((size_t)blocks * 2 * rows_tile * 2 * 4);
  L.bytes = L.o + up((size_t)blocks * 2 * rows_tile * c.head_dim * 4);
  return L;
}
int check_heads(const pcpb_kv_cache& c, int n_head, int max_nodes, char* err, size_t cap) {
  if (n_head < 1 || n_head % c.n_kv_head) return op_fail(err, cap, PCPB_E_INVALID, "n_head must be a multiple of n_kv_head");
  if (max_nodes < 1) return op_fail(err, cap, PCPB_E_INVALID, "max_nodes must be positive");
  if (max_nodes > MAX_NODES) return op_fail(err, cap, PCPB_E_TOO_LARGE, "at most %d nodes a sequence", MAX_NODES);
  if (c.batch > MAX_BATCH) return op_fail(err, cap, PCPB_E_TOO_LARGE, "at most %d sequences a call", MAX_BATCH);
  const long long items = (long long)c.n_kv_head * ((max_nodes * (long long)(n_head / c.n_kv_head) + RW - 1) / RW);
  if (items > 65535) return op_fail(err, cap, PCPB_E_TOO_LARGE, "too many query heads");
  return PCPB_OK;
}

template <int HD, int ROWS> cudaError_t launch_join(cudaStream_t st, const AttnArgs& A, int blocks) {
  const int rows = A.a.max_nodes * A.G, items = A.c.n_kv_head * ((rows + ROWS - 1) / ROWS);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(A.c.batch, items, (min(rows, ROWS) + 15) / 16); cfg.blockDim = dim3(256); cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_tree_join<HD, ROWS>, A, blocks);
}
template <int HD, int CODE> cudaError_t launch_rows(cudaStream_t st, const AttnArgs& A, int blocks) {
  const size_t smem = ((size_t)(A.c.batch + 2) * 8 + 15) / 16 * 16 + (size_t)Frag<HD, CODE>::WARPS * Ring<HD, CODE>::BYTES;
  static bool done[64] = {};
  const size_t most = (MAX_BATCH + 2) * 8 + 16 + (size_t)Frag<HD, CODE>::WARPS * Ring<HD, CODE>::BYTES;
  cudaError_t e = allow_smem(k_tree_rows<HD, CODE>, done, most);
  if (e != cudaSuccess) return e;
  k_tree_rows<HD, CODE><<<blocks, Frag<HD, CODE>::WARPS * 32, smem, st>>>(A);
  e = cudaGetLastError();
  return e == cudaSuccess ? launch_join<HD, RW>(st, A, blocks) : e;
}
template <int HD, int CODE> cudaError_t launch_tc(cudaStream_t st, const AttnArgs& A, int blocks) {
  static bool done[64] = {};
  cudaError_t e = allow_smem(k_tree_tc<HD, CODE>, done, TcCfg<HD>::BYTES);
  if (e != cudaSuccess) return e;
  k_tree_tc<HD, CODE><<<blocks, TC_THREADS, TcCfg<HD>::BYTES, st>>>(A);
  e = cudaGetLastError();
  return e == cudaSuccess ? launch_join<HD, TR>(st, A, blocks) : e;
}
// Rows of a kv head from which on the tensor-core kernel takes over.  Its time hardly depends on the rows (up to 128), the other one's grows
// with every 8.  16 sequences of 4096, 8 kv heads x 128, this kernel against the other: bf16 8 rows 63 / 58 us, 12 rows 64 / 99; e4m3 16 rows
// 97 / 81, 24 rows 98 / 99, 32 rows 99 / 135.
constexpr int TC_FROM_BF16 = 9, TC_FROM_CODES = 25;
bool use_tc(const pcpb_kv_cache& c, int G, int max_nodes) { return c.head_dim != 32 && max_nodes * G >= (c.dtype == PCPB_BF16 ? TC_FROM_BF16 : TC_FROM_CODES); }
template <int HD, int CODE> cudaError_t launch_any(cudaStream_t st, const AttnArgs& A, int blocks) {
  if constexpr (HD != 32)
    if (use_tc(A.c, A.G, A.a.max_nodes)) return launch_tc<HD, CODE>(st, A, blocks);
  return launch_rows<HD, CODE>(st, A, blocks);
}
template <int HD> cudaError_t launch_code(cudaStream_t st, const AttnArgs& A, int blocks) {
  if (A.c.dtype == PCPB_BF16) return launch_any<HD, PCPB_BF16>(st, A, blocks);
  if (A.c.dtype == PCPB_I8) return launch_any<HD, PCPB_I8>(st, A, blocks);
  return launch_any<HD, PCPB_E4M3>(st, A, blocks);
}

}  // namespace
}  // namespace pcpb

using namespace pcpb;

extern "C" size_t pcpb_op_tree_attention_workspace(int device, const pcpb_kv_cache* cache, int n_head, int max_nodes, char* err, size_t cap) {
  if (err && cap) err[0] = 0;
  pcpb_kv_cache c;
  if (check_cache(cache, &c, err, cap) || check_heads(c, n_head, max_nodes, err, cap)) return 0;
  return layout(c, sm_count(device), use_tc(c, n_head / c.n_kv_head, max_nodes) ? TR : RW).bytes;
}

extern "C" int pcpb_op_tree_attention(void* stream, const pcpb_kv_cache* cache, const pcpb_tree_attn* args, int32_t* status, char* err, size_t cap) {
  if (err && cap) err[0] = 0;
  AttnArgs A;
  int rc = check_cache(cache, &A.c, err, cap);
  if (rc) return rc;
  if (!args) return op_fail(err, cap, PCPB_E_INVALID, "null arguments");
  A.a = *args; A.status = status;
  const pcpb_tree_attn& a = A.a;
  if ((rc = check_heads(A.c, a.n_head, a.max_nodes, err, cap))) return rc;
  A.G = a.n_head / A.c.n_kv_head;
  if (a.n_rows < 0) return op_fail(err, cap, PCPB_E_INVALID, "negative row count");
  if (a.n_rows == 0) return PCPB_OK;
  if (!a.q || !a.k || !a.v || !a.out || !a.cu_nodes || !a.ctx_len || !a.workspace) return op_fail(err, cap, PCPB_E_INVALID, "null argument");
  if (!rows_aligned(a.q, a.q_row, a.q_head, 2) || !rows_aligned(a.k, a.k_row, a.k_head, 2) || !rows_aligned(a.v, a.v_row, a.v_head, 2) ||
      !rows_aligned(a.out, a.out_row, a.out_head, 2))
    return op_fail(err, cap, PCPB_E_INVALID, "rows of q, k, v and out must start on 16-byte boundaries");
  if (!aligned16(a.workspace)) return op_fail(err, cap, PCPB_E_INVALID, "the workspace must start on a 16-byte boundary");
  OpDevice d(err, cap);
  on_cache(d, A.c);
  d.on(a.q, "q"); d.on(a.k, "k"); d.on(a.v, "v"); d.on(a.out, "out"); d.on(a.lse, "lse"); d.on(a.cu_nodes, "cu_nodes"); d.on(a.parent, "parent");
  d.on(a.ctx_len, "ctx_len"); d.on(a.workspace, "workspace"); d.on(status, "status");
  if (d.enter()) return d.rc;
  const int blocks = sm_count(d.dev);
  const Layout L = layout(A.c, blocks, use_tc(A.c, A.G, a.max_nodes) ? TR : RW);
  if (a.workspace_bytes < L.bytes)
    return op_fail(err, cap, PCPB_E_INVALID, "workspace of %zu bytes, %zu are needed (pcpb_op_tree_attention_workspace)", a.workspace_bytes, L.bytes);
  uint8_t* ws = (uint8_t*)a.workspace;
  A.plan = (long long*)(ws + L.plan); A.part_ml = (float*)(ws + L.ml); A.part_o = (float*)(ws + L.o);
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e;
  if (A.c.head_dim == 128) e = launch_code<128>(st, A, blocks);
  else if (A.c.head_dim == 64) e = launch_code<64>(st, A, blocks);
  else e = launch_code<32>(st, A, blocks);
  return d.done(e);
}
