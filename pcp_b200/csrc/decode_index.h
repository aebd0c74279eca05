// Index arithmetic of the decode operators, the same code on the device and in the CPU tests (plain C++, no CUDA header).
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define PCPB_HD __host__ __device__ __forceinline__
#else
#define PCPB_HD inline
#endif

namespace pcpb {

// Lengths of one sequence as they may be used: n nodes (or entries) from n0 on, ctx cached positions; bad: something was clipped.
struct SeqLen { int n0, n, ctx, bad; };
PCPB_HD SeqLen clip_seq(int lo, int hi, int ctx, int n_rows, int max_nodes, int top) {
  SeqLen s;
  s.bad = lo < 0 || hi < lo || hi > n_rows || hi - lo > max_nodes || ctx < 0 || ctx > top;
  if (s.bad) {
    lo = lo < 0 ? 0 : lo > n_rows ? n_rows : lo;
    hi = hi < lo ? lo : hi > n_rows ? n_rows : hi;
    if (hi - lo > max_nodes) hi = lo + max_nodes;
    ctx = ctx < 0 ? 0 : ctx > top ? top : ctx;
  }
  s.n0 = lo; s.n = hi - lo; s.ctx = ctx;
  return s;
}
// A node's parent as it may be followed: a number below its own, or -1.
PCPB_HD int clip_parent(int p, int i, int* bad) {
  const int b = p < -1 || p >= i;
  *bad |= b;
  return b ? -1 : p;
}
// A block-table entry as it may be used: a page of the cache, or -1.
PCPB_HD int clip_page(int p, int n_pages) { return p >= 0 && p < n_pages ? p : -1; }
// Element offset of row `off` of head h in a page (64 bits: a cache may hold more than 2^31 elements)
PCPB_HD long long page_row(int page, long long page_stride, int h, int page_tokens, int off, int width) {
  return (long long)page * page_stride + ((long long)h * page_tokens + off) * width;
}

// Equal shares of `total` tiles for `blocks` blocks: block c has [c share, min(total, (c + 1) share)).
PCPB_HD long long tile_share(long long total, int blocks) { return (total + blocks - 1) / blocks; }
// An item's tiles [first, first + count) lie in blocks c0 .. c1.  Block c0 holds its part in slot 2 c0 (the item starts with the
// block) or 2 c0 + 1, every later block in slot 2 c.
struct Parts { int c0, c1, slot0; };
PCPB_HD Parts parts_of(long long first, int count, long long share) {
  Parts p;
  p.c0 = (int)(first / share); p.c1 = (int)((first + count - 1) / share);
  p.slot0 = 2 * p.c0 + (first == share * p.c0 ? 0 : 1);
  return p;
}
PCPB_HD int part_slot(const Parts& p, int c) { return c == p.c0 ? p.slot0 : 2 * c; }

}  // namespace pcpb
