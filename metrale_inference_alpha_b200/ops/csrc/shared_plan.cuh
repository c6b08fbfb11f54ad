// How the work over prefixes is shared out: what the kernels of shared_prefix.cuh and the join of shared_attn.cu compute alike.
//
// Per kv head, the query rows behind a prefix (tokens x heads of a group) are numbered token * G + head and cut into units of 2 * 128 rows, or one of
// 128 where no more are left (heads of 256 dims: all of 128). All units' tiles of cached tokens lie one behind the other on a line; a tile of a double
// unit takes two places of it, since it takes about twice the time. Of the line's W places every CTA takes as many, give or take one: units that it covers
// whole, and parts of its first and last one. A part that holds a unit's first tile leaves its outputs by row (`first`), the others, at most
// one a CTA, by CTA (`rest`).
#pragma once
#include "common.cuh"
#include "shared_attn.h"

namespace mbs {

constexpr int kMaxGroups = 1024, kRowTile = 128;

template <int D>
struct Shape {
  static constexpr bool kDouble = D <= 128;                // double units
  static constexpr int kT = kDouble ? 128 : 64;            // cached tokens of a tile
};

// Groups of a call, in shared memory: first sequences (rising and inside the batch, whatever the caller's are), rows of the prefix, first place on the line
struct Plan {
  int start[kMaxGroups + 1];
  int len[kMaxGroups];
  int base[kMaxGroups + 1];
};

__device__ __forceinline__ int row_count(const Plan& s, int g, int per_seq) { return (s.start[g + 1] - s.start[g]) * per_seq; }      // per_seq: rows of a sequence

// units of a group for a kv head: double ones, and single ones behind them
template <int D>
__device__ __forceinline__ void unit_count(int rows, int& doubles, int& singles) {
  if constexpr (Shape<D>::kDouble) {
    const int rest = rows & 255;
    doubles = (rows >> 8) + (rest > 128);
    singles = rest > 0 && rest <= 128;
  } else {
    doubles = 0;
    singles = (rows + 127) >> 7;
  }
}
template <int D>
__device__ __forceinline__ int line_of_head(int rows, int tiles) {
  int doubles, singles;
  unit_count<D>(rows, doubles, singles);
  return tiles * (2 * doubles + singles);                  // the launcher sees to it that a call's line has fewer than 2^31 places
}

// by one warp
template <int D>
__device__ __forceinline__ void make_plan(const MbSharedArgs& p, Plan& s, int per_seq, int lane) {
  if (p.groups == 1) {                                     // the usual call, without the sums over groups
    const int a = p.group_start[0], b = p.group_start[1], n = p.prefix_len[0];
    const int first = min(max(a, 0), p.num_seqs), next = max(first, min(max(b, 0), p.num_seqs));
    const int len = next > first ? min(max(n, 0), p.max_prefix) : 0;
    if (lane == 0) {
      if (p.status && (a < 0 || b > p.num_seqs || b < a || (next > first && n > p.max_prefix))) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
      s.start[0] = first;
      s.start[1] = next;
      s.len[0] = len;
      s.base[0] = 0;
      s.base[1] = p.Hkv * line_of_head<D>((next - first) * per_seq, (len + Shape<D>::kT - 1) / Shape<D>::kT);
    }
    return;
  }
  int top = 0, len0 = lane < p.groups ? p.prefix_len[lane] : 0;            // asked for beside the first sequences
  for (int g0 = 0; g0 <= p.groups; g0 += 32) {
    const int g = g0 + lane;
    int a = 0;
    if (g <= p.groups) {
      a = p.group_start[g];
      const int next = g < p.groups ? p.group_start[g + 1] : a;
      if (p.status && (a < 0 || a > p.num_seqs || next < a)) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
      a = min(max(a, 0), p.num_seqs);
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, a, d);
      if (lane >= d) a = max(a, y);
    }
    a = max(a, top);
    if (g <= p.groups) s.start[g] = a;
    top = __shfl_sync(0xffffffffu, a, 31);
  }
  __syncwarp();
  int at = 0;
  for (int g0 = 0; g0 < p.groups; g0 += 32) {
    const int g = g0 + lane;
    int n = 0;
    if (g < p.groups) {
      int len = max(g0 == 0 ? len0 : p.prefix_len[g], 0);
      if (s.start[g + 1] <= s.start[g]) len = 0;
      if (len > p.max_prefix) {
        if (p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
        len = p.max_prefix;
      }
      s.len[g] = len;
      n = p.Hkv * line_of_head<D>(row_count(s, g, per_seq), (len + Shape<D>::kT - 1) / Shape<D>::kT);
    }
    int x = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (g < p.groups) s.base[g] = at + x - n;
    at += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) s.base[p.groups] = at;
}

// The line's W places over `ctas`: the first place of CTA c, and the CTA that has place x
struct Share {
  int each, more;                          // CTAs in front of `more` have a place more
  __device__ __forceinline__ Share(int W, int ctas) : each(W / ctas), more(W % ctas) {}
  __device__ __forceinline__ int first(int c) const { return c * each + min(c, more); }
  __device__ __forceinline__ int owner(int x) const { return x < more * (each + 1) ? x / (each + 1) : more + (x - more * (each + 1)) / each; }
};
// CTAs that take part: short prefixes are latency, so every place may go to a CTA of its own
__device__ __forceinline__ int used_ctas(int W, int ctas) { return max(1, min(ctas, W)); }

struct Part {
  int group, kvh, row0, rows, two;         // a unit: its first row in the group, its rows, whether it is a double one
  int t0, t1;                              // tiles of the part
};
// tiles [t0, t1) of a unit that begins at place `at` with `tiles` of them, which lie in places [b0, b1)
__device__ __forceinline__ void tiles_in(int at, int tiles, int two, int b0, int b1, int& t0, int& t1) {
  t0 = (max(b0 - at, 0) + two) >> two;
  t1 = (min(max(b1 - at, 0), tiles << two) + two) >> two;
}

// a / b for quotients below 2^20, by a product that is off by one at most
__device__ __forceinline__ unsigned quotient(unsigned a, unsigned b) {
  unsigned q = (unsigned)(__uint2float_rn(a) * __fdividef(1.f, __uint2float_rn(b)));
  int r = (int)(a - q * b);
  if (r < 0) {
    --q;
    r += b;
  }
  return r >= (int)b ? q + 1 : q;
}

// The part at `pos`, which moves behind it; false at the end. Parts without tiles are left out.
template <int D>
__device__ __forceinline__ bool next_part(const Plan& s, int groups, int per_seq, int& pos, int end, Part& x) {
  while (pos < end) {
    int lo = 0, hi = groups;               // base[lo] <= pos < base[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s.base[mid] <= pos) lo = mid;
      else hi = mid;
    }
    x.group = lo;
    const int rows = row_count(s, lo, per_seq), tiles = (s.len[lo] + Shape<D>::kT - 1) / Shape<D>::kT;
    int doubles, singles;
    unit_count<D>(rows, doubles, singles);
    const unsigned head = (unsigned)tiles * (2 * doubles + singles), in = pos - s.base[lo];
    x.kvh = quotient(in, head);
    const unsigned w = in - x.kvh * head, d = 2u * tiles * doubles;
    x.two = w < d;
    const unsigned size = (unsigned)tiles << x.two, v = x.two ? w : w - d, u = quotient(v, size);
    x.row0 = x.two ? u * 256 : doubles * 256 + u * 128;
    const int at = pos - (int)(v - u * size);
    x.rows = min(rows - x.row0, x.two ? 256 : 128);
    tiles_in(at, tiles, x.two, pos, end, x.t0, x.t1);
    pos = min(end, at + (int)size);
    if (x.t1 > x.t0) return true;
  }
  return false;
}

// Workspace of a call: `first` outputs [2][Hkv][D / 4][rows] of four dims, `rest` [ctas][2][D / 4][128], each with maxima (log2 domain) and sums. A single
// unit's tiles are taken in turn by two accumulators, whose results are the two of the leading dim; double units and heads of 256 dims use the first.
struct Ws {
  size_t first, first_ml, rest, rest_ml, own, own_ml, bytes;
  int ctas, parts, step;                   // parts of a sequence's own rows; tokens whose own rows are attended at once
  int G, per_seq;                          // query heads of a group, rows of a sequence
};

}  // namespace mbs
