// Cuts a paged cache to a budget of rows a kv head: of n rows of a (sequence, kv head) the last `recent` stay and, of the others, those of the
// largest mass (of equal ones the first), `keep` in all, in their order. Rows, mass and the list of them move together.
//
//   select  finds the mass of the last row that stays, digit by digit from the top (11, 11 and 10 bits of an order-preserving image, a histogram in
//           shared memory each), then writes the list in order by counting ballots. A CTA holds its rows' keys in registers, 32 a thread, and up to
//           eight CTAs of a cluster add up their histograms: mass is read once.
//   move    copies the rows. A kept row's place is never behind it, so in place only a row's own round can be in its way: each round is read before
//           any of it is written, and later rounds' rows lie behind everything that is written before them.
#include "common.cuh"
#include "kv_mass.h"

namespace {

using mbm::context;

// Flat slot of row j of a sequence, which a cache of the device's memory holds in 31 bits; a block that the cache does not have is reported and read as
// block 0, or not written (-1).
template <bool WRITE = false>
__device__ __forceinline__ int slot_in(const MbEvictArgs& a, const int* table, int j) {
  const int bi = a.block_shift >= 0 ? j >> a.block_shift : j / a.block_size;
  const int b = __ldg(table + bi);
  if ((unsigned)b >= (unsigned long long)a.num_blocks) {
    if (a.status) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
    return WRITE ? -1 : j - bi * a.block_size;
  }
  return b * a.block_size + (j - bi * a.block_size);
}

// Larger key, larger mass; a NaN is the least, and both zeros are one.
__device__ __forceinline__ uint32_t key_of(float f) {
  if (f != f) f = -INFINITY;
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive prefix of `v` over the block (1024 threads), and the block's total
__device__ __forceinline__ int excl_scan(int v, int* warp_tot, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  __syncthreads();
  if (lane == 31) warp_tot[warp] = inc;
  __syncthreads();
  const int c = warp_tot[lane];
  total = __reduce_add_sync(0xffffffffu, c);
  return __reduce_add_sync(0xffffffffu, lane < warp ? c : 0) + inc - v;
}

constexpr int kMaxPer = 32, kSegment = 1024 * kMaxPer, kMaxCluster = 8, kBins = 2048;

__device__ __forceinline__ int2 dsmem_ld_s2(const int* local, uint32_t rank) {
  int2 v;
  asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(mb::dsmem_addr(mb::smem_u32(local), rank)) : "memory");
  return v;
}

// A cluster of CTAs (often of one) a (sequence, kv head). CTA r has rows [r * 1024 E, ...) of it, a warp 32 E of them, E at most PER.
template <int PER>
__global__ void __launch_bounds__(1024) evict_select_kernel(const MbEvictArgs a) {
  __shared__ __align__(8) int hist[3][kBins], s_total[2];
  __shared__ int2 s_pair[1024];
  __shared__ int warp_tot[3][32], s_gt[32], s_eq[32];
  const int h = blockIdx.x, s = blockIdx.y, cluster = gridDim.z, rank = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto sync_all = [&] {
    if (cluster > 1) mb::cluster_sync_all();
    else __syncthreads();
  };
  mb::pdl_launch_dependents();                                         // the copies' CTAs come up under this and wait for its end
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), m = min(n, a.keep), old = n - min(n, a.recent);
  const float* x = a.mass + s * a.mass_seq + h * a.mass_head;
  const int E = (n + 1024 * cluster - 1) / (1024 * cluster);           // rows of a thread
  const int i0 = (rank * 32 + warp) * 32 * E + lane;                   // its e-th is i0 + 32 e
  float f[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) f[e] = e < E && i0 + 32 * e < n ? x[i0 + 32 * e] : 0.f;
#pragma unroll
  for (int i = 0; i < 3 * kBins; i += 1024) (&hist[0][0])[i + tid] = 0;
  if (tid == 0 && rank == 0) {
    a.first[s * a.Hkv + h] = a.in_place ? m : 0;
    if (h == 0) a.new_len[s] = m;
  }
  __syncthreads();
  uint32_t prefix = 0;
  int need = n > m ? m - a.recent : old;                               // rows wanted of the first `old`
  if (need > 0 && need < old) {
    uint32_t mask = 0;
    for (int d = 0; d < 3; ++d) {
      const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bins = d < 2 ? 2048 : 1024;
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (e < E) {
          const uint32_t k = key_of(f[e]);
          if (i0 + 32 * e < old && (k & mask) == prefix) atomicAdd(&hist[d][(k >> shift) & (bins - 1)], 1);
        }
      sync_all();
      // bins from the top, two a thread: b and b - 1, over the cluster
      {
        const int b = bins - 1 - 2 * tid;
        int2 c = make_int2(0, 0);
        if (b > 0) {
          if (cluster > 1) {
            int2 y[kMaxCluster];
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) y[r] = r < cluster ? dsmem_ld_s2(&hist[d][b - 1], r) : make_int2(0, 0);
#pragma unroll
            for (int r = 0; r < kMaxCluster; ++r) c = make_int2(c.x + y[r].y, c.y + y[r].x);
          } else {
            c = make_int2(hist[d][b], hist[d][b - 1]);
          }
        }
        s_pair[tid] = c;
        const int mine = __reduce_add_sync(0xffffffffu, c.x + c.y);
        if (lane == 0) warp_tot[d][warp] = mine;
      }
      __syncthreads();
      // every warp finds the warp whose bins take the count across `need`, and the bin among them
      auto inclusive = [&](int v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += y;
        }
        return v;
      };
      const int tot = warp_tot[d][lane], upto = inclusive(tot);
      const int w = __ffs(__ballot_sync(0xffffffffu, upto >= need)) - 1;
      const int rest = need - __shfl_sync(0xffffffffu, upto - tot, w);
      const int2 c = s_pair[w * 32 + lane];
      const int in = inclusive(c.x + c.y), l = __ffs(__ballot_sync(0xffffffffu, in >= rest)) - 1;
      const int left = rest - __shfl_sync(0xffffffffu, in - c.x - c.y, l), top = __shfl_sync(0xffffffffu, c.x, l);
      const int b = bins - 1 - 2 * (w * 32 + l);
      prefix |= (uint32_t)(left > top ? b - 1 : b) << shift;
      need = left > top ? left - top : left;
      mask |= (uint32_t)(bins - 1) << shift;
    }
  } else if (need <= 0) {                                              // no key is above it, and none of those equal to it is wanted
    prefix = 0xffffffffu;
    need = 0;
  }                                                                    // else all of them: every key is above 0
  // ---- rows that stay: those above the key and the recent ones, and the first `need` equal to it
  uint32_t above = 0, equal = 0;                                       // bit e: this thread's e-th row
  int gt = 0, eq = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (e < E) {
      const int i = i0 + 32 * e;
      const uint32_t k = key_of(f[e]);
      const bool is_above = i < n && (i >= old || k > prefix), is_equal = i < old && k == prefix;
      above |= (uint32_t)is_above << e;
      equal |= (uint32_t)is_equal << e;
      gt += __popc(__ballot_sync(0xffffffffu, is_above));
      eq += __popc(__ballot_sync(0xffffffffu, is_equal));
    }
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  // rows in front of this warp's: of its own CTA, and of the CTAs in front
  int gt_before = __reduce_add_sync(0xffffffffu, lane < warp ? s_gt[lane] : 0), eq_before = __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0);
  if (cluster > 1) {
    if (warp == 31 && lane == 0) {
      s_total[0] = gt_before + gt;
      s_total[1] = eq_before + eq;
    }
    mb::cluster_sync_all();
    for (int r = 0; r < rank; ++r) {
      const int2 y = dsmem_ld_s2(s_total, r);
      gt_before += y.x;
      eq_before += y.y;
    }
    mb::cluster_sync_all();                                            // a CTA's shared memory outlives what others read of it
  }
  // every row's mass is in registers by now, in all CTAs: it may be written over
  float* y = a.mass_out + s * a.out_seq + h * a.out_head;
  int* kept = a.kept + ((size_t)s * a.Hkv + h) * a.keep;
  int* slots = a.slots + ((size_t)s * a.Hkv + h) * a.keep;
  const int* table = a.block_table + s * a.table_ld;
  const uint32_t before = (1u << lane) - 1;
  int first = 0x7fffffff;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (e < E) {
      const int i = i0 + 32 * e;
      const bool is_above = above >> e & 1, is_equal = equal >> e & 1;
      const uint32_t bg = __ballot_sync(0xffffffffu, is_above), be = __ballot_sync(0xffffffffu, is_equal);
      const int rank_eq = eq_before + __popc(be & before);
      const int to = gt_before + __popc(bg & before) + min(rank_eq, need);
      if (is_above || (is_equal && rank_eq < need)) {
        kept[to] = i;
        slots[to] = slot_in(a, table, i);
        y[to] = f[e];
      } else if (i < n) {
        first = min(first, i);
      }
      gt_before += __popc(bg);
      eq_before += __popc(be);
    }
  for (int i = m + rank * 1024 + tid; i < a.keep; i += 1024 * cluster) kept[i] = -1;
  for (int i = m + rank * 1024 + tid; i < a.max_ctx; i += 1024 * cluster) y[i] = 0.f;
  if (a.in_place) {
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first < m) atomicMin(&a.first[s * a.Hkv + h], first);
  }
}

// More rows than a cluster holds: one CTA, which reads the mass again for every digit of 8 bits and for the list.
__global__ void __launch_bounds__(1024) evict_select_long_kernel(const MbEvictArgs a) {
  __shared__ int hist[256], warp_tot[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need, s_first;
  const int h = blockIdx.x, s = blockIdx.y, tid = threadIdx.x;
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), m = min(n, a.keep), old = n - min(n, a.recent);
  const float* x = a.mass + s * a.mass_seq + h * a.mass_head;
  float* y = a.mass_out + s * a.out_seq + h * a.out_head;
  int* kept = a.kept + ((size_t)s * a.Hkv + h) * a.keep;
  int* slots = a.slots + ((size_t)s * a.Hkv + h) * a.keep;
  const int* table = a.block_table + s * a.table_ld;
  if (tid == 0) {
    s_first = m;
    if (h == 0) a.new_len[s] = m;
  }
  uint32_t prefix = 0, mask = 0;
  int need = n > m ? m - a.recent : old;
  if (need > 0 && need < old) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < old; i += 1024) {
        const uint32_t k = key_of(x[i]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
      }
      __syncthreads();
      const int b = 255 - tid, c = tid < 256 ? hist[b] : 0;
      int total;
      const int above = excl_scan(c, warp_tot, total);
      if (tid < 256 && above < need && need <= above + c) {
        s_prefix = prefix | ((uint32_t)b << shift);
        s_need = need - above;
      }
      __syncthreads();
      prefix = s_prefix;
      need = s_need;
      mask |= 255u << shift;
      __syncthreads();
    }
  } else if (need <= 0) {
    prefix = 0xffffffffu;
    need = 0;
  }
  // rows in order, 1024 at a time: a round's mass is read before any of it is written over
  int eq_before = 0, at = 0;
  for (int i0 = 0; i0 < n; i0 += 1024) {
    const int i = i0 + tid;
    const float f = i < n ? x[i] : 0.f;
    const uint32_t k = key_of(f);
    const bool eq = i < old && k == prefix;
    int total;
    const int rank = eq_before + excl_scan(eq, warp_tot, total);
    eq_before += total;
    const bool in = i < n && (i >= old || k > prefix || (eq && rank < need));
    const int to = at + excl_scan(in, warp_tot, total);
    at += total;
    if (in) {
      kept[to] = i;
      slots[to] = slot_in(a, table, i);
      y[to] = f;
    }
    if (i < n && !in) atomicMin(&s_first, to);
  }
  __syncthreads();
  for (int i = m + tid; i < a.keep; i += 1024) kept[i] = -1;
  for (int i = m + tid; i < a.max_ctx; i += 1024) y[i] = 0.f;
  if (tid == 0) a.first[s * a.Hkv + h] = a.in_place ? s_first : 0;
}

// K (x even) or V of a (sequence, kv head), 2^lane_bits pieces of 16 bytes of its rows' width a CTA, THREADS >> lane_bits times DEEP rows a round. In
// place a CTA takes all rounds in order; into blocks of their own rows do not get into each other's way, and every CTA takes one.
template <int THREADS, int DEEP, bool IN_PLACE>
__global__ void __launch_bounds__(THREADS) evict_move_kernel(const MbEvictArgs a, int lane_bits) {
  mb::pdl_wait();
  const int lanes = 1 << lane_bits, strips = a.row_bytes / (16 * lanes), strip = (blockIdx.x >> 1) % strips, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
  const int m = a.new_len[s], step = THREADS >> lane_bits, round = step * DEEP;
  const int* slots = a.slots + ((size_t)s * a.Hkv + h) * a.keep;
  uint8_t* cache = reinterpret_cast<uint8_t*>(blockIdx.x & 1 ? a.v_cache : a.k_cache);
  const int* to = a.dst_table + s * a.dst_ld;
  const size_t pitch = (size_t)a.Hkv * a.row_bytes, col = (size_t)h * a.row_bytes + (size_t)(strip * lanes + (tid & (lanes - 1))) * 16;
  int r0 = (IN_PLACE ? a.first[s * a.Hkv + h] : ((int)blockIdx.x >> 1) / strips * round) + (tid >> lane_bits);
  const int last = IN_PLACE ? m : min(m, r0 - (tid >> lane_bits) + round);
  // whole CTAs go round together
  for (; r0 - (tid >> lane_bits) < last; r0 += round) {
    uint4 v[DEEP];
    int dst[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      const int r = r0 + k * step;
      dst[k] = -1;
      if (r < m) {
        v[k] = *reinterpret_cast<const uint4*>(cache + slots[r] * pitch + col);
        dst[k] = slot_in<true>(a, to, r);
      }
    }
    if (IN_PLACE) __syncthreads();
#pragma unroll
    for (int k = 0; k < DEEP; ++k)
      if (dst[k] >= 0) *reinterpret_cast<uint4*>(cache + dst[k] * pitch + col) = v[k];
  }
}

}  // namespace

extern "C" int mb_kv_evict(const MbEvictArgs* given, cudaStream_t stream) {
  if (!given) return MB_ERR_BAD_ARG;
  MbEvictArgs args = *given, *a = &args;
  if ( a->num_seqs <= 0 || a->num_seqs > 65535 || a->Hkv <= 0 || a->Hkv > 65535 || a->keep <= 0 || a->recent < 0 || a->recent > a->keep || a->max_ctx < 0 ||
      a->block_size <= 0 || a->num_blocks <= 0 || a->row_bytes < 64 || (a->row_bytes & (a->row_bytes - 1)) || !a->mass || !a->mass_out || !a->ctx_len || !a->kept ||
      !a->new_len || !a->first || !a->slots || !a->block_table || !a->dst_table || !a->k_cache || !a->v_cache)
    return MB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return MB_ERR_UNSUPPORTED;
  if (a->num_blocks * a->block_size >= (1ll << 31)) return MB_ERR_TOO_LARGE;
  a->block_shift = (a->block_size & (a->block_size - 1)) == 0 ? 31 - __builtin_clz(a->block_size) : -1;
  const long long heads = (long long)a->Hkv * a->num_seqs;
  cudaError_t e;
  if (a->max_ctx <= kSegment * kMaxCluster) {
    // eight rows a thread, in as many CTAs as the chip holds at once; where there are more, up to 32
    int cluster = 1;
    while (cluster * kSegment < a->max_ctx || (cluster < kMaxCluster && cluster * 8192 < a->max_ctx && heads * cluster * 2 <= 2 * 148)) cluster *= 2;
    auto kern = cluster * 8192 >= a->max_ctx ? evict_select_kernel<8> : evict_select_kernel<kMaxPer>;
    e = mb::launch_kernel_ex(kern, dim3(a->Hkv, a->num_seqs, cluster), dim3(1024), 0, stream, cluster, false, *a);
  } else {
    e = mb::launch_kernel_ex(evict_select_long_kernel, dim3(a->Hkv, a->num_seqs), dim3(1024), 0, stream, 1, false, *a);
  }
  if (e != cudaSuccess) return (int)e;
  const int held = a->keep < a->max_ctx ? a->keep : a->max_ctx, pieces = a->row_bytes / 16;
  if (held == 0) return 0;
  if (a->in_place) {
    // the rows of a strip follow each other, so narrow strips, down to a sector, while they give the chip more CTAs to run at once
    int lanes = pieces, bits = 0;
    while (lanes > 2 && 2 * heads * (pieces / lanes) < 148) lanes /= 2;
    while (1 << bits < lanes) ++bits;
    return (int)mb::launch_kernel_ex(evict_move_kernel<512, 8, true>, dim3(2 * (pieces / lanes), a->Hkv, a->num_seqs), dim3(512), 0, stream, 1, true, *a, bits);
  }
  int bits = 0;
  while (1 << bits < pieces) ++bits;
  const int round = (256 >> bits) * 8, rounds = (held + round - 1) / round;
  return (int)mb::launch_kernel_ex(evict_move_kernel<256, 8, false>, dim3(2 * rounds, a->Hkv, a->num_seqs), dim3(256), 0, stream, 1, true, *a, bits);
}
