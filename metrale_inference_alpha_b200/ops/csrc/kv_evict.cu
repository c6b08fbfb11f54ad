// Cuts a paged cache to a budget of rows a kv head: of n rows of a (sequence, kv head) the last `recent` stay and, of the others, those of the
// largest mass (of equal ones the first), `keep` in all, in their order. Rows, mass and the list of them move together.
//
//   select  finds the mass of the last row that stays, digit by digit from the top (11, 11 and 10 bits of an order-preserving image, a histogram in
//           shared memory each), then writes the list in order by counting ballots. A CTA holds its rows' mass in registers, up to 64 a thread, and
//           up to eight CTAs of a cluster add up their histograms: mass is read once.
//   move    copies the rows. A kept row's place is never behind it, so in place only a row's own round can be in its way: each round is read before
//           any of it is written, and later rounds' rows lie behind everything that is written before them.
//
// Selection is bound by the latency of its passes over the registers (8 sequences of 9001 to 32749 rows, 8 heads: 25 us, 6 MB read), copies into other
// blocks by memory (4000 rows of each, 8 heads of 128 bf16: 49 us, 262 MB moved, 5.4 TB/s with what L2 keeps); together 74. One sequence of 4352 to 4096
// in place, e4m3, 20 us, three of 70 to 500 to 128 8: latency of both. (B200, in a graph.)
#include "common.cuh"
#include "kv_mass.h"
#include "smem_limit.h"

namespace {

using mbm::context;

// Flat slot of row j of a sequence, which a cache of the device's memory holds in 31 bits; a block that the cache does not have is reported and read as
// block 0, or not written (-1).
__device__ __forceinline__ int block_of(const MbEvictArgs& a, int j) {
  return (int)((unsigned long long)(unsigned)j * a.block_magic >> a.block_shift);        // j / block_size for j < 2^30
}
template <bool WRITE = false>
__device__ __forceinline__ int slot_of(const MbEvictArgs& a, int j, int b) {
  const int bi = block_of(a, j);
  if ((unsigned)b >= (unsigned long long)a.num_blocks) {
    if (a.status) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
    return WRITE ? -1 : j - bi * a.block_size;
  }
  return b * a.block_size + (j - bi * a.block_size);
}
template <bool WRITE = false>
__device__ __forceinline__ int slot_in(const MbEvictArgs& a, const int* table, int j) {
  return slot_of<WRITE>(a, j, __ldg(table + block_of(a, j)));
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

constexpr int kThreads = 512, kWarps = kThreads / 32, kMaxPer = 64, kSegment = kThreads * kMaxPer, kMaxCluster = 8, kBins = 4 * kThreads, kStaged = 2048;

__device__ __forceinline__ int4 dsmem_ld_s4(const int* local, uint32_t rank) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(mb::dsmem_addr(mb::smem_u32(local), rank))
               : "memory");
  return v;
}
// over the first WIDTH lanes
template <int WIDTH = 32>
__device__ __forceinline__ int inclusive(int v, int lane) {
#pragma unroll
  for (int o = 1; o < WIDTH; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  return v;
}

// A cluster of CTAs (often of one) a (sequence, kv head). CTA r has rows [r * 512 E, ...) of it, a warp 32 E of them, E at most PER.
template <int PER>
__global__ void __launch_bounds__(kThreads, PER <= 16 ? 2 : 1) evict_select_kernel(const MbEvictArgs a) {
  __shared__ __align__(16) int hist[3][kBins], s_total[4];
  __shared__ __align__(16) int4 s_bins[kThreads];
  __shared__ int warp_tot[3][kWarps], s_gt[kWarps], s_eq[kWarps], s_block[kStaged];
  const int h = blockIdx.x, s = blockIdx.y, cluster = gridDim.z, rank = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  auto sync_all = [&] {
    if (cluster > 1) mb::cluster_sync_all();
    else __syncthreads();
  };
  mb::pdl_launch_dependents();                                         // the copies' CTAs come up under this and wait for its end
  const int n = context(a.ctx_len, s, a.max_ctx, a.status), m = min(n, a.keep), old = n - min(n, a.recent);
  const float* x = a.mass + s * a.mass_seq + h * a.mass_head;
  const int E = (n + kThreads * cluster - 1) / (kThreads * cluster);   // rows of a thread
  const int i0 = (rank * kWarps + warp) * 32 * E + lane;               // its e-th is i0 + 32 e
  float f[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) f[e] = e < E && i0 + 32 * e < n ? x[i0 + 32 * e] : 0.f;
  // the CTA's rows' blocks come along: looked up one by one behind the selection they were a third of the time
  const int* table = a.block_table + s * a.table_ld;
  const int row0 = rank * kThreads * E, block0 = block_of(a, row0), blocks = row0 < n ? block_of(a, min(n, row0 + kThreads * E) - 1) - block0 + 1 : 0;
  const bool staged = blocks <= kStaged;
  if (staged)
    for (int i = tid; i < blocks; i += kThreads) s_block[i] = __ldg(table + block0 + i);
#pragma unroll
  for (int i = 0; i < 3; ++i) *reinterpret_cast<int4*>(&hist[i][4 * tid]) = make_int4(0, 0, 0, 0);
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
      const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, bins = d < 2 ? kBins : kBins / 2;
#pragma unroll
      for (int e = 0; e < PER; ++e)
        if (e < E) {
          const uint32_t k = key_of(f[e]);
          if (i0 + 32 * e < old && (k & mask) == prefix) atomicAdd(&hist[d][(k >> shift) & (bins - 1)], 1);
        }
      sync_all();
      // bins from the top, four a thread, over the cluster
      {
        const int b = bins - 4 - 4 * tid;
        int4 c = make_int4(0, 0, 0, 0);
        if (b >= 0) {
          if (cluster > 1) {
            for (int r0 = 0; r0 < cluster; r0 += 4) {
              int4 y[4];
#pragma unroll
              for (int r = 0; r < 4; ++r) y[r] = r0 + r < cluster ? dsmem_ld_s4(&hist[d][b], r0 + r) : make_int4(0, 0, 0, 0);
#pragma unroll
              for (int r = 0; r < 4; ++r) c = make_int4(c.x + y[r].x, c.y + y[r].y, c.z + y[r].z, c.w + y[r].w);
            }
          } else {
            c = *reinterpret_cast<const int4*>(&hist[d][b]);
          }
        }
        s_bins[tid] = c;
        const int mine = __reduce_add_sync(0xffffffffu, c.x + c.y + c.z + c.w);
        if (lane == 0) warp_tot[d][warp] = mine;
      }
      __syncthreads();
      // every warp finds the warp whose bins take the count across `need`, the lane of it and the bin
      const int tot = lane < kWarps ? warp_tot[d][lane] : 0, upto = inclusive<kWarps>(tot, lane);
      const int w = __ffs(__ballot_sync(0xffffffffu, lane < kWarps && upto >= need)) - 1;
      need -= __shfl_sync(0xffffffffu, upto - tot, w);
      const int4 c = s_bins[w * 32 + lane];
      const int sum = c.x + c.y + c.z + c.w, in = inclusive(sum, lane), l = __ffs(__ballot_sync(0xffffffffu, in >= need)) - 1;
      need -= __shfl_sync(0xffffffffu, in - sum, l);
      const int4 q = s_bins[w * 32 + l];
      int b = bins - 1 - 4 * (w * 32 + l);
      for (const int c1 : {q.w, q.z, q.y}) {
        if (need <= c1) break;
        need -= c1;
        --b;
      }
      prefix |= (uint32_t)b << shift;
      mask |= (uint32_t)(bins - 1) << shift;
    }
  } else if (need <= 0) {                                              // no key is above it, and none of those equal to it is wanted
    prefix = 0xffffffffu;
    need = 0;
  }                                                                    // else all of them: every key is above 0
  // ---- rows that stay: those above the key and the recent ones, and the first `need` equal to it
  auto stays = [&](int e, bool& equal) {
    const int i = i0 + 32 * e;
    const uint32_t k = key_of(f[e]);
    equal = i < old && k == prefix;
    return i < n && (i >= old || k > prefix);
  };
  int gt = 0, eq = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (e < E) {
      bool equal;
      gt += __popc(__ballot_sync(0xffffffffu, stays(e, equal)));
      eq += __popc(__ballot_sync(0xffffffffu, equal));
    }
  if (lane == 0) {
    s_gt[warp] = gt;
    s_eq[warp] = eq;
  }
  __syncthreads();
  // rows in front of this warp's: of its own CTA, and of the CTAs in front
  int gt_before = __reduce_add_sync(0xffffffffu, lane < warp ? s_gt[lane] : 0), eq_before = __reduce_add_sync(0xffffffffu, lane < warp ? s_eq[lane] : 0);
  if (cluster > 1) {
    if (warp == kWarps - 1 && lane == 0) {
      s_total[0] = gt_before + gt;
      s_total[1] = eq_before + eq;
    }
    mb::cluster_sync_all();
    const int4 y = lane < rank ? dsmem_ld_s4(s_total, lane) : make_int4(0, 0, 0, 0);       // a lane a CTA
    gt_before += __reduce_add_sync(0xffffffffu, y.x);
    eq_before += __reduce_add_sync(0xffffffffu, y.y);
    mb::cluster_sync_all();                                            // a CTA's shared memory outlives what others read of it
  }
  // every row's mass is in registers by now, in all CTAs: it may be written over
  float* y = a.mass_out + s * a.out_seq + h * a.out_head;
  int* kept = a.kept + ((size_t)s * a.Hkv + h) * a.keep;
  int* slots = a.slots + ((size_t)s * a.Hkv + h) * a.keep;
  const uint32_t before = (1u << lane) - 1;
  int first = 0x7fffffff;
#pragma unroll
  for (int e = 0; e < PER; ++e)
    if (e < E) {
      const int i = i0 + 32 * e;
      bool is_equal;
      const bool is_above = stays(e, is_equal);
      const uint32_t bg = __ballot_sync(0xffffffffu, is_above), be = __ballot_sync(0xffffffffu, is_equal);
      const int rank_eq = eq_before + __popc(be & before);
      const int to = gt_before + __popc(bg & before) + min(rank_eq, need);
      if (is_above || (is_equal && rank_eq < need)) {
        kept[to] = i;
        slots[to] = staged ? slot_of(a, i, s_block[block_of(a, i) - block0]) : slot_in(a, table, i);
        y[to] = f[e];
      } else if (i < n) {
        first = min(first, i);
      }
      gt_before += __popc(bg);
      eq_before += __popc(be);
    }
  for (int i = m + rank * kThreads + tid; i < a.keep; i += kThreads * cluster) kept[i] = -1;
  for (int i = m + rank * kThreads + tid; i < a.max_ctx; i += kThreads * cluster) y[i] = 0.f;
  if (a.in_place) {
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0 && first < m) atomicMin(&a.first[s * a.Hkv + h], first);
  }
}

// More rows than a cluster holds: one CTA, which reads the mass again for every digit of 8 bits and for the list. Bound by that CTA's passes: 8 heads of 300007
// e4m3 rows to 4096, with their copies, 461 us, a million 1500 (262144, in a cluster, 61); contexts of this length are cut seldom.
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

// K (x even) or V of a (sequence, kv head) into blocks of its own: 256 >> bits rows at a time of 2^bits pieces of 16 bytes, eight rows a thread.
constexpr int kDeep = 8;

__global__ void __launch_bounds__(256) evict_copy_kernel(const MbEvictArgs a, int bits) {
  mb::pdl_wait();
  const int h = blockIdx.y, s = blockIdx.z, m = a.new_len[s], step = 256 >> bits, r0 = (blockIdx.x >> 1) * step * kDeep + (threadIdx.x >> bits);
  const int* slots = a.slots + ((size_t)s * a.Hkv + h) * a.keep;
  uint8_t* cache = reinterpret_cast<uint8_t*>(blockIdx.x & 1 ? a.v_cache : a.k_cache);
  const int* to = a.dst_table + s * a.dst_ld;
  const size_t pitch = (size_t)a.Hkv * a.row_bytes, col = (size_t)h * a.row_bytes + (threadIdx.x & ((1 << bits) - 1)) * 16;
  int src[kDeep], dst[kDeep];
  uint4 v[kDeep];
#pragma unroll
  for (int k = 0; k < kDeep; ++k) src[k] = r0 + k * step < m ? slots[r0 + k * step] : -1;
#pragma unroll
  for (int k = 0; k < kDeep; ++k) dst[k] = src[k] >= 0 ? __ldg(to + block_of(a, r0 + k * step)) : -1;
#pragma unroll
  for (int k = 0; k < kDeep; ++k)
    if (src[k] >= 0) v[k] = *reinterpret_cast<const uint4*>(cache + src[k] * pitch + col);
#pragma unroll
  for (int k = 0; k < kDeep; ++k) dst[k] = src[k] >= 0 ? slot_of<true>(a, r0 + k * step, dst[k]) : -1;
#pragma unroll
  for (int k = 0; k < kDeep; ++k)
    if (dst[k] >= 0) *reinterpret_cast<uint4*>(cache + dst[k] * pitch + col) = v[k];
}

// The same inside the sequence's own blocks. A row's place is never behind it, so that only a round's own rows can be in its way: a cluster brings
// 64 KB a CTA into shared memory, waits for that everywhere, and writes. Later rounds' rows lie behind all that is written before them.
constexpr int kRoundB = 64 * 1024;

__global__ void __launch_bounds__(256) evict_move_kernel(const MbEvictArgs a, int bits) {
  extern __shared__ __align__(16) uint8_t smem[];
  mb::pdl_wait();
  const int cluster = gridDim.x >> 1, rank = blockIdx.x % cluster, h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, m = a.new_len[s];
  const int* slots = a.slots + ((size_t)s * a.Hkv + h) * a.keep;
  uint8_t* cache = reinterpret_cast<uint8_t*>(blockIdx.x / cluster ? a.v_cache : a.k_cache);
  const int* table = a.block_table + s * a.table_ld;
  const size_t pitch = (size_t)a.Hkv * a.row_bytes, col = (size_t)h * a.row_bytes + (tid & ((1 << bits) - 1)) * 16;
  const int step = 256 >> bits, mine = kRoundB / 16 >> bits;           // rows at a time, rows of a round
  constexpr int kLoads = kRoundB / (256 * 16);
  for (int r0 = a.first[s * a.Hkv + h]; r0 < m; r0 += mine * cluster) {
    const int b = r0 + rank * mine + (tid >> bits), e = min(m, r0 + (rank + 1) * mine);
    int at[kLoads];
#pragma unroll
    for (int k = 0; k < kLoads; ++k) at[k] = b + k * step < e ? slots[b + k * step] : -1;
#pragma unroll
    for (int k = 0; k < kLoads; ++k)
      if (at[k] >= 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(mb::smem_u32(smem + (k * 256 + tid) * 16)), "l"(cache + at[k] * pitch + col) : "memory");
#pragma unroll
    for (int k = 0; k < kLoads; ++k) at[k] = b + k * step < e ? slot_in<true>(a, table, b + k * step) : -1;
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (cluster > 1) mb::cluster_sync_all();
    else __syncthreads();
#pragma unroll
    for (int k = 0; k < kLoads; ++k)                                   // what a thread brought it takes away
      if (at[k] >= 0) *reinterpret_cast<uint4*>(cache + at[k] * pitch + col) = *reinterpret_cast<const uint4*>(smem + (k * 256 + tid) * 16);
  }
}

}  // namespace

extern "C" int mb_kv_evict(const MbEvictArgs* given, cudaStream_t stream) {
  if (!given) return MB_ERR_BAD_ARG;
  MbEvictArgs args = *given, *a = &args;
  if (a->num_seqs <= 0 || a->num_seqs > 65535 || a->Hkv <= 0 || a->Hkv > 65535 || a->keep <= 0 || a->recent < 0 || a->recent > a->keep || a->max_ctx <= 0 ||
      a->block_size <= 0 || a->num_blocks <= 0 || a->row_bytes < 64 || (a->row_bytes & (a->row_bytes - 1)) || !a->mass || !a->mass_out || !a->ctx_len || !a->kept ||
      !a->new_len || !a->first || !a->slots || !a->block_table || !a->dst_table || !a->k_cache || !a->v_cache)
    return MB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache)) & 15) return MB_ERR_UNSUPPORTED;
  if (a->num_blocks * a->block_size >= (1ll << 31)) return MB_ERR_TOO_LARGE;
  // ceil(2^k / d) with 2^(k - 30) >= d, so that the product is off by less than 1 / d below 2^30
  int k = 30;
  while (1ll << (k - 30) < a->block_size) ++k;
  a->block_shift = k;
  a->block_magic = (unsigned)(((1ull << k) + a->block_size - 1) / a->block_size);
  const long long heads = (long long)a->Hkv * a->num_seqs;
  cudaError_t e;
  if (a->max_ctx <= kSegment * kMaxCluster) {
    // 16 rows a thread, in as many CTAs as the chip's 148 SMs hold at once (two each); where there are more, up to 64. Fewer take a kernel with less of its loops to pass.
    int cluster = 1;
    while (cluster * kSegment < a->max_ctx || (cluster < kMaxCluster && cluster * kThreads * 16 < a->max_ctx && heads * cluster * 2 <= 2 * 148)) cluster *= 2;
    const int per = (a->max_ctx + cluster * kThreads - 1) / (cluster * kThreads);
    auto kern = per <= 1 ? evict_select_kernel<1> : per <= 4 ? evict_select_kernel<4> : per <= 16 ? evict_select_kernel<16> : evict_select_kernel<kMaxPer>;
    e = mb::launch_kernel_ex(kern, dim3(a->Hkv, a->num_seqs, cluster), dim3(kThreads), 0, stream, cluster, false, *a);
  } else {
    e = mb::launch_kernel_ex(evict_select_long_kernel, dim3(a->Hkv, a->num_seqs), dim3(1024), 0, stream, 1, false, *a);
  }
  if (e != cudaSuccess) return (int)e;
  const int held = a->keep < a->max_ctx ? a->keep : a->max_ctx;
  int bits = 0;
  while (16 << bits < a->row_bytes) ++bits;
  if (!a->in_place) {
    const int round = (256 >> bits) * kDeep;
    return (int)mb::launch_kernel_ex(evict_copy_kernel, dim3(2 * ((held + round - 1) / round), a->Hkv, a->num_seqs), dim3(256), 0, stream, 1, mb_pdl_enabled() != 0, *a, bits);
  }
  static std::atomic<uint64_t> asked{0};
  e = mb::allow_smem(reinterpret_cast<const void*>(evict_move_kernel), kRoundB, asked);
  if (e != cudaSuccess) return (int)e;
  const int mine = kRoundB / a->row_bytes;
  int cluster = 1;                                                     // rounds as large as leave the chip (148 SMs) something to do
  while (cluster < kMaxCluster && 2 * heads * cluster < 2 * 148 && cluster * mine < held) cluster *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * cluster, a->Hkv, a->num_seqs);
  cfg.blockDim = dim3(256);
  cfg.dynamicSmemBytes = kRoundB;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = mb_pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, evict_move_kernel, (const MbEvictArgs)*a, bits);
}
