// Prompts over a latent cache in expanded form: a cached row's keys and values are made for every head, k = [W_k c | rotated part], v = W_v c, and attended
// as usual. Per head and pair 192 + 128 multiply-adds instead of the 576 + 512 of the absorbed form, for 512 x 256 a cached row and head in front.
//
// Three launches: cached rows to consecutive ones (6 us for 8192 of them, latency), the expansion (30 us for 16 heads: 1.15 PFLOP/s), and attention
// (260 us: 1.32 PFLOP/s of what the mask leaves, the tensor pipe 69 % busy, the special function units 56 %). Expanded rows are bf16, as cached keys and
// values would be: half a step of 2^-8 each, which is as much again as the rounding of the outputs.
#include "common.cuh"
#include "shared_attn.h"
#include "attention_rows.cuh"
#include "gemm_args.h"
#include "smem_limit.h"
#include "tensormap.h"

namespace {

using namespace mbr;

constexpr int kRow = 576, kLat = 512, kQk = 192, kNope = 128, kV = 128;

struct AttnParams {
  const int* q_start;
  const int* q_len;
  const int* ctx_len;
  const int* first;          // [seqs]: a sequence's first expanded row
  const int* bad;            // [expanded rows / 32]: the place in its sequence of the first row that is no number, or 2^31 - 1
  void* out;
  uint32_t* status;
  long long q_rows, kv_rows;
  int H, head0, max_q_len, max_ctx;
  float scale;
};

// ---- cached rows to consecutive ones, sequence s from first[s] on, a multiple of 128
struct GatherParams {
  const __nv_bfloat16* cache;
  const int* block_table;
  long long table_ld;
  const int* ctx_len;
  __nv_bfloat16* lat;
  int* first;
  int* bad;
  uint32_t* status;
  long long num_blocks, kv_rows;
  int num_seqs, block_size, max_ctx;
};

constexpr int kGather = 32;                                // rows of a CTA, four a warp

__global__ void __launch_bounds__(256) gather_kernel(const GatherParams p) {
  mb::pdl_wait();
  mb::pdl_launch_dependents();
  __shared__ long long s_at;
  __shared__ int s_seq, s_bad[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r0 = (long long)blockIdx.x * kGather;
  if (tid == 0) s_seq = -1;
  __syncthreads();
  if (warp == 0) {
    long long at = 0;
    for (int s0 = 0; s0 < p.num_seqs; s0 += 32) {
      const int s = s0 + lane;
      int n = 0;
      if (s < p.num_seqs) n = p.ctx_len[s];
      const long long len = (min(max(n, 0), p.max_ctx) + 127) & ~127;
      long long x = len;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
      }
      const long long end = at + x, begin = end - len;
      if (s < p.num_seqs) {
        if (blockIdx.x == 0) {
          p.first[s] = (int)min(begin, p.kv_rows);
          if ((n > p.max_ctx || end > p.kv_rows) && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
        }
        if (r0 >= begin && r0 < end) {
          s_seq = s;
          s_at = begin;
        }
      }
      at = __shfl_sync(0xffffffffu, end, 31);
      if (blockIdx.x > 0 && at > r0) break;
    }
  }
  __syncthreads();
  const int s = s_seq;
  if (s < 0) return;
  const int j0 = (int)(r0 - s_at) + warp * 4, n = min(max(p.ctx_len[s], 0), p.max_ctx);
  // a warp's rows: places first, then everything that is read, then the stores
  const uint4* src[4];
  uint4 v[4][3];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int j = j0 + r;
    src[r] = nullptr;
    if (j < n) {
      int b = p.block_table[s * p.table_ld + j / p.block_size];
      if (b < 0 || b >= p.num_blocks) {
        if (lane == 0 && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
        b = 0;
      }
      src[r] = reinterpret_cast<const uint4*>(p.cache + ((size_t)b * p.block_size + j % p.block_size) * kRow);
    }
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int i = 0; i < 3; ++i) v[r][i] = src[r] && lane + 32 * i < kRow / 8 ? src[r][lane + 32 * i] : make_uint4(0, 0, 0, 0);
  int bad = 0x7fffffff;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {                          // the latent: 64 pieces of 8
      const uint32_t x[4] = {v[r][i].x, v[r][i].y, v[r][i].z, v[r][i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) odd |= (x[k] & 0x7f80u) == 0x7f80u || (x[k] & 0x7f800000u) == 0x7f800000u;
    }
    odd = __any_sync(0xffffffffu, odd);
    if (odd) bad = min(bad, j0 + r);
    uint4* dst = reinterpret_cast<uint4*>(p.lat + (r0 + warp * 4 + r) * kRow) + lane;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (lane + 32 * i < kRow / 8) dst[32 * i] = odd && i < 2 ? make_uint4(0, 0, 0, 0) : v[r][i];
  }
  if (lane == 0) s_bad[warp] = bad;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) bad = min(bad, s_bad[w]);
    p.bad[blockIdx.x] = bad;
  }
}

// ---- calls in which nothing can be attended, since a maximum or a sum is 0 or q has no rows: what the others report is looked at here. One CTA.
struct NothingParams {
  const int* q_start;
  const int* q_len;
  const int* ctx_len;
  uint32_t* status;
  long long q_rows, kv_rows;
  int num_seqs, max_q_len, max_ctx;
};

__global__ void __launch_bounds__(256) nothing_kernel(const NothingParams p) {
  mb::pdl_wait();
  __shared__ unsigned long long s_rows;
  if (threadIdx.x == 0) s_rows = 0;
  __syncthreads();
  bool beyond = false;
  unsigned long long rows = 0;
  for (int s = threadIdx.x; s < p.num_seqs; s += 256) {
    const int n = p.ctx_len[s], qlen = p.q_len[s];
    beyond |= n > p.max_ctx || qlen > p.max_q_len || (qlen > 0 && (p.q_start[s] < 0 || (long long)p.q_start[s] + qlen > p.q_rows));
    rows += (min(max(n, 0), p.max_ctx) + 127) & ~127;
  }
  if (rows) atomicAdd(&s_rows, rows);
  __syncthreads();
  if ((beyond || s_rows > (unsigned long long)p.kv_rows) && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
}

// ---- expansion: kv[row, head, 256] = w[head] c[row], a product whose sums are 512 long
// A pair of CTAs owns units of 256 cached rows of one head (tcgen05.mma.cta_group::2, M = N = 256). Its rows stay in shared memory, 128 of them in either
// CTA, while the heads' weights go by, half of a head's in either: with rows fetched again for every head, as the plain product of gemm_rows.cu does, 16
// heads of 8192 rows read 268 MB out of L2 at some 6 TB/s and took 45 us; here it is half of that, and 30 us. The ring is as deep as shared memory lets it
// be: weights come as fast as its 96 KB cover L2's latency (of five places 33 us). Units are numbered heads fastest and shared out in runs of equal length.
//   warp 0      weights by TMA, 64 of the 512 at a time, a ring of six        warp 10   rows, when a run comes to others
//   warp 1      the leader's issues the products, two accumulators in turn    warps 2-9 take them to bf16, lane = row
constexpr int kExpThreads = 352, kExpRing = 6, kExpK = kLat / 64, kExpPiece = 128 * 128;
constexpr int kExpSmem = (kExpK + kExpRing) * kExpPiece + 1024;

struct ExpandParams {
  __nv_bfloat16* out;        // [rows, heads, 256]
  long long rows;
  int heads, units;
  uint32_t* status;
};

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kExpThreads, 1)
expand_kernel(const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmW, const ExpandParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* sC = smem_raw + ((1024u - (mb::smem_u32(smem_raw) & 1023u)) & 1023u);   // 8 x [128 rows x 128 B]
  uint8_t* sW = sC + kExpK * kExpPiece;
  __shared__ __align__(8) uint64_t c_full[kExpK], w_full[kExpRing];                // used in the leader: both CTAs' bytes
  __shared__ __align__(8) uint64_t c_empty, w_empty[kExpRing], acc_full[2];        // in each CTA
  __shared__ __align__(8) uint64_t acc_empty[2];                                   // used in the leader: both CTAs' warps
  __shared__ uint32_t s_tmem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = mb::cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int u0 = (int)((long long)p.units * pair / pairs), u1 = (int)((long long)p.units * (pair + 1) / pairs);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kExpK; ++i) mb::mbar_init(&c_full[i], 1);
    for (int i = 0; i < kExpRing; ++i) {
      mb::mbar_init(&w_full[i], 1);
      mb::mbar_init(&w_empty[i], 1);
    }
    mb::mbar_init(&c_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mb::mbar_init(&acc_full[i], 1);
      mb::mbar_init(&acc_empty[i], 2 * 8);
    }
    mb::mbar_fence_init();
  }
  if (warp == 1) mb::tmem_alloc2(&s_tmem, 512);
  mb::tc_fence_before();
  __syncthreads();
  mb::cluster_sync_all();                                  // barriers of both CTAs stand before either signals the other
  mb::tc_fence_after();
  const uint32_t tmem = s_tmem;
  mb::pdl_launch_dependents();
  if (warp == 0) {
    if (mb::elect_one()) {
      // weights stood before the kernel in front, which has waited for them: they are not waited for
      const int total = (u1 - u0) * kExpK;
      int g = 0;
      for (; g < total; ++g) {
        const int s = g % kExpRing, h = (u0 + g / kExpK) % p.heads;
        if (!mb::mbar_wait(&w_empty[s], ((g / kExpRing) & 1) ^ 1, p.status, MB_ST_TIMEOUT_TMA)) break;
        if (rank == 0) mb::mbar_expect_tx(&w_full[s], 2 * kExpPiece);
        mb::tma_load_2d_pair(sW + s * kExpPiece, &tmW, mb::dsmem_addr(mb::smem_u32(&w_full[s]), 0), g % kExpK * 64, h * 256 + (int)rank * 128);
      }
      // given up: the leader sees both CTAs' copies through, or waits until its waits give up; the pair leaves together
      if (g < total && rank == 0)
        for (int i = g > kExpRing ? g - kExpRing : 0; i < g; ++i) mb::mbar_wait(&w_full[i % kExpRing], (i / kExpRing) & 1, p.status, MB_ST_TIMEOUT_TMA);
    }
    __syncwarp();
  } else if (warp == 10) {
    if (mb::elect_one()) {
      mb::pdl_wait();
      int run = 0;
      for (int u = u0; u < u1; u += p.heads - u % p.heads, ++run) {
        const bool ok = run == 0 || mb::mbar_wait(&c_empty, (run - 1) & 1, p.status, MB_ST_TIMEOUT_TMA);
        if (!ok) {
          if (rank == 0)
            for (int i = 0; i < kExpK; ++i) mb::mbar_wait(&c_full[i], (run - 1) & 1, p.status, MB_ST_TIMEOUT_TMA);
          break;
        }
        for (int i = 0; i < kExpK; ++i) {
          if (rank == 0) mb::mbar_expect_tx(&c_full[i], 2 * kExpPiece);
          mb::tma_load_2d_pair(sC + i * kExpPiece, &tmC, mb::dsmem_addr(mb::smem_u32(&c_full[i]), 0), i * 64, (u / p.heads * 2 + (int)rank) * 128);
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && mb::elect_one()) {
      constexpr uint32_t kId = mb::umma_idesc(1, 1, 256, 256);
      const uint64_t dC = mb::umma_desc_sw128(mb::smem_u32(sC)), dW = mb::umma_desc_sw128(mb::smem_u32(sW));
      bool ok = true;
      int g = 0, run = 0;
      for (int u = u0; u < u1 && ok; ++u) {
        const int it = u - u0, buf = it & 1;
        const bool fresh = u == u0 || u % p.heads == 0;    // the first unit of these rows
        if (fresh && u > u0) ++run;
        ok = mb::mbar_wait(&acc_empty[buf], ((it >> 1) & 1) ^ 1, p.status, MB_ST_TIMEOUT_MMA);
        for (int i = 0; i < kExpK && ok; ++i, ++g) {
          const int s = g % kExpRing;
          if (fresh) ok = mb::mbar_wait(&c_full[i], run & 1, p.status, MB_ST_TIMEOUT_MMA);
          ok = ok && mb::mbar_wait(&w_full[s], (g / kExpRing) & 1, p.status, MB_ST_TIMEOUT_MMA);
          if (!ok) break;
          mb::tc_fence_after();
#pragma unroll
          for (int j = 0; j < 4; ++j)
            mb::umma2_f16(tmem + buf * 256, dC + i * (kExpPiece >> 4) + ((j * 32) >> 4), dW + s * (kExpPiece >> 4) + ((j * 32) >> 4), kId, (i | j) != 0);
          mb::tc_commit2(&w_empty[s]);
        }
        if (!ok) break;
        // the last signal that the pair waits for comes last: none may arrive at a CTA that has left
        if ((u + 1) % p.heads == 0 && u + 1 < u1) mb::tc_commit2(&c_empty);
        mb::tc_commit2(&acc_full[buf]);
      }
    }
    __syncwarp();
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    const uint32_t src = tmem + ((uint32_t)(q * 32) << 16) + half * 128;
    const uint32_t empty0 = mb::dsmem_addr(mb::smem_u32(&acc_empty[0]), 0);
    mb::pdl_wait();                                        // the results' place may still be read by the kernels in front of the one in front
    for (int u = u0; u < u1; ++u) {
      const int it = u - u0, buf = it & 1, h = u % p.heads;
      const long long row = (long long)(u / p.heads) * 256 + (int)rank * 128 + q * 32 + lane;
      const bool ok = mb::mbar_wait(&acc_full[buf], (it >> 1) & 1, p.status, MB_ST_TIMEOUT_EPI);
      if (!__all_sync(0xffffffffu, ok)) break;
      mb::tc_fence_after();
      float v[128];
#pragma unroll
      for (int c = 0; c < 128; c += 32) mb::tmem_ld32_async(src + buf * 256 + c, v + c);
      mb::tmem_ld_wait(v);
      mb::tc_fence_before();
      __syncwarp();
      if (lane == 0) mb::mbar_arrive_cluster(empty0 + buf * 8);
      if (row < p.rows) {
        __nv_bfloat16* dst = p.out + ((size_t)row * p.heads + h) * 256 + half * 128;
#pragma unroll
        for (int c = 0; c < 128; c += 16) {                // whole sectors: a warp's store touches 32 rows
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = pack2<false>(v[c + 2 * i], v[c + 2 * i + 1]);
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(dst + c), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                       "r"(w[6]), "r"(w[7])
                       : "memory");
        }
      }
    }
    mb::tc_fence_before();
  }
  __syncthreads();
  mb::cluster_sync_all();                                  // nothing of the pair signals or reads a CTA that has left
  if (warp == 1) {
    mb::tc_fence_after();
    mb::tmem_dealloc2(tmem, 512);
  }
}

// ---- attention: two tiles of 128 query tokens of one head a CTA on the tensor cores
//   warps 0-3, 4-7   softmax of row tile 0 / 1, thread = row: S from TMEM, the weights back to TMEM (over S) in two halves of 64 tokens
//   warp 8           copies by TMA: Q once; per 128 cached tokens five pieces of 16 KB in a ring of eight: K in three spans of 64 dims (the
//                    third is the rotated part, which all heads share), V in two halves of 64 tokens
//   warp 9           issues the products: S0 S1 | PV0 S0' PV1 S1' | ..., so that one tile's softmax runs under the other tile's products. With a warp for
//                    either tile's the two batches were interleaved and done at the same time, and both softmaxes then ran at once (8192 tokens of 16
//                    heads then took 325 us in place of 300)
//   warps 10, 11     give their registers to the softmax
// Weights through shared memory, which would let S of the next tile be made under the softmax, were slower (331 us in place of 314 then):
// 128 x 128 products of operands in shared memory read 128 bytes a cycle, all that it has.
constexpr int kT = 128, kPiece = 16384, kRing = 8, kPer = 5, kThreads = 384;
constexpr int kQTile = 3 * kPiece;
constexpr int kSmem = 2 * kQTile + kRing * kPiece + 1024;

template <int N>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

__global__ void __launch_bounds__(kThreads, 1)
mla_prompt_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                  const __grid_constant__ CUtensorMap tmR, const AttnParams p) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* sQ = smem_raw + ((1024u - (mb::smem_u32(smem_raw) & 1023u)) & 1023u);   // 2 row tiles x 3 spans x [128 rows x 128 B]
  uint8_t* sR = sQ + 2 * kQTile;
  __shared__ __align__(8) uint64_t q_full, k_full[2], v_full[2], empty[kRing], s_full[2], p_full[2][2], o_full[2];
  __shared__ uint32_t s_tmem;
  const int h = blockIdx.x, seq = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  mb::pdl_wait();
  const int qlen = p.q_len[seq], qs = p.q_start[seq], ctx = min(max(p.ctx_len[seq], 0), p.max_ctx);
  const long long first = p.first[seq];
  const int row0 = ((int)gridDim.y - 1 - (int)blockIdx.y) * 256;                   // the longest rows first
  if (row0 >= qlen) return;
  if (qlen > p.max_q_len || p.ctx_len[seq] > p.max_ctx || qs < 0 || (long long)qs + qlen > p.q_rows || first + ((ctx + 127) & ~127) > p.kv_rows) {
    if (tid == 0 && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
    return;
  }
  const int past = ctx - qlen;
  auto tiles_of = [&](int w) {                            // cached tiles that row tile w sees
    const int rows = min(qlen - row0 - w * 128, 128);
    return rows <= 0 ? 0 : (max(past + row0 + w * 128 + rows, 0) + kT - 1) / kT;
  };
  const int n0 = tiles_of(0), n1 = tiles_of(1), n = max(n0, n1);

  if (tid == 0) {
    mb::mbar_init(&q_full, 1);
    for (int i = 0; i < kRing; ++i) mb::mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) {
      mb::mbar_init(&k_full[i], 3);                       // of every second tile: the ring does not hold the pieces of three
      mb::mbar_init(&v_full[i], 2);
      mb::mbar_init(&s_full[i], 1);
      mb::mbar_init(&p_full[i][0], 4);
      mb::mbar_init(&p_full[i][1], 4);
      mb::mbar_init(&o_full[i], 1);
    }
    mb::mbar_fence_init();
  }
  if (warp == 9) mb::tmem_alloc(&s_tmem, 512);
  mb::tc_fence_before();
  __syncthreads();
  mb::tc_fence_after();
  mb::pdl_launch_dependents();                            // a dependent kernel allocates TMEM: not before this CTA has its own
  const uint32_t tmem = s_tmem;                           // S0 0-127, S1 128-255, O0 256-383, O1 384-511

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    more_regs<216>();                                     // 216 + 216 + 72 are the 3 x 168 of the launch
    const int w = warp >> 2, tok = row0 + w * 128 + (tid & 127);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128, tO = tmem + lanes + 256 + w * 128;
    const bool live = tok < qlen;
    const int limit = live ? past + tok + 1 : 0;          // cached tokens [0, limit) are visible
    const int mine = w ? n1 : n0;
    const float sc = p.scale * 1.44269504088896f;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int j = 0; j < mine; ++j) {
      ok = mb::mbar_wait(&s_full[w], j & 1, p.status, MB_ST_TIMEOUT_MMA);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      mb::tc_fence_after();
      float s[kT];
#pragma unroll
      for (int c = 0; c < kT; c += 32) mb::tmem_ld32_async(tS + c, s + c);
      mb::tmem_ld_wait(s);
      const int seen = limit - j * kT;                    // columns below this are visible
      if (!__all_sync(0xffffffffu, seen >= kT)) {
#pragma unroll
        for (int i = 0; i < kT; ++i)
          if (i >= seen) s[i] = -INFINITY;
      }
      float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int i = 4; i < kT; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], s[i]);
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
      float alpha = 1.f;
      const bool move = mx > m_run + 8.f;                 // also true on a row's first finite tile
      if (move) {
        alpha = ex2(m_run - mx);                          // 0 when the row had seen nothing yet
        m_run = mx;
      }
      if (j > 0 && __any_sync(0xffffffffu, move)) {       // S seen: the products that were issued in front of it are done
#pragma unroll
        for (int c = 0; c < kV; c += 16) {
          float ov[16];
          mb::tmem_ld16(tO + c, ov);
#pragma unroll
          for (int i = 0; i < 16; ++i) ov[i] *= alpha;
          mb::tmem_st16(tO + c, ov);
        }
      }
      const float nm = m_run == -INFINITY ? 0.f : -m_run;
      const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          float2 t = fma2(make_float2(s[q * 64 + 2 * i], s[q * 64 + 2 * i + 1]), sc2, nm2);
          t.x = ex2(t.x);
          t.y = ex2(t.y);
          sum[i & 1] = add2(sum[i & 1], t);
          pk[i] = pack2<false>(t.x, t.y);
        }
        tmem_st32(tS + q * 32, pk);
        mb::tmem_st_wait();
        mb::tc_fence_before();
        __syncwarp();
        if (lane == 0) mb::mbar_arrive(&p_full[w][q]);
      }
      l_run = l_run * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
    }
    // the first cached token that is no number, of those that the tile sees: it lies in the expanded rows as zeros
    int bad = 0x7fffffff;
    for (int j = lane; j < mine * (kT / kGather); j += 32) bad = min(bad, p.bad[first / kGather + j]);
    bad = __reduce_min_sync(0xffffffffu, bad);
    if (ok && mine > 0) {
      ok = mb::mbar_wait(&o_full[w], 0, p.status, MB_ST_TIMEOUT_MMA);
      mb::tc_fence_after();
    }
    if (__all_sync(0xffffffffu, ok)) {                    // uniform: tcgen05.ld is a whole-warp instruction
      const float inv = limit > bad ? __int_as_float(0x7fffffff) : l_run == 0.f ? 0.f : 1.f / l_run;
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.out) + ((size_t)(qs + (live ? tok : 0)) * p.H + p.head0 + h) * kV);
#pragma unroll 1
      for (int c0 = 0; c0 < kV; c0 += 64) {
        float o[64];
        if (mine > 0) {
          mb::tmem_ld32_async(tO + c0, o);
          mb::tmem_ld32_async(tO + c0 + 32, o + 32);
          mb::tmem_ld_wait(o);
        } else {
#pragma unroll
          for (int i = 0; i < 64; ++i) o[i] = 0.f;
        }
        if (live) {
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            uint32_t v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = inv == 0.f ? 0u : pack2<false>(o[c * 8 + 2 * i] * inv, o[c * 8 + 2 * i + 1] * inv);
            dst[c0 / 8 + c] = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
    mb::tc_fence_before();
  } else {
    fewer_regs<72>();
    if (warp == 8 && mb::elect_one() && n > 0) {
      // ---------------------------------------------------------- copies
      const int hq = (p.head0 + h) * kQk, hk = h * 256;
      mb::mbar_expect_tx(&q_full, n1 ? 2 * kQTile : kQTile);
      for (int w = 0; w < (n1 ? 2 : 1); ++w)
        for (int c = 0; c < 3; ++c) mb::tma_load_2d(sQ + w * kQTile + c * kPiece, &tmQ, &q_full, hq + c * 64, qs + row0 + w * 128);
      int slot = 0, i = 0;
      uint32_t parity = 1;
      bool ok = true;
      auto bring = [&](int j, int c) {                    // piece c of tile j
        if (!ok) return;
        ok = mb::mbar_wait(&empty[slot], parity, p.status, MB_ST_TIMEOUT_TMA);
        if (!ok) return;
        const int at = (int)first + j * kT;
        uint8_t* dst = sR + slot * kPiece;
        uint64_t* bar = c < 3 ? &k_full[j & 1] : &v_full[j & 1];
        mb::mbar_expect_tx(bar, kPiece);
        if (c < 2) {
          mb::tma_load_2d(dst, &tmK, bar, hk + c * 64, at);
        } else if (c == 2) {
          mb::tma_load_2d(dst, &tmR, bar, kLat, at);
        } else {
          for (int d = 0; d < 2; ++d) mb::tma_load_2d(dst + d * (kPiece / 2), &tmV, bar, hk + kNope + d * 64, at + (c - 3) * 64);
        }
        ++i;
        if (++slot == kRing) {
          slot = 0;
          parity ^= 1;
        }
      };
      for (int j = 0; j < n && ok; ++j)
        for (int c = 0; c < kPer; ++c) bring(j, c);
      // given up: no copy may still be under way when the CTA ends. A tile whose pieces were not all asked for is waited for until the wait gives up: its
      // copies are through by then
      if (!ok) {
        mb::mbar_wait(&q_full, 0, p.status, MB_ST_TIMEOUT_TMA);
        for (int j = max(0, (i - 1) / kPer - 1); j <= (i - 1) / kPer; ++j) {
          mb::mbar_wait(&k_full[j & 1], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_TMA);
          mb::mbar_wait(&v_full[j & 1], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_TMA);
        }
      }
    }
    if (warp == 9 && mb::elect_one() && n > 0) {
      // ---------------------------------------------------------- products
      constexpr uint32_t kIdS = mb::umma_idesc(1, 1, 128, kT), kIdO = mb::umma_idesc(1, 1, 128, kV, 0, 1);
      // descriptors count 16 bytes: an operand's next step is an addition
      const uint64_t dQ = mb::umma_desc_sw128(mb::smem_u32(sQ)), dK = mb::umma_desc_sw128(mb::smem_u32(sR)),
                     dV = mb::umma_desc_sw128_mn(mb::smem_u32(sR), kPiece / 2, 1024);
      // Every wait takes this thread a hundred cycles, met or not, so that tiles have a barrier for their keys and one for their values, which the first
      // row tile waits for
      auto scores = [&](int w, int j) {
        if (w == 0 || j >= n0) {
          if (!mb::mbar_wait(&k_full[j & 1], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_MMA)) return false;
          mb::tc_fence_after();
        }
#pragma unroll
        for (int c = 0; c < 3; ++c) {
          const int i = j * kPer + c;
          const uint64_t q = dQ + w * (kQTile >> 4) + ((c * kPiece) >> 4), k = dK + (i % kRing) * (kPiece >> 4);
#pragma unroll
          for (int s = 0; s < 4; ++s) mb::umma_f16(tmem + w * 128, q + ((s * 32) >> 4), k + ((s * 32) >> 4), kIdS, (c | s) != 0);
        }
        mb::tc_commit(&s_full[w]);
        return true;
      };
      auto values = [&](int w, int j) {
        if ((w == 0 || j >= n0) && !mb::mbar_wait(&v_full[j & 1], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_MMA)) return false;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int i = j * kPer + 3 + h;
          if (!mb::mbar_wait(&p_full[w][h], j & 1, p.status, MB_ST_TIMEOUT_MMA)) return false;
          mb::tc_fence_after();
          const uint64_t v = dV + (i % kRing) * (kPiece >> 4);
#pragma unroll
          for (int s = 0; s < 4; ++s) umma_f16_ta(tmem + 256 + w * 128, tmem + w * 128 + (h * 4 + s) * 8, v + ((s * 2048) >> 4), kIdO, (j | h | s) != 0);
        }
        return true;
      };
      auto release = [&](int i, int k) {
        for (; k > 0; --k, ++i) mb::tc_commit(&empty[i % kRing]);
      };
      bool ok = mb::mbar_wait(&q_full, 0, p.status, MB_ST_TIMEOUT_MMA);
      if (ok && n0 > 0) ok = scores(0, 0);
      if (ok && n1 > 0) ok = scores(1, 0);
      if (ok) release(0, 3);
      for (int j = 0; j < n && ok; ++j) {
        if (j < n0) {
          ok = values(0, j);
          if (!ok) break;
          if (j + 1 < n0) ok = scores(0, j + 1);
          else mb::tc_commit(&o_full[0]);
          if (!ok) break;
        }
        if (j < n1) ok = values(1, j);
        if (!ok) break;
        release(j * kPer + 3, 2);
        if (j + 1 < n1) ok = scores(1, j + 1);
        else if (j + 1 == n1) mb::tc_commit(&o_full[1]);
        if (!ok) break;
        if (j + 1 < n) release((j + 1) * kPer, 3);
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 9) {
    mb::tc_fence_after();
    mb::tmem_dealloc(tmem, 512);
  }
}

}  // namespace

// Workspace: the cached rows one behind the other, sequences' first rows, places of rows that are no numbers, expanded keys and values of `each` heads
struct Layout {
  size_t first, bad, kv, bytes;
};
static Layout layout(long long rows, int seqs, int each) {
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  Layout l;
  l.first = up((size_t)rows * kRow * 2);
  l.bad = l.first + up((size_t)seqs * 4);
  l.kv = l.bad + up((size_t)rows / kGather * 4);
  l.bytes = l.kv + (size_t)rows * each * 512;
  return l;
}

extern "C" {

size_t mb_mla_prompt_ws(long long kv_rows, int num_seqs, int each) { return layout(kv_rows, num_seqs, each).bytes; }

int mb_mla_prompt(const MbMlaPromptArgs* a, cudaStream_t stream) {
  if (a && (a->q_rows == 0 || a->kv_rows == 0 || a->max_q_len == 0 || a->max_ctx == 0)) {
    if (a->q_rows < 0 || a->kv_rows < 0 || a->max_q_len < 0 || a->max_ctx < 0 || a->num_seqs <= 0 || !a->q_start || !a->q_len || !a->ctx_len) return MB_ERR_BAD_ARG;
    const NothingParams n{a->q_start, a->q_len, a->ctx_len, a->status, a->q_rows, a->kv_rows, a->num_seqs, a->max_q_len, a->max_ctx};
    return (int)mb::launch_kernel(nothing_kernel, dim3(1), dim3(256), 0, stream, n);
  }
  if (!a || !a->q || !a->cache || !a->block_table || !a->q_start || !a->q_len || !a->ctx_len || !a->w || !a->out || a->num_blocks <= 0 || a->q_rows <= 0 ||
      a->kv_rows <= 0 || a->kv_rows % 128 || a->num_seqs <= 0 || a->num_seqs > 65535 || a->H <= 0 || a->H > 65535 || a->block_size <= 0 || a->max_q_len <= 0 ||
      a->max_ctx <= 0 || a->each <= 0)
    return MB_ERR_BAD_ARG;
  const unsigned tiles = ((unsigned)a->max_q_len + 255) / 256;
  if (tiles > 65535 || a->kv_rows >= (1ll << 31)) return MB_ERR_TOO_LARGE;
  const Layout l = layout(a->kv_rows, a->num_seqs, a->each);
  if (!a->ws || a->ws_bytes < l.bytes) return MB_ERR_TOO_LARGE;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a->ws);
  int *first = reinterpret_cast<int*>(ws + l.first), *bad = reinterpret_cast<int*>(ws + l.bad);
  const GatherParams g{(const __nv_bfloat16*)a->cache, a->block_table, a->table_ld, a->ctx_len, (__nv_bfloat16*)ws, first, bad, a->status, a->num_blocks, a->kv_rows,
                       a->num_seqs, a->block_size, a->max_ctx};
  cudaError_t e = mb::launch_kernel(gather_kernel, dim3((unsigned)(a->kv_rows / kGather)), dim3(256), 0, stream, g);
  if (e != cudaSuccess) return (int)e;
  static std::atomic<uint64_t> asked{0};
  e = mb::allow_smem(reinterpret_cast<const void*>(mla_prompt_kernel), kSmem, asked);
  if (e != cudaSuccess) return (int)e;
  static std::atomic<uint64_t> asked_too{0};
  e = mb::allow_smem(reinterpret_cast<const void*>(expand_kernel), kExpSmem, asked_too);
  if (e != cudaSuccess) return (int)e;
  const int pairs = a->sm_count > 1 ? a->sm_count / 2 : 74;
  CUtensorMap tm[5];
  int rc = mbh::encode_2d(&tm[0], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a->q, (uint64_t)a->H * kQk, a->q_rows, (uint64_t)a->H * kQk * 2, 64, 128);
  if (!rc) rc = mbh::encode_2d(&tm[3], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, ws, kRow, a->kv_rows, kRow * 2, 64, 128);
  for (int h = 0; h < a->H && !rc; h += a->each) {
    const int n = a->H - h < a->each ? a->H - h : a->each;
    const __nv_bfloat16* wh = reinterpret_cast<const __nv_bfloat16*>(a->w) + (size_t)h * 256 * kLat;
    void* kv = ws + l.kv;
    const long long units = (a->kv_rows + 255) / 256 * n;
    if (units > 0x7fffffff) return MB_ERR_TOO_LARGE;
    // 128 rows are half a unit, and mb_gemm has tiles of that size. The whole call replayed, here / by mb_gemm: 128 rows of 128 heads 21.8 / 20.8 us, of 64 18.0 / 18.2,
    // of 16 17.4 / 17.5; 256 rows of 128 heads 25.7 / 38.4, of 64 21.1 / 26.1, of 16 20.7 / 24.7. Among other calls: 384 rows of 128 59.9 / 65.7, 512 of 64 36.0 / 36.8,
    // 1024 of 16 34.9 / 36.9, of 64 59.6 / 70.3, 8192 of 16 294 / 306
    if (a->kv_rows > 128) {
      const ExpandParams x{(__nv_bfloat16*)kv, a->kv_rows, n, (int)units, a->status};
      rc = mbh::encode_2d(&tm[4], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, wh, kLat, (uint64_t)n * 256, kLat * 2, 64, 128);
      if (!rc) rc = (int)mb::launch_kernel_cluster(expand_kernel, dim3(2 * (unsigned)(units < pairs ? units : pairs)), dim3(kExpThreads), kExpSmem, stream, 1, tm[3], tm[4], x);
    } else {
      MbGemmArgs m{};
      m.M = (int)a->kv_rows; m.N = n * 256; m.K = kLat; m.ldo = n * 256; m.W = wh;
      m.X = ws; m.ldx = kRow; m.out = kv; m.alpha = 1.f; m.status = a->status; m.sm_count = a->sm_count;
      m.flags = a->gemm_flags;                             // without a workspace the product is not split
      rc = mb_gemm(&m, stream);
    }
    if (!rc) rc = mbh::encode_2d(&tm[1], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv, (uint64_t)n * 256, a->kv_rows, (uint64_t)n * 512, 64, 128);
    if (!rc) rc = mbh::encode_2d(&tm[2], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, kv, (uint64_t)n * 256, a->kv_rows, (uint64_t)n * 512, 64, 64);
    if (rc) return rc;
    const AttnParams p{a->q_start, a->q_len, a->ctx_len, first, bad, a->out, a->status, a->q_rows, a->kv_rows, a->H, h, a->max_q_len, a->max_ctx, a->scale};
    rc = (int)mb::launch_kernel_ex(mla_prompt_kernel, dim3(n, tiles, a->num_seqs), dim3(kThreads), kSmem, stream, 1, mb_pdl_enabled() != 0, tm[0], tm[1], tm[2], tm[3], p);
  }
  return rc;
}

}  // extern "C"
