// The weight that a prompt's last tokens give to what is cached: mass[s, h, j] += sum over observed rows r of p[r, j], p = softmax of the
// causal logits of the group's queries. K is read, V is not; the prompt's outputs are the prefill kernels' business.
//
// The normaliser of a row is known when all of its keys are done, so the logits are computed twice:
//   rows pass   128 query rows stay in shared memory, tiles of keys go by; a thread owns a row and keeps its maximum and sum
//   keys pass   128 keys stay, tiles of query rows go by; a thread owns a key and adds up 2^(z - normaliser of the row). Where there are few rows these
//               stay and blocks of keys go by
// They are the same kernel with the operands exchanged: what a thread owns is a lane of the accumulator in tensor memory, so that neither pass
// sums across lanes. Query rows of a kv head are numbered token * G + head of the group, as in attention_rows.cu.
//
// Both operands come by TMA: keys from the cache, 16 tokens a box, or from a copy in the workspace (an e4m3 cache's as f16, any cache's whose blocks are
// not whole boxes), which a kernel in front makes; query rows of the keys pass from the copy that the rows pass makes of its own (with an e4m3 cache
// f16, scaled by a power of two, one for 128 rows that are alike, else one per row). A first form had four warps gather and widen tiles on the way into
// shared memory, every CTA the same ones: that took the issue slots of the exponentials, 4096 observers at 8192 e4m3 tokens 819 us.
//
// Roles (384 threads, two CTAs per SM, so that one's beginning and end are under the other's exponentials): warps 0-3 and 4-7 own 128 lanes each and half
// of a tile's columns; warps 8 and 9 bring the rows' normalisers (keys pass), warp 10 issues the products into two accumulators, so that products run
// under the exponentials, warp 11 the copies. With 256 lanes a CTA and one of them per SM, 4096 observers at 8192 e4m3 tokens took 766 us, sixteen prompts
// of 17 to 1151 tokens under 64 observers 55.
//
// Bound by its exponentials, two a logit at 16 a cycle and SM: 4096 observers at 8192 e4m3 tokens, 40 / 8 heads of 128, take 729 us (1.0 G logits a
// pass, 2.8 T exponentials a second; the special function units 76 and 68 % busy, the tensor pipe 38 and 32), 32 observers 31, a launch's
// latency three times. At dim 256 products from shared memory count as much: 2 prompts of 1001 and 1531 at up to 4431 tokens, 16 / 2 heads, 163 us. (B200, in a graph.)
//
// Long rows and long columns are cut into parts, by rules on the sequence's own lengths alone, and joined in order: every output has one writer and
// every sum one order.
#include "attention_rows.cuh"
#include "common.cuh"
#include "kv_mass.h"
#include "smem_limit.h"
#include "tensormap.h"

namespace {

using namespace mbr;

constexpr int kThreads = 384, kSums = 256, kHeld = 128, kMaxKeyParts = 32, kMaxRowParts = 16, kInfo = 8, kBox = 16;
template <int N>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// observed rows of a sequence, and its cached tokens; what the call was not sized for is reported and cut
struct Span {
  int n, rows, tok0, past;     // cached tokens, observed rows (tokens x group), first observed token, tokens in front of the portion (may be negative)
};
__device__ __forceinline__ Span span_of(const MbMassArgs& a, int s, int G) {
  int n = a.ctx_len[s], ql = a.q_len[s];
  const long long start = a.q_start[s];
  bool bad = n > a.max_ctx || ql > a.max_q_len;
  n = max(min(n, a.max_ctx), 0);
  ql = max(min(ql, a.max_q_len), 0);
  if (ql > 0 && (start < 0 || start + ql > a.q_rows)) {
    bad = true;
    ql = 0;
  }
  if (bad && a.status && threadIdx.x == 0) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
  const int seen = min(a.last, ql);
  return {n, seen * G, (int)start + ql - seen, n - seen};
}

// Keys of a part of a row, rows of a part of a column: few rows want many parts to fill the chip, many rows do that by themselves. (512 or 1024 keys,
// 64 observers: sixteen prompts of 17 to 1151 tokens 48 / 44 us, one of 16000 35 / 40.)
__host__ __device__ __forceinline__ int key_part(int n, int rows) {
  const int least = rows <= 512 ? (n <= 2048 ? 1024 : 512) : rows <= 4096 ? 2048 : 8192, even = ((n + kMaxKeyParts - 1) / kMaxKeyParts + 127) & ~127;
  return even > least ? even : least;
}
__host__ __device__ __forceinline__ int row_part(int rows) {
  const int even = ((rows + kMaxRowParts - 1) / kMaxRowParts + 127) & ~127;
  return even > 4096 ? even : 4096;
}
__host__ __device__ __forceinline__ int parts_of(int n, int part) { return n <= part ? 1 : (n + part - 1) / part; }

// Workspace: the query rows as operands [seqs * Hkv * rows, D], and behind them room for a tile; the keys, where they are copied [seqs * tokens, Hkv, D];
// {maximum, sum} of every row and part of its keys, log2 domain [seqs * Hkv * rows, key parts]; with an e4m3 cache the power of two that a row's scores are
// too large by; sums of the columns' parts [row parts, seqs * Hkv, columns]
struct Ws {
  long long rows, cols, tokens;
  // slices: CTAs that a block of rows is shared out over; joined: a row's parts are, before the keys pass; few: tiles of rows that stay in a CTA of the
  // keys pass, where keys go by, `each` blocks of them, else 0
  int key_parts, row_parts, slices, paged, joined, few, each;
  size_t keys, ml, scale, sums, bytes;
};
// From this many observed rows on, a bf16 cache's keys are copied too: every tile of them goes by often, and comes as one box instead of eight
constexpr int kCopyRows = 1024;
// With more parts of a row than this they are joined by a kernel of its own: every CTA of the keys pass would join them again, for all rows. 64 observers at
// 16000 bf16 tokens, 16 / 2 heads of 256 (32 parts) 47 -> 35 us, three of 16207, 16 / 1 of 128 (16 parts, 1024 rows) 74 -> 67. CTAs with few rows are fewer and join more
// themselves: 8 prompts of 4000 to 8192 tokens, 128 rows (16 parts) 80 -> 71, one of 32768, 160 rows (32 parts) 65.5 -> 63.2 with the kernel.
constexpr int kJoin = 4, kFewJoin = 16;
// Up to so many tiles of 128 rows stay in a CTA of the keys pass while keys go by, two at 64 and 128 dims and one at 256, which shared memory holds beside a
// ring. With a CTA a block of keys, which brings them and their normalisers each time: 32 at 8192 e4m3 34 us instead of 31, 8 prompts of 4000 to 8192, 128
// rows 118 instead of 71, one of 32768, 160 rows 85 instead of 63. The sums and their order are the same.
constexpr int kFewCtas = 2 * 148;                          // as many as the chip holds at once (148: one of 32768 81 us, 592: 69)

// What a part of a row, a sum relative to 2^m, has of a sum relative to 2^top. A part that sees nothing has no maximum and a sum of zero. One whose scores are
// all NaN has no maximum either (fmaxf passes them by), but its sum is NaN, and so is the row's. (Asking the sum for zero took 4096 at 8192 from 729 to 747 us.)
__device__ __forceinline__ float share_of(float m, float l, float top) { return l * (m == -INFINITY ? 0.f : ex2(m - top)); }

inline Ws workspace(int seqs, int Hq, int Hkv, int D, int block_size, int seen, int max_ctx, bool fp8) {
  Ws w;
  auto even = [](size_t x) { return (x + 127) & ~size_t(127); };
  w.rows = (long long)seen * (Hq / Hkv);
  w.cols = (max_ctx + 3) & ~3ll;
  w.tokens = (max_ctx + 255) & ~255ll;
  w.paged = !fp8 && block_size % kBox == 0 && w.rows < kCopyRows;
  // more parts than any sequence of the call has: fewer rows than the most may mean more of them
  w.key_parts = parts_of(max_ctx, 512) < kMaxKeyParts ? parts_of(max_ctx, 512) : kMaxKeyParts;
  w.row_parts = parts_of((int)w.rows, row_part((int)w.rows));
  w.slices = parts_of(max_ctx, key_part(max_ctx, (int)w.rows));
  w.few = w.rows <= (D == 256 ? kHeld : 2 * kHeld) ? (int)((w.rows + kHeld - 1) / kHeld) : 0;
  w.joined = w.slices > (w.few ? kFewJoin : kJoin);
  const long long units = (long long)seqs * Hkv * ((max_ctx + kHeld - 1) / kHeld);
  w.each = (int)((units + kFewCtas - 1) / kFewCtas);
  const size_t n = (size_t)seqs * Hkv * w.rows;
  w.keys = even((n + 128) * D * 2);
  w.ml = w.keys + (w.paged ? 0 : even((size_t)seqs * w.tokens * Hkv * D * 2));
  w.scale = w.ml + even(n * w.key_parts * 8);
  w.sums = w.scale + (fp8 ? even(n * 4) : 0);
  w.bytes = w.sums + (w.row_parts > 1 ? (size_t)w.row_parts * seqs * Hkv * w.cols * 4 : 0);
  return w;
}

// Rows of an e4m3 cache as f16, of a bf16 cache as they are, one sequence behind the other: 16 values a thread.
template <bool FP8>
__global__ void __launch_bounds__(256) observe_copy_kernel(const MbMassArgs a, const Ws ws) {
  mb::pdl_launch_dependents();
  const int s = blockIdx.y, n = a.q_len[s] > 0 ? min(a.ctx_len[s], a.max_ctx) : 0, per = a.Hkv * a.D / 16;        // of a cached token
  const int* table = a.block_table + s * a.table_ld;
  uint4* out = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(a.ws) + ws.keys) + (size_t)s * ws.tokens * per * 2;
  // a CTA takes 8192 values at a time: whole tokens, or a part of one
  const int tokens = max(1, 512 / per), parts = (per + 511) / 512;
  for (int u = blockIdx.x; u < (n + tokens - 1) / tokens * parts; u += gridDim.x) {
    const int j0 = u / parts * tokens, c0 = u % parts * 512;
    for (int i = threadIdx.x; i < 512; i += 256) {
      const int j = j0 + i / per, c = c0 + i % per;                       // a token that takes more than 512 has i / per = 0
      if (j >= n || i / per >= tokens || c >= per) continue;
      const size_t at = (size_t)mbm::slot_of(table, j, a.block_size, a.num_blocks, a.status) * per + c, to = (size_t)j * per + c;
      if constexpr (FP8) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(a.k_cache) + at);
        out[2 * to] = make_uint4(e4m3x2(x.x), e4m3x2(x.x >> 16), e4m3x2(x.y), e4m3x2(x.y >> 16));
        out[2 * to + 1] = make_uint4(e4m3x2(x.z), e4m3x2(x.z >> 16), e4m3x2(x.w), e4m3x2(x.w >> 16));
      } else {
        out[2 * to] = __ldg(reinterpret_cast<const uint4*>(a.k_cache) + 2 * at);
        out[2 * to + 1] = __ldg(reinterpret_cast<const uint4*>(a.k_cache) + 2 * at + 1);
      }
    }
  }
}

template <int D>
struct Cfg {
  static constexpr int kN = 128;                             // rows of a tile that goes by
  // A tile comes in chunks of 64 dims, a swizzled span of 128 bytes each, which go round a ring of stages. (Tiles of 64 rows would take the products as
  // long as tiles of 128: they are bound by reading the 128 held rows from shared memory.)
  static constexpr int kDims = 64, kChunks = D / kDims;
  static constexpr int kStages = D == 256 ? 2 : 4;
  static constexpr int kHeldB = kHeld * D * 2, kChunkB = kN * kDims * 2;
  static constexpr int kSmem = kHeldB + kStages * kChunkB + 1024;
  static constexpr uint32_t kCols = 2 * kN;                  // two accumulators
};

// stages of a ring beside few rows' tiles that stay; two tiles go over a block of keys twice, which the ring then holds whole
__host__ __device__ constexpr int few_stages(int D, int tiles) { return D == 256 || (D == 128 && tiles == 2) ? 2 : 4; }
template <int D>
constexpr int few_smem(int tiles) { return tiles * Cfg<D>::kHeldB + few_stages(D, tiles) * Cfg<D>::kChunkB + 1024; }

enum Pass { kRowsPass, kKeysPass, kFewPass };

template <int D, bool FP8, Pass PASS>
__global__ void __launch_bounds__(kThreads, 2)
observe_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmQ, const MbMassArgs a, const Ws ws, int g_magic) {
  using C = Cfg<D>;
  constexpr bool KEYS = PASS != kRowsPass, FEW = PASS == kFewPass;        // a thread owns a key; and these go by
  constexpr int kN = C::kN, kMost = FEW ? 4 : C::kStages, kChunks = C::kChunks;
  const int kStages = FEW ? few_stages(D, ws.few) : C::kStages;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* sHeld = smem_raw + ((1024u - (mb::smem_u32(smem_raw) & 1023u)) & 1023u);   // D / 64 spans x [128 rows x 128 B]
  uint8_t* sRing = sHeld + (FEW ? ws.few : 1) * C::kHeldB;                        // kStages x [kN rows x 128 B]
  __shared__ __align__(8) uint64_t held_full, full[kMost], empty[kMost], info_full[kInfo], info_free[kInfo], s_full[2], s_free[2];
  __shared__ uint32_t s_tmem;
  __shared__ int s_row[kHeld];                                 // rows pass, e4m3: the exponent of a row's largest element
  __shared__ float2 s_half[FEW ? 2 : 1][kHeld];                           // sums of the second half of the columns
  __shared__ __align__(16) float s_lse[kInfo][kN];           // keys pass: the query rows' normalisers, negative, and their factors
  __shared__ __align__(16) float s_factor[KEYS && FP8 ? kInfo : 1][kN];
  __shared__ __align__(8) int s_alike[KEYS && FP8 ? kInfo : 1][4];         // 32 rows' factors are those of the first of 64
  __shared__ int s_nan;                                      // keys pass: the last row whose normaliser is not a number
  __shared__ int2 s_top[kSums / 32];                         // rows pass, e4m3: the largest exponent of a row's largest element, and the smallest
  const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.Hq / a.Hkv;
  const Span x = span_of(a, s, G);
  const int kp = key_part(x.n, x.rows), kparts = parts_of(x.n, kp), rp = row_part(x.rows), rparts = parts_of(x.rows, rp);
  auto tok_of = [&](int r) { return G == 1 ? r : (int)__umulhi((unsigned)r, (unsigned)g_magic); };
  auto limit_of = [&](int r) { return x.past + tok_of(r) + 1; };       // keys in front of this one are visible to row r
  // ---- what stays, and the range of what goes by
  // A column's parts are a CTA each. So are a row's where the call's longest portion has as many; shorter portions, whose rows have more of them, share
  // `slices` CTAs out.
  const int slices = KEYS ? ws.row_parts : ws.slices, blocks = gridDim.x / slices, share = KEYS ? 1 : (kparts + slices - 1) / slices;
  const int part = FEW ? 0 : blockIdx.x / blocks * share;
  const int at0 = (FEW ? (int)blockIdx.x * ws.each : KEYS ? (int)blockIdx.x % blocks : blocks - 1 - (int)blockIdx.x % blocks) * kHeld;   // the longest first
  const int own = KEYS ? x.n : x.rows;
  if (part >= (KEYS ? rparts : kparts) || at0 >= own || x.rows == 0 || x.n == 0) {
    mb::pdl_wait();                                       // a grid ends behind the one in front of it, even where it does nothing
    return;
  }
  int begin, end;
  if constexpr (FEW) {
    begin = 0;
    end = x.rows;
  } else if constexpr (KEYS) {
    // the first row that sees the first of these keys
    const int first = max(0, at0 - x.past) * G;
    begin = max(part * rp, first & ~(kN - 1));
    end = min(x.rows, (part + 1) * rp);
  } else {
    begin = part * kp;
    end = min(min(x.n, begin + share * kp), limit_of(min(x.rows, at0 + kHeld) - 1));
  }
  // few rows: their tiles one after the other for each block of keys
  const int turns = FEW ? (x.rows + kN - 1) / kN : 1, more = turns - 1;
  const int tiles = FEW ? min(ws.each, (own - at0 + kHeld - 1) / kHeld) * turns : end > begin ? (end - begin + kN - 1) / kN : 0;
  const size_t row0 = ((size_t)s * a.Hkv + h) * ws.rows;     // of the workspace's rows
  float2* ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(a.ws) + ws.ml) + row0 * ws.key_parts;
  uint4* wq = reinterpret_cast<uint4*>(a.ws) + row0 * (D / 8);
  float* wscale = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.ws) + ws.scale) + row0;

  // ---- rows pass: the query rows, which stay: 128 of them, rows behind the last one are zeros. They are asked for while the barriers are made.
  constexpr int kPieces = D / 8, kStep = kSums / kPieces, kLoads = kHeld / kStep, kBatch = kLoads < 8 ? kLoads : 8;
  const int c = tid % kPieces, hr0 = tid / kPieces;
  uint4 v[kBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int hr = hr0 + kStep * (i0 + i), at = min(at0 + hr, own - 1), tq = tok_of(at);
      v[i] = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(a.q) + ((size_t)(x.tok0 + tq) * a.Hq + h * G + (at - tq * G)) * D) + c);
      if (at0 + hr >= own) v[i] = make_uint4(0, 0, 0, 0);
    }
  };
  if (!KEYS && warp < 8) {
    int hi = 0, lo = 255;
#pragma unroll 1
    for (int i0 = 0; i0 < (FP8 ? kLoads : kBatch); i0 += kBatch) {
      load(i0);
      if constexpr (FP8) {
        // the exponent of a row's largest element; bits of a bf16 without its sign order like the values
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          uint32_t top = __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu), __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu));
#pragma unroll
          for (int d = 1; d < kPieces; d <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
          const int e = (int)(max(top & 0xffff, top >> 16) >> 7);
          if (c == 0) s_row[hr0 + kStep * (i0 + i)] = e;
          hi = max(hi, e);
          if (e > 0) lo = min(lo, e);
        }
      }
    }
    if constexpr (FP8) {
      hi = __reduce_max_sync(0xffffffffu, hi);
      lo = __reduce_min_sync(0xffffffffu, lo);
      if (lane == 0) s_top[warp] = make_int2(hi, lo);
    }
  }
  if (tid == kThreads - 1) {
    mb::mbar_init(&held_full, KEYS ? 1 : kSums / 32);
    for (int i = 0; i < kMost; ++i) {
      mb::mbar_init(&full[i], 1);
      mb::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < kInfo; ++i) {
      mb::mbar_init(&info_full[i], 2);
      mb::mbar_init(&info_free[i], kSums / 32);
    }
    for (int i = 0; i < 2; ++i) {
      mb::mbar_init(&s_full[i], 1);
      mb::mbar_init(&s_free[i], kSums / 32);
    }
    s_nan = -1;
    mb::mbar_fence_init();
    mb::tma_prefetch_desc(&tmK);
    if (KEYS) mb::tma_prefetch_desc(&tmQ);
  }
  if (warp == 10) mb::tmem_alloc(&s_tmem, C::kCols);
  mb::tc_fence_before();
  __syncthreads();
  mb::tc_fence_after();
  const uint32_t tmem = s_tmem;
  // A dependent kernel allocates TMEM: not before this CTA has its own. What the kernel in front writes, only some warps read, and these wait for it: the
  // copies of keys and query rows, the normalisers.
  mb::pdl_launch_dependents();
  // of a row's scores, in the log2 domain; never 0, which would make numbers of the -inf that a mask leaves. A cache's scale that is negative or NaN is none, and
  // leaves no numbers.
  auto factor = [&](float row) {
    const float f = a.scale * (FP8 ? *a.k_scale : 1.f) * 1.44269504088896f * row;
    return !FP8 || f >= 0.f ? fmaxf(f, 1.17549435e-38f) : NAN;
  };

  if (warp < 8) {
    more_regs<88>();
    const int half = warp >> 2, r = tid & 127;
    int mine = at0 + r;
    constexpr int kCols = kN / 2, kW = 32;                   // columns of a thread, and of a round
    float row_scale = 1.f;                                   // what this thread's row's scores are too large by
    if constexpr (!KEYS) {
      // f16 has less range than bf16: the power of two that takes a row's largest element to [2^14, 2^15). Zeros and subnormal rows as if their
      // exponent were 15, infinities and NaN as they are.
      auto lift = [](int e) { return e == 255 ? 0 : 141 - max(e, 15); };
      int up = 0;
      bool alike = true;
      if constexpr (FP8) {
        // Rows whose largest elements are within 2^12 of each other take the power of the largest, so that their scores have one factor: the smallest then
        // still keeps 8 bits of elements down to 2^-19 of its largest, and the rest to 2^-27 of it.
        int hi = 0, lo = 255;
#pragma unroll
        for (int i = 0; i < kSums / 32; ++i) {
          hi = max(hi, s_top[i].x);
          lo = min(lo, s_top[i].y);
        }
        alike = hi < 255 && hi - lo <= 12;
        up = lift(hi);
      }
      // The first part's CTA leaves the rows for the keys pass.
#pragma unroll 1
      for (int i0 = 0; i0 < kLoads; i0 += kBatch) {
        if (kLoads > kBatch && (FP8 || i0 > 0)) load(i0);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const int hr = hr0 + kStep * (i0 + i);
          if constexpr (FP8) {
            const int mine_up = alike ? up : lift(s_row[hr]);
            const float f = __int_as_float((127 + mine_up) << 23);
            const uint32_t y[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
            uint32_t z[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 p = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&y[j]));
              z[j] = pack2<true>(p.x * f, p.y * f);
            }
            v[i] = make_uint4(z[0], z[1], z[2], z[3]);
            if (c == 0 && part == 0 && at0 + hr < own) wscale[at0 + hr] = __int_as_float((127 - mine_up) << 23);
          }
          if (part == 0 && at0 + hr < own) wq[(size_t)(at0 + hr) * kPieces + c] = v[i];
          *reinterpret_cast<uint4*>(sHeld + (c >> 3) * (kHeld * 128) + sw_off(hr, c & 7)) = v[i];
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mb::mbar_arrive(&held_full);
      if constexpr (FP8) row_scale = __int_as_float((127 - (alike ? up : lift(s_row[r]))) << 23);
    }
    const float sc = factor(row_scale);
    const int limit = KEYS ? 0 : mine < own ? limit_of(mine) : 0;
    const uint32_t tS = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * kCols;
    float m_run = -INFINITY, l_run = 0.f;                    // keys pass: l_run is the column's sum
    bool ok = true;
    // rows pass: a part of a row's keys is done; the halves of the columns are joined
    int mine_part = part, flush_at = (part + 1) * kp;
    auto flush = [&] {
      if (half) s_half[0][r] = make_float2(m_run, l_run);
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (!half && mine < own) {
        const float2 y = s_half[0][r];
        const float top = fmaxf(m_run, y.x);
        const float l = share_of(m_run, l_run, top) + share_of(y.x, y.y, top);
        ml[(size_t)mine * ws.key_parts + mine_part] = make_float2(top, l);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      m_run = -INFINITY;
      l_run = 0.f;
      ++mine_part;
      flush_at += kp;
    };
    // Columns that count for any lane of this warp end here; the others' weights are zeros, whose exponentials few rows would pay for (160 rows of 5 heads: a
    // block of 128 and one of 32; 32 observers at 8192 e4m3 tokens 41 -> 34 us, at the price of 716 -> 723 for 4096).
    int reach = KEYS ? (at0 + (warp & 3) * 32 < own ? end : 0) : min(end, __reduce_max_sync(0xffffffffu, limit));
    float old = 0.f;                                         // few rows: the mass that is added to
    int blocks_left = FEW ? tiles / turns : 0;
    for (int t = 0; t < tiles; ++t) {
      const int at_row = FEW ? (t & more) * kN : begin + t * kN, slot = FEW ? t & more : t % kInfo;
      const int b = t & 1, used = min(reach - (at_row + half * kCols), kCols);
      if (FEW && (t & more) == 0 && !half && mine < own) old = a.mass[s * a.mass_seq + h * a.mass_head + mine];
      ok = mb::mbar_wait(&s_full[b], (t >> 1) & 1, a.status, MB_ST_TIMEOUT_MMA);
      if (KEYS) ok = ok && mb::mbar_wait(&info_full[slot], FEW ? 0 : (t / kInfo) & 1, a.status, MB_ST_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      mb::tc_fence_after();
      auto taken = [&](uint64_t* bar) {
        __syncwarp();
        if (lane == 0) mb::mbar_arrive(bar);
      };
      if (used <= 0) {
        mb::tc_fence_before();
        taken(&s_free[b]);
        if (KEYS && !FEW) taken(&info_free[slot]);
      }
      // 32 columns at a time: the code of a tile is half as long, which a short call waits for from L2
#pragma unroll 1
      for (int c0 = 0; c0 < used; c0 += kW) {
        float z[kW];
        mb::tmem_ld32_async(tS + b * kN + c0, z);
        mb::tmem_ld_wait(z);
        if (c0 + kW >= used) {
          mb::tc_fence_before();
          taken(&s_free[b]);                                // the accumulator is in registers
        }
        const int from = at_row + half * kCols + c0;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if constexpr (KEYS) {
          // these rows' first one sees the least: all of these keys, or a row each is asked. Behind the last row is whatever memory holds.
          if (__any_sync(0xffffffffu, mine >= limit_of(from) || from + kW > end)) {
#pragma unroll
            for (int i = 0; i < kW; ++i)
              if (mine >= limit_of(from + i) || from + i >= end) z[i] = -INFINITY;
          }
          const float4* lse = reinterpret_cast<const float4*>(&s_lse[slot][half * kCols + c0]);
          auto add = [&](auto factors) {
#pragma unroll
            for (int i = 0; i < kW / 4; ++i) {
              const float4 n4 = lse[i], f4 = factors(i);
              float2 p = fma2(make_float2(z[4 * i], z[4 * i + 1]), make_float2(f4.x, f4.y), make_float2(n4.x, n4.y));
              float2 q = fma2(make_float2(z[4 * i + 2], z[4 * i + 3]), make_float2(f4.z, f4.w), make_float2(n4.z, n4.w));
              p.x = ex2(p.x);
              p.y = ex2(p.y);
              q.x = ex2(q.x);
              q.y = ex2(q.y);
              sum[0] = add2(sum[0], p);
              sum[1] = add2(sum[1], q);
            }
          };
          if constexpr (FP8) {
            const float4* own4 = reinterpret_cast<const float4*>(&s_factor[slot][half * kCols + c0]);
            const int2 alike = *reinterpret_cast<const int2*>(&s_alike[slot][half * 2]);
            if (alike.x && alike.y) {
              const float f = own4->x;
              const float4 same = make_float4(f, f, f, f);
              add([&](int) { return same; });
            } else {
              add([&](int i) { return own4[i]; });
            }
          } else {
            const float4 same = make_float4(sc, sc, sc, sc);
            add([&](int) { return same; });
          }
          l_run += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          if (!FEW && c0 + kW >= used) taken(&info_free[slot]);
        } else {
          const int seen = min(limit, end) - from;             // columns in front of this one are visible
          if (!__all_sync(0xffffffffu, seen >= kW)) {
#pragma unroll
            for (int i = 0; i < kW; ++i)
              if (i >= seen) z[i] = -INFINITY;
          }
          const float2 sc2 = make_float2(sc, sc);
          auto add = [&] {
            const float nm = m_run == -INFINITY ? 0.f : -m_run;
            const float2 nm2 = make_float2(nm, nm);
            sum[0] = sum[1] = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kW / 2; ++i) {
              float2 p = fma2(make_float2(z[2 * i], z[2 * i + 1]), sc2, nm2);
              p.x = ex2(p.x);
              p.y = ex2(p.y);
              sum[i & 1] = add2(sum[i & 1], p);
            }
            return (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
          };
          // What a row is relative to need not be its maximum, as long as nothing overflows and something of it is near 1: the largest of its first tile
          // with a visible column stands until a tile's sum passes 2^60.
          float tile;
          for (int again = 0;; again = 1) {
            tile = add();
            const bool move = m_run == -INFINITY || !(tile < 0x1p60f);
            if (again || !__any_sync(0xffffffffu, move)) break;
            float mx4[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
            for (int i = 4; i < kW; ++i) mx4[i & 3] = fmaxf(mx4[i & 3], z[i]);
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
            if (move && mx > m_run) {
              l_run *= ex2(m_run - mx);
              m_run = mx;
            }
          }
          l_run += tile;
        }
      }
      if (!KEYS && begin + (t + 1) * kN == flush_at) flush();
      if (FEW && (t & more) == more) {
        // a block of keys is done; the other half's sums have two places, so that one barrier a block is enough
        const int place = (t / turns) & 1;
        if (s_nan >= 0 && mine < limit_of(s_nan)) l_run = NAN;
        if (half) s_half[place][r].y = l_run;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (!half && mine < own) a.mass[s * a.mass_seq + h * a.mass_head + mine] = old + (l_run + s_half[place][r].y);
        --blocks_left;
        l_run = 0.f;
        mine += kHeld;
        reach = mine - lane < own ? end : 0;
      }
    }
    for (; blocks_left > 0; --blocks_left) asm volatile("bar.sync 1, 256;" ::: "memory");    // a wait ran out: the other warps' barriers count this one
    if constexpr (KEYS && !FEW) {
      if (s_nan >= 0 && mine < limit_of(s_nan)) l_run = NAN;
      if (half) s_half[0][r].y = l_run;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (!half && mine < own) {
        l_run += s_half[0][r].y;
        if (ws.row_parts > 1)
          reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.ws) + ws.sums)[((size_t)part * a.num_seqs * a.Hkv + (size_t)s * a.Hkv + h) * ws.cols + mine] = l_run;
        else
          a.mass[s * a.mass_seq + h * a.mass_head + mine] += l_run;
      }
    } else if constexpr (!KEYS) {
      while (mine_part < min(part + share, kparts)) flush();   // parts behind what these rows see are empty
    }
    mb::tc_fence_before();
  } else {
    fewer_regs<64>();
    if (KEYS && warp < 10) {
      // ---------------------------------------------------------- factors and normalisers of a tile's rows, two a thread
      const int t = tid - kSums, left = ws.joined ? 1 : kparts;
      mb::pdl_wait();
      // the parts of the next tile's normalisers are on their way while this one's are joined
      constexpr int kTake = FEW ? 8 : 4;
      float2 y[2][kTake];
      float yscale[2] = {1.f, 1.f};
      auto look = [&](int tile) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = min(begin + tile * kN + t + 64 * e, end - 1);
#pragma unroll
          for (int k = 0; k < kTake; ++k) y[e][k] = k < left ? ml[(size_t)at * ws.key_parts + k] : make_float2(-INFINITY, 0.f);
          if (FP8) yscale[e] = wscale[at];
        }
      };
      const int infos = FEW ? turns : tiles;
      if (infos > 0) look(0);
      for (int tile = 0; tile < infos; ++tile) {
        const int slot = tile % kInfo;
        float f[2], lse[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int at = begin + tile * kN + t + 64 * e;
          float m = -INFINITY, l = 0.f;
          for (int i = 0; i < left; i += kTake) {
            if (i > 0) {
#pragma unroll
              for (int k = 0; k < kTake; ++k) y[e][k] = i + k < left ? ml[(size_t)min(at, end - 1) * ws.key_parts + i + k] : make_float2(-INFINITY, 0.f);
            }
#pragma unroll
            for (int k = 0; k < kTake; ++k) {
              const float top = fmaxf(m, y[e][k].x);
              l = share_of(m, l, top) + share_of(y[e][k].x, y[e][k].y, top);
              m = top;
            }
          }
          f[e] = factor(yscale[e]);
          lse[e] = at < end && l != 0.f ? m + log2f(l) : INFINITY;       // rows behind the last one and rows without weight add nothing
          // An infinite query's is NaN, which the -inf of a mask would not survive. Its row adds nothing here; since later rows see more, the last such row
          // says which keys have no number in the end.
          if (lse[e] != lse[e]) {
            atomicMax(&s_nan, at);
            lse[e] = INFINITY;
          }
        }
        const bool ok = mb::mbar_wait(&info_free[slot], ((tile / kInfo) & 1) ^ 1, a.status, MB_ST_TIMEOUT_EPI);
        if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          s_lse[slot][t + 64 * e] = -lse[e];
          if constexpr (FP8) s_factor[slot][t + 64 * e] = f[e];
        }
        if constexpr (FP8) {
          asm volatile("bar.sync 2, 64;" ::: "memory");
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool alike = __all_sync(0xffffffffu, f[e] == s_factor[slot][64 * e]);
            if (lane == 0) s_alike[slot][2 * e + (warp & 1)] = alike;
          }
        }
        __syncwarp();
        if (lane == 0) mb::mbar_arrive(&info_full[slot]);
        if (tile + 1 < infos) look(tile + 1);
      }
    }
    if (warp == 10 && mb::elect_one()) {
      // ---------------------------------------------------------- products
      constexpr uint32_t kF = FP8 ? 0 : 1, kId = mb::umma_idesc(kF, kF, 128, kN);
      // an address is the low bits of a descriptor, in units of 16 bytes
      const uint64_t dH = mb::umma_desc_sw128(mb::smem_u32(sHeld)), dR = mb::umma_desc_sw128(mb::smem_u32(sRing));
      bool ok = mb::mbar_wait(&held_full, 0, a.status, MB_ST_TIMEOUT_MMA);
      const int chunks = tiles * kChunks;
      int st = 0, turn = 0;
      for (int j = 0; j < chunks && ok; ++j) {
        const int tile = j / kChunks, q = j % kChunks, b = tile & 1, row_tile = FEW ? tile & more : 0;
        if (FEW && q == 0 && row_tile > 0) {                 // the same chunks again, all of which are in the ring
          st -= kChunks;
          if (st < 0) {
            st += kStages;
            turn ^= 1;
          }
        }
        ok = mb::mbar_wait(&full[st], turn, a.status, MB_ST_TIMEOUT_MMA);
        if (q == 0) ok = ok && mb::mbar_wait(&s_free[b], ((tile >> 1) & 1) ^ 1, a.status, MB_ST_TIMEOUT_MMA);
        if (!ok) break;
        mb::tc_fence_after();
        const uint64_t dC = dR + (uint32_t)(st * (C::kChunkB >> 4)), dA = dH + (uint32_t)((row_tile * kChunks + q) * (kHeld * 128 >> 4));
#pragma unroll
        for (int k = 0; k < 4; ++k) mb::umma_f16(tmem + b * kN, (FEW ? dC : dA) + (k * 32 >> 4), (FEW ? dA : dC) + (k * 32 >> 4), kId, (q | k) != 0);
        if (q == kChunks - 1) mb::tc_commit(&s_full[b]);
        if (row_tile == more) mb::tc_commit(&empty[st]);
        if (++st == kStages) {
          st = 0;
          turn ^= 1;
        }
      }
      // nobody may free the accumulators under products in flight
      const int last = chunks / turns - 1;                   // of the chunks that came
      if (ok && last >= 0) mb::mbar_wait(&empty[last % kStages], (last / kStages) & 1, a.status, MB_ST_TIMEOUT_MMA);
    }
    if (warp == 11) {
      // ---------------------------------------------------------- copies
      const int* table = a.block_table + s * a.table_ld;
      int bad = 0;
      // where the box of 16 tokens from key j on begins; a box behind the context reads the null block, a block that the cache does not have block 0
      auto box_at = [&](int j) {
        if (j >= x.n) return 0;
        const int bi = j / a.block_size, b = __ldg(table + bi);
        const bool out = (unsigned)b >= (unsigned)a.num_blocks;
        bad |= out;
        return (out ? 0 : b) * a.block_size + (j - bi * a.block_size);
      };
      // 64 dims of 128 keys from `from` on; lane l < 8 holds the places of their boxes
      auto keys = [&](uint8_t* dst, uint64_t* bar, int dim, int from, int place) {
        if (ws.paged) {
          if (lane < kN / kBox) mb::tma_load_3d(dst + lane * (kBox * 128), &tmK, bar, dim, h, place);
        } else if (lane == 0) {
          mb::tma_load_3d(dst, &tmK, bar, dim, h, (int)(s * ws.tokens) + from);
        }
      };
      if (!KEYS || !ws.paged) mb::pdl_wait();
      // few rows stay, once the kernel in front has left them
      auto hold = [&] {
        if (ws.paged) mb::pdl_wait();
        if (lane == 0) {
          mb::mbar_expect_tx(&held_full, turns * C::kHeldB);
          for (int i = 0; i < turns * kChunks; ++i) mb::tma_load_2d(sHeld + i * (kHeld * 128), &tmQ, &held_full, i % kChunks * 64, (int)row0 + i / kChunks * kN);
        }
        __syncwarp();
      };
      if constexpr (KEYS && !FEW) {
        if (lane == 0) mb::mbar_expect_tx(&held_full, C::kHeldB);
        __syncwarp();
        const int place = ws.paged ? box_at(at0 + (lane & 7) * kBox) : 0;
        for (int q = 0; q < kChunks; ++q) keys(sHeld + q * (kHeld * 128), &held_full, q * 64, at0, place);
      }
      if (KEYS && !FEW && ws.paged) mb::pdl_wait();
      const int chunks = tiles / turns * kChunks, key0 = FEW ? at0 : begin;
      int st = 0, turn = 1, place = 0;
      if ((!KEYS || FEW) && ws.paged && chunks > 0) place = box_at(key0 + (lane & 7) * kBox);
      for (int j = 0; j < chunks; ++j) {
        const int tile = j / kChunks, q = j % kChunks, from = key0 + tile * kN;
        if (FEW && j == min(kStages, chunks) - 1) hold();    // keys of the cache need not wait for it
        if (!__all_sync(0xffffffffu, mb::mbar_wait(&empty[st], turn, a.status, MB_ST_TIMEOUT_TMA))) break;
        if (lane == 0) mb::mbar_expect_tx(&full[st], C::kChunkB);
        __syncwarp();
        uint8_t* dst = sRing + st * C::kChunkB;
        if constexpr (KEYS && !FEW) {
          if (lane == 0) mb::tma_load_2d(dst, &tmQ, &full[st], q * 64, (int)row0 + from);
        } else {
          keys(dst, &full[st], q * 64, from, place);
          if (ws.paged && q == kChunks - 1) place = box_at(from + kN + (lane & 7) * kBox);
        }
        if (++st == kStages) {
          st = 0;
          turn ^= 1;
        }
      }
      if (bad && a.status) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
      // copies in flight write shared memory: the CTA stays until the products have taken the last of them
      if (KEYS && !FEW && tiles == 0) mb::mbar_wait(&held_full, 0, a.status, MB_ST_TIMEOUT_TMA);
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 10) {
    mb::tc_fence_after();
    mb::tmem_dealloc(tmem, C::kCols);
  }
}

// Rows whose keys were cut into parts: {maximum, sum} over them in order, in the place of the first.
__device__ __forceinline__ float2 joined(const float2* p, int parts) {
  float m = -INFINITY, l = 0.f;
  for (int i = 0; i < parts; i += 8) {                       // eight parts' loads in flight
    float2 y[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = i + k < parts ? p[i + k] : make_float2(-INFINITY, 0.f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float top = fmaxf(m, y[k].x);
      l = share_of(m, l, top) + share_of(y[k].x, y[k].y, top);
      m = top;
    }
  }
  return make_float2(m, l);
}
__global__ void __launch_bounds__(128) observe_rows_join_kernel(const MbMassArgs a, const Ws ws) {
  mb::pdl_launch_dependents();
  const int h = blockIdx.y, s = blockIdx.z, row = blockIdx.x * 128 + threadIdx.x;
  const Span x = span_of(a, s, a.Hq / a.Hkv);
  mb::pdl_wait();
  if (row >= x.rows) return;
  float2* ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(a.ws) + ws.ml) + (((size_t)s * a.Hkv + h) * ws.rows + row) * ws.key_parts;
  *ml = joined(ml, parts_of(x.n, key_part(x.n, x.rows)));
}

// Columns whose rows were cut into parts: their sums in order.
__global__ void __launch_bounds__(256) observe_join_kernel(const MbMassArgs a, const Ws ws) {
  const int h = blockIdx.y, s = blockIdx.z, j = blockIdx.x * 256 + threadIdx.x;
  mb::pdl_wait();
  const Span x = span_of(a, s, a.Hq / a.Hkv);
  if (j >= x.n || x.rows == 0) return;
  const int parts = parts_of(x.rows, row_part(x.rows));
  const float* sums = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(a.ws) + ws.sums) + ((size_t)s * a.Hkv + h) * ws.cols + j;
  float sum = 0.f;
  for (int p = 0; p < parts; ++p) sum += sums[(size_t)p * a.num_seqs * a.Hkv * ws.cols];
  a.mass[s * a.mass_seq + h * a.mass_head + j] += sum;
}

template <int D, bool FP8, Pass PASS>
int launch(const MbMassArgs& a, const Ws& ws, const CUtensorMap* tm, cudaStream_t stream) {
  constexpr bool KEYS = PASS != kRowsPass;
  auto kern = observe_kernel<D, FP8, PASS>;
  const int smem = PASS == kFewPass ? few_smem<D>(ws.few) : Cfg<D>::kSmem;
  static std::atomic<uint64_t> asked{0};
  const cudaError_t e = mb::allow_smem(reinterpret_cast<const void*>(kern), PASS == kFewPass ? few_smem<D>(D == 256 ? 1 : 2) : Cfg<D>::kSmem, asked);
  if (e != cudaSuccess) return (int)e;
  const int G = a.Hq / a.Hkv;
  const unsigned magic = G == 1 ? 0 : (unsigned)(((1ull << 32) + G - 1) / G);
  const long long blocks = PASS == kFewPass ? ((a.max_ctx + kHeld - 1) / kHeld + ws.each - 1) / ws.each : ((KEYS ? (long long)a.max_ctx : ws.rows) + kHeld - 1) / kHeld * (KEYS ? ws.row_parts : ws.slices);
  if (blocks > 0x7fffffffll) return MB_ERR_TOO_LARGE;
  return (int)mb::launch_kernel_ex(kern, dim3((unsigned)blocks, a.Hkv, a.num_seqs), dim3(kThreads), smem, stream, 1, mb_pdl_enabled() && (KEYS || !ws.paged), tm[0], tm[1], a, ws,
                                   (int)magic);
}

template <int D, bool FP8>
int all(const MbMassArgs& a, const Ws& ws, cudaStream_t stream) {
  uint8_t* p = reinterpret_cast<uint8_t*>(a.ws);
  CUtensorMap tm[2];
  const long long slots = ws.paged ? a.num_blocks * a.block_size : a.num_seqs * ws.tokens, rows = (long long)a.num_seqs * a.Hkv * ws.rows + 128;
  if (slots >= (1ll << 31) || rows >= (1ll << 31)) return MB_ERR_TOO_LARGE;
  int rc = mbh::encode_3d(&tm[0], CU_TENSOR_MAP_DATA_TYPE_UINT16, ws.paged ? a.k_cache : p + ws.keys, D, a.Hkv, slots, D * 2, (uint64_t)a.Hkv * D * 2, 64, 1,
                          ws.paged ? kBox : Cfg<D>::kN);
  if (rc) return rc;
  rc = mbh::encode_2d(&tm[1], CU_TENSOR_MAP_DATA_TYPE_UINT16, p, D, rows, D * 2, 64, Cfg<D>::kN);
  if (rc) return rc;
  if (!ws.paged) {
    const long long work = (long long)a.max_ctx * a.Hkv * D / 8192 + 1;
    observe_copy_kernel<FP8><<<dim3((unsigned)(work < 4096 ? work : 4096), a.num_seqs), 256, 0, stream>>>(a, ws);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
  }
  rc = launch<D, FP8, kRowsPass>(a, ws, tm, stream);
  if (!rc && ws.joined)
    rc = (int)mb::launch_kernel_ex(observe_rows_join_kernel, dim3((unsigned)((ws.rows + 127) / 128), a.Hkv, a.num_seqs), dim3(128), 0, stream, 1, mb_pdl_enabled() != 0,
                                   a, ws);
  return rc ? rc : ws.few ? launch<D, FP8, kFewPass>(a, ws, tm, stream) : launch<D, FP8, kKeysPass>(a, ws, tm, stream);
}

}  // namespace

extern "C" {

size_t mb_prompt_mass_ws(int num_seqs, int Hq, int Hkv, int D, int block_size, int seen, int max_ctx, int fp8) {
  return workspace(num_seqs, Hq, Hkv, D, block_size, seen, max_ctx, fp8 != 0).bytes;
}

int mb_prompt_mass(const MbMassArgs* a, cudaStream_t stream) {
  if (!a || a->num_seqs <= 0 || a->num_seqs > 65535 || a->Hkv <= 0 || a->Hkv > 65535 || a->Hq % a->Hkv || (a->D != 64 && a->D != 128 && a->D != 256) ||
      a->block_size <= 0 || a->num_blocks <= 0 || a->max_ctx <= 0 || a->last <= 0 || a->last > a->max_q_len || !a->q || !a->k_cache || !a->block_table ||
      !a->q_start || !a->q_len || !a->ctx_len || !a->mass || (a->fp8 && !a->k_scale))
    return MB_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->ws)) & 15) return MB_ERR_UNSUPPORTED;
  if (a->num_blocks * a->block_size >= (1ll << 31)) return MB_ERR_TOO_LARGE;
  if ((long long)a->last * (a->Hq / a->Hkv) > (1ll << 25)) return MB_ERR_TOO_LARGE;     // rows that tok_of divides exactly
  const Ws ws = workspace(a->num_seqs, a->Hq, a->Hkv, a->D, a->block_size, a->last, a->max_ctx, a->fp8 != 0);
  if (!a->ws || a->ws_bytes < ws.bytes) return MB_ERR_TOO_LARGE;
  int rc;
  if (a->D == 64) rc = a->fp8 ? all<64, true>(*a, ws, stream) : all<64, false>(*a, ws, stream);
  else if (a->D == 128) rc = a->fp8 ? all<128, true>(*a, ws, stream) : all<128, false>(*a, ws, stream);
  else rc = a->fp8 ? all<256, true>(*a, ws, stream) : all<256, false>(*a, ws, stream);
  if (rc || ws.row_parts == 1) return rc;
  return (int)mb::launch_kernel_ex(observe_join_kernel, dim3((a->max_ctx + 255) / 256, a->Hkv, a->num_seqs), dim3(256), 0, stream, 1, mb_pdl_enabled() != 0, *a, ws);
}

}  // extern "C"
