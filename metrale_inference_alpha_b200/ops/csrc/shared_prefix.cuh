// Attention of all query rows behind a prefix over that prefix, heads of 64 and 128 dims: outputs, maxima and sums of every part (shared_plan.cuh) for the
// join of shared_attn.cu.
//
// As in attention_rows.cu the rows are tokens x heads of a group, 128 a tile, products on the tensor cores with S, P and O in TMEM, and two tiles in
// turn, so that the softmax of one runs under the products of the other. Behind a prefix few rows are the rule: where a unit has one tile of rows (up to
// 128), both accumulators take the cached tiles of this one in turn. Roles (one CTA an SM, registers moved with setmaxnreg):
//   warps 0-3, 4-7   softmax of accumulator 0 / 1, thread = row; they load their rows' queries and write their outputs
//   warps 8, 10, 11  copies by TMA, a box of up to 16 cached rows each (as many as lie in one block), into rings of pieces of keys and of values; a
//                    warp fills every third place of a ring, since it needs some 90 cycles a box
//   warp 9           the products
//   warps 12-15      (e4m3 cache) make f16 of the values as stored: exact, one conversion per two
// A piece of a bf16 cache is 64 dims of 128 keys, or 64 values of 128 dims. All roles run on from part to part; queries wait for the products of the part in
// front of theirs only.
//
// e4m3 keys are multiplied as they are, by queries that are the sum of two e4m3 numbers: scaled by the power of two that takes a row's largest element to
// [2^7, 2^8), an element's 8 bits are the 4 of its rounding and a remainder of 4, which e4m3 holds exactly down to 2^-2. Elements that are less than
// 2^-9 of the row's largest are off by 2^-17 of it at most, those under 2^-18 of it vanish. That is as many products as of f16 operands, at twice the rate;
// keys of f16 made from e4m3 kept the converting warps busy for as long again as values do (128 sequences behind 32768 tokens 203 us in place of 149).
//
// What bounds it: a double tile takes some 4400 cycles, of which the softmax of either accumulator, and its products and their commits behind it, are one
// chain; a part costs 8000 to 10000 more (queries, first copies, outputs), so that prefixes of a few tiles a CTA are latency. 128 sequences behind 8192
// e4m3 tokens (40 / 8 heads) 48 us: the tensor pipe 29 % busy, the special function units 29 %, HBM 5 %. 61 behind five of 16000 bf16 (64 rows a
// unit and less) 66 us: 243 MB at 3.7 TB/s.
// Weights are f16, held 2^7 larger than the running maximum says, as in attention_rows.cu.
#pragma once
#include "softmax_rows.cuh"
#include "shared_plan.cuh"
#include "smem_limit.h"
#include "tensormap.h"

namespace mbs {

using namespace mbr;
template <int N>
__device__ __forceinline__ void more_regs() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void fewer_regs() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

constexpr float kLift = 7.f;                              // log2 of what f16 weights are held larger by

// Where a part's results lie: element (r, dims 4 c .. 4 c + 3) at o[c * pitch + r], maximum and sum at ml[r]
struct Place {
  float4* o;
  float2* ml;
  size_t pitch;
};
template <int D>
__device__ __forceinline__ Place place_first(const MbSharedArgs& p, const Ws& w, const Plan& s, int group, int kvh, int row, int side) {
  const size_t R = (size_t)p.num_seqs * w.per_seq, at = (size_t)s.start[group] * w.per_seq + row, h = (size_t)side * p.Hkv + kvh;
  uint8_t* ws = reinterpret_cast<uint8_t*>(p.ws);
  return {reinterpret_cast<float4*>(ws + w.first) + h * (D / 4) * R + at, reinterpret_cast<float2*>(ws + w.first_ml) + h * R + at, R};
}
template <int D>
__device__ __forceinline__ Place place_rest(const MbSharedArgs& p, const Ws& w, int cta, int side) {
  const size_t i = (size_t)cta * 2 + side;
  uint8_t* ws = reinterpret_cast<uint8_t*>(p.ws);
  return {reinterpret_cast<float4*>(ws + w.rest) + i * (D / 4) * kRowTile, reinterpret_cast<float2*>(ws + w.rest_ml) + i * kRowTile, kRowTile};
}

// A unit's query rows, every `by`th from one on: one division in front
struct QueryRow {
  const __nv_bfloat16* q;
  size_t ld;                               // heads of a token
  int tok, head, G, by_tok, by_head, kvh;
  __device__ __forceinline__ QueryRow(const MbSharedArgs& p, const Part& x, int G_, int tok0, int row, int by)
      : q(reinterpret_cast<const __nv_bfloat16*>(p.q)), ld(p.Hq), G(G_), kvh(x.kvh) {
    const int at = x.row0 + row, t = at / G;
    tok = tok0 + t;
    head = at - t * G;
    by_tok = by / G;
    by_head = by - by_tok * G;
  }
  __device__ __forceinline__ const __nv_bfloat16* row(int D) const { return q + (tok * ld + kvh * G + head) * D; }
  __device__ __forceinline__ void step() {
    tok += by_tok;
    head += by_head;
    if (head >= G) {
      head -= G;
      ++tok;
    }
  }
};

// A factor of scores in the log2 domain, with the scale of an e4m3 cache in it: never 0, which would make numbers of the -inf that a mask leaves (a scale of 0
// makes scores equal: no score is so large that the smallest normal number does not). A scale that is negative turns the sign of the queries, since the largest
// score is found before the factor; one that is NaN leaves no numbers.
__device__ __forceinline__ float score_factor(float f) { return f >= 0.f ? fmaxf(f, 1.17549435e-38f) : __int_as_float(0x7fffffff); }

// Queries of row r0 + r of a unit, 16-byte piece c of D / 8; an e4m3 cache wants them in f16, scaled (`scale`: what scores are then too small by), times `sign`
template <int D, bool FP8>
__device__ __forceinline__ uint4 query_piece(uint4 v, float sign, float& scale) {
  if constexpr (FP8) {
    // bf16 bits without the sign order like the values: the row's largest over its D / 8 lanes
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __vmaxu2(top, x[j] & 0x7fff7fffu);
#pragma unroll
    for (int d = 1; d < D / 8; d <<= 1) top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, d));
    const int e = (int)(max(top & 0xffff, top >> 16) >> 7);
    const int up = e == 255 ? 0 : 141 - max(e, 15);        // zeros and subnormal rows as if their exponent were 15, infinities and NaN as they are
    const float f = sign * __int_as_float((127 + up) << 23);
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[j]));
      h[j] = pack2<true>(y.x * f, y.y * f);
    }
    scale = __int_as_float((127 - up) << 23);
    return make_uint4(h[0], h[1], h[2], h[3]);
  }
  return v;
}

// Byte offset of 16-byte piece c of row r of an operand of e4m3 numbers, whose rows are D bytes
template <int D>
__device__ __forceinline__ uint32_t query_slot(int r, int c) {
  return (uint32_t)(r * D + ((D == 128 ? c ^ (r & 7) : c ^ ((r >> 1) & 3)) << 4));
}

// A query row as two e4m3 numbers an element, for keys of e4m3, in two tiles of 128 rows of D bytes. Sixteen elements come from the two places that their
// numbers go to, times `sign`. Returns what the row's scores are too large by.
template <int D>
__device__ __forceinline__ float query_pairs(uint8_t* tile, int r, float sign) {
  uint32_t top = 0;                                        // bf16 bits without the sign order like the values
#pragma unroll 4
  for (int c = 0; c < D / 8; ++c) {
    const uint4 v = *reinterpret_cast<const uint4*>(tile + (c & 1) * (128 * D) + query_slot<D>(r, c >> 1));
    top = __vmaxu2(top, __vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu));
    top = __vmaxu2(top, __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  }
  const int e = (int)(max(top & 0xffff, top >> 16) >> 7), up = e == 255 ? 0 : 134 - max(e, 8);
  const float f = sign * __int_as_float((127 + up) << 23);
#pragma unroll 1
  for (int c = 0; c < D / 16; ++c) {
    uint8_t *a = tile + query_slot<D>(r, c), *b = a + 128 * D;
    const uint4 va = *reinterpret_cast<const uint4*>(a), vb = *reinterpret_cast<const uint4*>(b);
    const uint32_t x[8] = {va.x, va.y, va.z, va.w, vb.x, vb.y, vb.z, vb.w};
    uint32_t h[2][4] = {};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float2 y = make_float2(__uint_as_float(x[j] << 16) * f, __uint_as_float(x[j] & 0xffff0000u) * f);
      if (e == 255) {                                      // the type has no infinities: they become NaN
        if (isinf(y.x)) y.x = __int_as_float(0x7fffffff);
        if (isinf(y.y)) y.y = __int_as_float(0x7fffffff);
      }
      const uint32_t one = __nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3), back = e4m3x2(one);
      const float2 z = __half22float2(*reinterpret_cast<const __half2*>(&back));
      const uint32_t two = __nv_cvt_float2_to_fp8x2(make_float2(y.x - z.x, y.y - z.y), __NV_SATFINITE, __NV_E4M3);
      h[0][j >> 1] |= one << (16 * (j & 1));
      h[1][j >> 1] |= two << (16 * (j & 1));
    }
    *reinterpret_cast<uint4*>(a) = make_uint4(h[0][0], h[0][1], h[0][2], h[0][3]);
    *reinterpret_cast<uint4*>(b) = make_uint4(h[1][0], h[1][1], h[1][2], h[1][3]);
  }
  return __int_as_float((127 - up) << 23);
}

// Operand rows of 64 bytes: pieces of 16 bytes exchanged by (row / 2) mod 4, eight rows 512 bytes
__device__ __forceinline__ uint64_t umma_desc_sw64(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(512 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)4 << 61;
  return d;
}

// K and V tiles of kT cached tokens of this CTA's parts, one after the other, into two stages each: 128 threads, t the number of this one
template <int D, bool FP8, int kT>
__device__ __forceinline__ void load_tiles(const MbSharedArgs& p, const Ws& ws, const Plan& plan, int begin, int end, uint8_t* sK, uint8_t* sV, uint64_t* k_full,
                                           uint64_t* k_empty, uint64_t* v_full, uint64_t* v_empty, int t) {
  constexpr int kTileB = kT * D * 2;
  const int lane = t & 31;
  constexpr int kPieces = FP8 ? D / 16 : D / 8;         // 16-byte pieces of a cached row
  constexpr int kStep = 128 / kPieces, kN = kT / kStep; // rows between a thread's pieces, and how many it has
  const int r0 = t / kPieces, c = t % kPieces;
  const size_t row_bytes = (size_t)D * (FP8 ? 1 : 2), pitch = (size_t)p.Hkv * row_bytes;
  const int shift = (p.block_size & (p.block_size - 1)) == 0 ? 31 - __clz(p.block_size) : -1;
  int pos = begin;
  Part x;
  x.t0 = x.t1 = 0;
  int at = 0;                                           // the tile whose places are looked up next
  bool more = true;
  // the places in the cache of this thread's rows of the next tile (-1: behind the prefix, or no tile), looked up a tile before they are read
  int bad = 0;
  auto places = [&](int* place, size_t& off) {
    if (more && at == x.t1) {
      more = next_part<D>(plan, p.groups, ws.per_seq, pos, end, x);
      at = x.t0;
    }
    if (!more) {
#pragma unroll
      for (int i = 0; i < kN; ++i) place[i] = -1;
      return false;
    }
    const int len = plan.len[x.group];
    const int* bt = p.prefix_table + (size_t)x.group * p.prefix_ld;
    off = x.kvh * row_bytes + (size_t)c * 16;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int tok = at * kT + r0 + i * kStep, in = min(tok, len - 1);
      const int bi = shift >= 0 ? in >> shift : in / p.block_size;
      int blk = bt[bi];
      const bool out = (unsigned)blk >= (unsigned long long)p.num_blocks;
      bad |= out;
      blk = out ? 0 : blk;
      place[i] = tok < len ? blk * p.block_size + (in - bi * p.block_size) : -1;
    }
    ++at;
    return true;
  };
  bool ok = true;
  if constexpr (FP8) {
    uint4 kr[kN], vr[kN];
    int next[kN];
    size_t off = 0;
    auto fetch = [&](const void* cache, uint4* raw) {
      const uint8_t* base = reinterpret_cast<const uint8_t*>(cache) + off;
#pragma unroll
      for (int i = 0; i < kN; ++i)
        raw[i] = next[i] >= 0 ? __ldg(reinterpret_cast<const uint4*>(base + (size_t)next[i] * pitch)) : make_uint4(0, 0, 0, 0);
    };
    auto put = [&](uint8_t* tile, const uint4* raw) {
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = r0 + i * kStep;
        const uint32_t y[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
        uint32_t h[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          h[2 * k] = e4m3x2(y[k]);
          h[2 * k + 1] = e4m3x2(y[k] >> 16);
        }
        uint8_t* half = tile + (c >> 2) * (kT * 128);
        *reinterpret_cast<uint4*>(half + sw_off(r, (c & 3) * 2)) = make_uint4(h[0], h[1], h[2], h[3]);
        *reinterpret_cast<uint4*>(half + sw_off(r, (c & 3) * 2 + 1)) = make_uint4(h[4], h[5], h[6], h[7]);
      }
    };
    bool have = places(next, off);
    fetch(p.k_cache, kr);
    fetch(p.v_cache, vr);
    bool then = places(next, off);
    for (int j = 0; have; ++j) {
      const int b = j & 1;
      const uint32_t ph = ((j >> 1) & 1) ^ 1;
      ok = mb::mbar_wait(&k_empty[b], ph, p.status, MB_ST_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      put(sK + b * kTileB, kr);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mb::mbar_arrive(&k_full[b]);
      fetch(p.k_cache, kr);
      ok = mb::mbar_wait(&v_empty[b], ph, p.status, MB_ST_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      put(sV + b * kTileB, vr);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mb::mbar_arrive(&v_full[b]);
      fetch(p.v_cache, vr);
      have = then;
      then = places(next, off);
    }
  } else {
    int now[kN], next[kN];
    size_t off = 0, ahead = 0;
    auto copy = [&](const void* cache, uint8_t* tile) {
      const uint8_t* base = reinterpret_cast<const uint8_t*>(cache) + off;
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r = r0 + i * kStep;
        const bool there = now[i] >= 0;
        const uint8_t* src = base + (there ? (size_t)now[i] * pitch : 0);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mb::smem_u32(tile + (c >> 3) * (kT * 128) + sw_off(r, c & 7))),
                     "l"(src), "r"(there ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // the copies of a tile are announced while the next tile's are in flight
    auto announce = [&](uint64_t* bar) {
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mb::mbar_arrive(bar);
    };
    bool have = places(next, ahead);
    int j = 0;
    for (; have; ++j) {
      const int b = j & 1;
      const uint32_t ph = ((j >> 1) & 1) ^ 1;
#pragma unroll
      for (int i = 0; i < kN; ++i) now[i] = next[i];
      off = ahead;
      have = places(next, ahead);
      ok = mb::mbar_wait(&k_empty[b], ph, p.status, MB_ST_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      copy(p.k_cache, sK + b * kTileB);
      if (j > 0) {
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        announce(&v_full[b ^ 1]);
      }
      ok = mb::mbar_wait(&v_empty[b], ph, p.status, MB_ST_TIMEOUT_TMA);
      if (!__all_sync(0xffffffffu, ok)) break;
      copy(p.v_cache, sV + b * kTileB);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      announce(&k_full[b]);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (__all_sync(0xffffffffu, ok) && j > 0) announce(&v_full[(j - 1) & 1]);
  }
  if (bad && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
}

// How cached rows are copied: boxes of 16 >> bits rows, the largest that every block is a multiple of
struct Boxes {
  int bits;
};

template <int D, bool FP8>
struct PrefixCfg {
  static constexpr int kT = 128, kThreads = FP8 ? 512 : 384;
  static constexpr int kQB = 128 * D * 2, kSpans = D / 64;
  // pieces of keys (bf16: a span of 64 dims, e4m3: a tile as stored) and of values (as many runs of tokens as there are spans)
  static constexpr int kKeyB = FP8 ? kT * D : 16384, kKeys = FP8 ? 1 : kSpans, kKeyRing = FP8 ? 49152 / kKeyB : 5;
  static constexpr int kValB = 16384, kVals = kSpans, kValTok = kT / kVals, kValRing = 4;
  static constexpr int kRawB = FP8 ? kT * D : 0, kRawRing = FP8 ? 32768 / kRawB : 0;     // values of a tile as stored
  static constexpr int kRing = kKeyRing * kKeyB + kValRing * kValB + kRawRing * kRawB;
  static constexpr int kSmem = 2 * kQB + kRing + 1024 + (int)sizeof(Plan);
};

// Places in a ring
template <int N>
struct Cursor {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void step() {
    if (++slot == N) {
      slot = 0;
      parity ^= 1;
    }
  }
  __device__ __forceinline__ void step(int n) {
    const int total = slot + n;
    parity ^= (total / N) & 1;
    slot = total % N;
  }
};

template <int D, bool FP8>
__global__ void __launch_bounds__(PrefixCfg<D, FP8>::kThreads, 1)
shared_prefix_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmK1,
                     const __grid_constant__ CUtensorMap tmV1, const Boxes boxes, const MbSharedArgs p, const Ws ws) {
  using C = PrefixCfg<D, FP8>;
  constexpr int kT = C::kT, kQB = C::kQB, kSpans = C::kSpans, kKeyRing = C::kKeyRing, kValRing = C::kValRing, kRaw = FP8 ? C::kRawRing : 1;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* sQ = smem_raw + ((1024u - (mb::smem_u32(smem_raw) & 1023u)) & 1023u);   // 2 row tiles x spans of 64 dims x [128 rows x 128 B]
  uint8_t* sK = sQ + 2 * kQB;                             // rings of keys, of values, of values as stored
  uint8_t* sV = sK + kKeyRing * C::kKeyB;
  uint8_t* sB = sV + kValRing * C::kValB;
  Plan& plan = *reinterpret_cast<Plan*>(sB + C::kRawRing * C::kRawB);
  __shared__ __align__(8) uint64_t q_full[2], q_raw[2], q_free, k_full[kKeyRing], k_empty[kKeyRing], v_full[kValRing], v_empty[kValRing], raw_full[kRaw], raw_empty[kRaw], s_full[2],
      p_full[2][2], o_full[2];
  __shared__ uint32_t s_tmem;
  __shared__ float s_qscale[FP8 ? 2 : 1][2][128];         // what a row's scores are too large by (e4m3 cache), of parts in turn
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = ws.G;
  mb::pdl_wait();
  if (warp == 0) {
    make_plan<D>(p, plan, ws.per_seq, lane);
  } else if (warp == 1 && lane == 0) {
    mb::mbar_init(&q_free, 1);
    for (int i = 0; i < 2; ++i) {
      mb::mbar_init(&q_full[i], 4);
      mb::mbar_init(&q_raw[i], 4);
      mb::mbar_init(&s_full[i], 1);
      mb::mbar_init(&p_full[i][0], 4);
      mb::mbar_init(&p_full[i][1], 4);
      mb::mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < kKeyRing; ++i) {
      mb::mbar_init(&k_full[i], 1);
      mb::mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < kValRing; ++i) {
      mb::mbar_init(&v_full[i], FP8 ? 4 : 1);
      mb::mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < kRaw; ++i) {
      mb::mbar_init(&raw_full[i], 1);
      mb::mbar_init(&raw_empty[i], 4);
    }
    mb::mbar_fence_init();
  }
  if (warp == 9) mb::tmem_alloc(&s_tmem, 512);
  mb::tc_fence_before();
  __syncthreads();
  mb::tc_fence_after();
  mb::pdl_launch_dependents();                            // behind this kernel's own wait: what the step before it wrote is there for them too
  const uint32_t tmem = s_tmem;                           // S0 0-127, S1 128-255, O0 256-, O1 384-
  const int W = plan.base[p.groups], used = used_ctas(W, ws.ctas);
  const Share share(W, used);
  const bool idle = (int)blockIdx.x >= used;
  const int begin = idle ? 0 : share.first(blockIdx.x), end = idle ? 0 : share.first(blockIdx.x + 1);
  int pos = begin;
  Part x;

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    if constexpr (FP8) more_regs<184>();                  // 184 + 184 + 72 + 72 are the 4 x 128 of the launch
    else more_regs<216>();                                // 216 + 216 + 72 are the 3 x 168
    const int w = warp >> 2, r = tid & 127;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + lanes + w * 128, tO = tmem + lanes + 256 + w * 128;
    const float ks = FP8 ? *p.k_scale : 1.f, sign = ks < 0.f ? -1.f : 1.f, sc0 = p.scale * fabsf(ks) * 1.44269504088896f;
    uint32_t part = 0, done = 0, outs = 0, raws = 0;      // parts, tiles, outputs and query tiles that this accumulator has had
    bool ok = true;
    while (ok && next_part<D>(plan, p.groups, ws.per_seq, pos, end, x)) {
      const int n = x.t1 - x.t0, mine = x.two ? n : (n + 1 - w) / 2;
      // a wait tells a phase from its neighbours only: no warp may be two parts ahead of one that waits, so every part's queries wait for all products
      // of the former one's
      if (part > 0) ok = mb::mbar_wait(&q_free, (part - 1) & 1, p.status, MB_ST_TIMEOUT_MMA);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      // Rows come by whole pieces, neighbours to neighbouring threads (a thread that read a row of its own met a cache line in each of its loads: 12000
      // cycles a part). Past the last one, up to a multiple of 32, they are zeros; those behind belong to warps that do not look at their scores. Where the
      // accumulators share the rows the first one's threads bring them.
      const int side = x.two ? w : 0, left = x.rows - side * 128;            // whose rows these are, and how many
      const bool live = r < left, some = (warp & 3) * 32 < left;
      float sc = sc0;
      if (side == w) {
        constexpr int kPieces = D / 8, kStep = 128 / kPieces;
        const int c = r % kPieces, first = r / kPieces, last = min(left, 128) - 1;
        QueryRow at(p, x, G, plan.start[x.group] * p.q_len, w * 128 + min(first, last), kStep);
        // bf16 as the products take it; else where the two numbers made of a piece's elements, and its neighbour's, will be
        uint8_t* dst = sQ + w * kQB + (FP8 ? (c & 1) * (128 * D) : (c >> 3) * (128 * 128));
#pragma unroll 4
        for (int i = 0; i < kPieces; ++i) {
          const int qr = first + kStep * i;
          if (kStep * i > (last | 31)) break;
          const uint32_t to = FP8 ? query_slot<D>(qr, c >> 1) : sw_off(qr, c & 7);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(mb::smem_u32(dst + to)), "l"(reinterpret_cast<const uint4*>(at.row(D)) + c),
                       "r"(qr <= last ? 16 : 0)
                       : "memory");
          if (qr + kStep <= last) at.step();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        if constexpr (FP8) {
          __syncwarp();
          if (lane == 0) mb::mbar_arrive(&q_raw[w]);
          ok = mb::mbar_wait(&q_raw[w], raws & 1, p.status, MB_ST_TIMEOUT_MMA);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          ++raws;
          if (some) {
            const float back = query_pairs<D>(sQ + w * kQB, r, sign);
            s_qscale[part & 1][w][r] = back;
            sc = score_factor(sc * back);
          }
        }
        fence_async_smem();
      } else if constexpr (FP8) {
        ok = mb::mbar_wait(&q_full[0], part & 1, p.status, MB_ST_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        sc = score_factor(sc * s_qscale[part & 1][0][r]);
      }
      __syncwarp();
      if (lane == 0) mb::mbar_arrive(&q_full[w]);
      const int len = plan.len[x.group];
      float m_run = -INFINITY, l_run = 0.f;
      auto rescale = [&](float alpha) {                   // S seen: the products that were issued in front of it are done
#pragma unroll
        for (int c = 0; c < D; c += 16) {
          float ov[16];
          mb::tmem_ld16(tO + c, ov);
#pragma unroll
          for (int k = 0; k < 16; ++k) ov[k] *= alpha;
          mb::tmem_st16(tO + c, ov);
        }
      };
      auto announce = [&](int h) {
        mb::tc_fence_before();
        __syncwarp();
        if (lane == 0) mb::mbar_arrive(&p_full[w][h]);
      };
      for (int i = 0; i < mine; ++i) {
        const int t = x.t0 + (x.two ? i : 2 * i + w);
        ok = mb::mbar_wait(&s_full[w], (done + i) & 1, p.status, MB_ST_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        mb::tc_fence_after();
        if (!some) {                                      // warps without rows hand on what the columns hold: it meets no other row
          announce(0);
          announce(1);
          continue;
        }
        softmax_tile<FP8>(tS, len - t * kT, sc, FP8 ? kLift : 0.f, i == 0, m_run, l_run, rescale, announce);
      }
      if (!ok) break;
      if (mine > 0) {
        ok = mb::mbar_wait(&o_full[w], outs & 1, p.status, MB_ST_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        mb::tc_fence_after();
        ++outs;
      }
      const Place to = x.t0 == 0 ? place_first<D>(p, ws, plan, x.group, x.kvh, x.row0 + (x.two ? w * 128 : 0), x.two ? 0 : w) : place_rest<D>(p, ws, blockIdx.x, w);
      if (mine > 0 && some) {
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          float o[32];
          mb::tmem_ld32_async(tO + c0, o);
          mb::tmem_ld_wait(o);
          if (live)
#pragma unroll
            for (int c = 0; c < 8; ++c) to.o[(c0 / 4 + c) * to.pitch + r] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        }
      }
      if (live) to.ml[r] = make_float2(m_run - (FP8 ? kLift : 0.f), l_run);
      mb::tc_fence_before();
      done += mine;
      ++part;
    }
  } else {
    fewer_regs<72>();
    if (warp < 12 && warp != 9) {
      // ---------------------------------------------------------- copies
      const int bits = boxes.bits, box = 16 >> bits, count = kT / box;       // rows of a box, boxes of a tile
      constexpr int kMost = 4;                                               // of a lane: 128 boxes of one row
      const int shift = (p.block_size & (p.block_size - 1)) == 0 ? 31 - __clz(p.block_size) : -1;
      const int nowhere = (int)(p.num_blocks * p.block_size);                // rows from here on read as zeros
      const int who = warp == 8 ? 0 : warp - 9;
      constexpr int kValSlots = FP8 ? kRaw : kValRing;
      uint64_t *val_full = FP8 ? raw_full : v_full, *val_empty = FP8 ? raw_empty : v_empty;
      Cursor<kKeyRing> at_key;
      Cursor<kValSlots> at_val;
      uint32_t keys_asked = 0, vals_asked = 0, key_parities = 0, val_parities = 0;      // slots that this warp has filled, with which parity the last time
      bool ok = true;
      int bad = 0;
      while (ok && next_part<D>(plan, p.groups, ws.per_seq, pos, end, x)) {
        const int len = plan.len[x.group];
        const int* bt = p.prefix_table + (size_t)x.group * p.prefix_ld;
        // a tile's boxes: lane l has boxes l, l + 32, ...; looked up a tile ahead
        auto places = [&](int t, int (&place)[kMost]) {
#pragma unroll
          for (int i = 0; i < kMost; ++i) {
            const int b = lane + 32 * i, tok = t * kT + b * box;
            place[i] = nowhere;
            if (b < count && t < x.t1 && tok < len) {
              const int bi = shift >= 0 ? tok >> shift : tok / p.block_size;
              int blk = bt[bi];
              if ((unsigned)blk >= (unsigned long long)p.num_blocks) {
                bad = 1;
                blk = 0;
              }
              place[i] = blk * p.block_size + (tok - bi * p.block_size);
            }
          }
        };
        int now[kMost], next[kMost];
        places(x.t0, next);
        for (int t = x.t0; t < x.t1 && ok; ++t) {
#pragma unroll
          for (int i = 0; i < kMost; ++i) now[i] = next[i];
          places(t + 1, next);
          // tokens [tok0, tok0 + n) of the tile, 128 bytes (or a whole shorter row) of each from byte c0 on, to dst
          auto bring = [&](bool keys, uint64_t* bar, uint8_t* dst, int tok0, int n, int c0) {
            constexpr int kRowB = FP8 ? D : 128;
            const CUtensorMap *m = keys ? &tmK : &tmV, *m1 = keys ? &tmK1 : &tmV1;
#pragma unroll
            for (int i = 0; i < kMost; ++i) {
              const int b = lane + 32 * i, in = b * box - tok0;              // the box's first row in the piece
              if (in < 0 || in >= n || b >= count) continue;
              const int left = len - (t * kT + b * box);
              if (FP8 || left <= 0 || left >= box) {
                mb::tma_load_3d(dst + in * kRowB, m, bar, c0, x.kvh, now[i]);
              } else {                                                       // the prefix ends inside: values behind it must be zeros
                for (int k = 0; k < box; ++k) mb::tma_load_3d(dst + (in + k) * kRowB, m1, bar, c0, x.kvh, k < left ? now[i] + k : nowhere);
              }
            }
          };
          // Whether a place is this warp's to fill, and it is empty. A place is always the same warp's: a wait tells a phase from its neighbours only, and a warp
          // that took another's place could be two rounds of it ahead of the products
          auto mine = [&](int owner, uint64_t* empty, uint32_t parity) {
            if (owner % 3 != who) return false;
            ok = ok && mb::mbar_wait(empty, parity ^ 1, p.status, MB_ST_TIMEOUT_TMA);
            if (!__all_sync(0xffffffffu, ok)) ok = false;
            return ok;
          };
          for (int c = 0; c < C::kKeys && ok; ++c) {
            if (mine(at_key.slot, &k_empty[at_key.slot], at_key.parity)) {
              uint64_t* bar = &k_full[at_key.slot];
              if (lane == 0) mb::mbar_expect_tx(bar, C::kKeyB);
              __syncwarp();
              bring(true, bar, sK + at_key.slot * C::kKeyB, 0, kT, c * 128);
              __syncwarp();
              keys_asked |= 1u << at_key.slot;
              key_parities = (key_parities & ~(1u << at_key.slot)) | at_key.parity << at_key.slot;
            }
            at_key.step();
          }
          for (int c = 0; c < (FP8 ? 1 : C::kVals) && ok; ++c) {
            if (mine(at_val.slot + (FP8 ? 1 : 2), &val_empty[at_val.slot], at_val.parity)) {
              uint64_t* bar = &val_full[at_val.slot];
              if (lane == 0) mb::mbar_expect_tx(bar, FP8 ? C::kRawB : C::kValB);
              __syncwarp();
              if constexpr (FP8) {
                bring(false, bar, sB + at_val.slot * C::kRawB, 0, kT, 0);
              } else {
                uint8_t* dst = sV + at_val.slot * C::kValB;
                for (int d = 0; d < kSpans; ++d) bring(false, bar, dst + d * (C::kValB / kSpans), c * C::kValTok, C::kValTok, d * 128);
              }
              __syncwarp();
              vals_asked |= 1u << at_val.slot;
              val_parities = (val_parities & ~(1u << at_val.slot)) | at_val.parity << at_val.slot;
            }
            at_val.step();
          }
        }
      }
      // given up: no copy may still be under way when the CTA ends
      if (!ok) {
        for (int i = 0; i < kKeyRing; ++i)
          if (keys_asked >> i & 1) mb::mbar_wait(&k_full[i], key_parities >> i & 1, p.status, MB_ST_TIMEOUT_TMA);
        for (int i = 0; i < kValSlots; ++i)
          if (vals_asked >> i & 1) mb::mbar_wait(&val_full[i], val_parities >> i & 1, p.status, MB_ST_TIMEOUT_TMA);
      }
      if (bad && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
    } else if (warp >= 12) {
      // ---------------------------------------------------------- e4m3 to f16
      if constexpr (FP8) {
        const int t128 = tid - 384;
        constexpr int kPieces = D / 16, kStep = 128 / kPieces, kN = kT / kStep;           // 16-byte pieces of a row, rows between a thread's, and how many
        const int c = t128 % kPieces, r0 = t128 / kPieces, sub = c >> 2, chunk = (c & 3) * 2;
        // half of the lanes stores its pieces in the other order: eight lanes' stores then meet eight bank groups
        const int odd = (D == 128 ? c >> 2 : c >> 1) & 1;
        Cursor<kRaw> raw;
        Cursor<kValRing> at;
        bool ok = true;
        while (ok && next_part<D>(plan, p.groups, ws.per_seq, pos, end, x)) {
          const int len = plan.len[x.group];
#pragma unroll 1
          for (int t = x.t0; t < x.t1 && ok; ++t) {
            const int left = len - t * kT;                 // rows from here on are zeros
            ok = mb::mbar_wait(&raw_full[raw.slot], raw.parity, p.status, MB_ST_TIMEOUT_TMA);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            const uint8_t* src = sB + raw.slot * C::kRawB + r0 * D + c * 16;
            uint4 y[kN];
#pragma unroll
            for (int i = 0; i < kN; ++i) y[i] = *reinterpret_cast<const uint4*>(src + kStep * i * D);
            __syncwarp();
            if (lane == 0) mb::mbar_arrive(&raw_empty[raw.slot]);
            raw.step();
#pragma unroll
            for (int v = 0; v < C::kVals; ++v) {
              ok = ok && mb::mbar_wait(&v_empty[at.slot], at.parity ^ 1, p.status, MB_ST_TIMEOUT_TMA);
              if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
              uint8_t* dst = sV + at.slot * C::kValB + sub * (C::kValB / kSpans);
#pragma unroll
              for (int i = v * kN / C::kVals; i < (v + 1) * kN / C::kVals; ++i) {
                const int r = r0 + kStep * i;
                if (r >= left) y[i] = make_uint4(0, 0, 0, 0);
                const uint32_t z[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
                uint32_t h[8];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  h[2 * k] = e4m3x2(z[k]);
                  h[2 * k + 1] = e4m3x2(z[k] >> 16);
                }
                uint8_t *to = dst + sw_off(r % C::kValTok, chunk), *also = dst + sw_off(r % C::kValTok, chunk + 1);
                const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
                *reinterpret_cast<uint4*>(odd ? also : to) = odd ? hi : lo;
                *reinterpret_cast<uint4*>(odd ? to : also) = odd ? lo : hi;
              }
              fence_async_smem();
              __syncwarp();
              if (lane == 0) mb::mbar_arrive(&v_full[at.slot]);
              at.step();
            }
          }
        }
      }
    } else if (warp == 9 && mb::elect_one()) {
      // ---------------------------------------------------------- products
      constexpr uint32_t kF = FP8 ? 0 : 1;                 // of f16 / bf16 operands; e4m3 is 0 among its own
      constexpr uint32_t kIdS = mb::umma_idesc(kF, kF, 128, kT), kIdO = mb::umma_idesc(kF, kF, 128, D, 0, 1);
      // descriptors count 16 bytes: an operand's next step is an addition
      const bool narrow = FP8 && D == 64;
      const uint64_t dQ = narrow ? umma_desc_sw64(mb::smem_u32(sQ)) : mb::umma_desc_sw128(mb::smem_u32(sQ)),
                     dK = narrow ? umma_desc_sw64(mb::smem_u32(sK)) : mb::umma_desc_sw128(mb::smem_u32(sK)),
                     dV = mb::umma_desc_sw128_mn(mb::smem_u32(sV), C::kValB / kSpans, 1024);
      Cursor<kKeyRing> key;                               // the part's first pieces
      Cursor<kValRing> val;
      uint32_t part = 0, done0 = 0, done1 = 0;            // parts, tiles that either accumulator has had
      bool ok = true;
      while (ok && next_part<D>(plan, p.groups, ws.per_seq, pos, end, x)) {
        const int n = x.t1 - x.t0, n0 = x.two ? n : (n + 1) / 2, n1 = x.two ? n : n / 2, by = x.two ? 1 : 2;
        Cursor<kKeyRing> k0 = key, k1 = key;              // where either accumulator's next keys and values lie
        Cursor<kValRing> v0 = val, v1 = val;
        if (!x.two) {
          k1.step(C::kKeys);
          v1.step(C::kVals);
        }
        // w: accumulator; `last`: nobody else takes these pieces
        auto scores = [&](int w, Cursor<kKeyRing>& at, bool last) {
          Cursor<kKeyRing> c = at;
#pragma unroll
          for (int h = 0; h < C::kKeys; ++h) {
            if (!mb::mbar_wait(&k_full[c.slot], c.parity, p.status, MB_ST_TIMEOUT_MMA)) return false;
            mb::tc_fence_after();
            const uint64_t q = dQ + (x.two ? w : 0) * (kQB >> 4) + ((h * 16384) >> 4), k = dK + c.slot * (C::kKeyB >> 4);
            if constexpr (FP8) {
#pragma unroll
              for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int s = 0; s < D / 32; ++s) mb::umma_f8f6f4(tmem + w * 128, q + ((t * 128 * D + s * 32) >> 4), k + ((s * 32) >> 4), kIdS, (t | s) != 0);
            } else {
#pragma unroll
              for (int s = 0; s < 4; ++s) mb::umma_f16(tmem + w * 128, q + ((s * 32) >> 4), k + ((s * 32) >> 4), kIdS, (h | s) != 0);
            }
            if (last) mb::tc_commit(&k_empty[c.slot]);
            c.step();
          }
          mb::tc_commit(&s_full[w]);
          at.step(by * C::kKeys);
          return true;
        };
        auto values = [&](int w, Cursor<kValRing>& at, bool last, uint32_t done, bool fresh) {
          Cursor<kValRing> c = at;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (!mb::mbar_wait(&v_full[c.slot], c.parity, p.status, MB_ST_TIMEOUT_MMA) ||
                !mb::mbar_wait(&p_full[w][h], done & 1, p.status, MB_ST_TIMEOUT_MMA))
              return false;
            mb::tc_fence_after();
            const uint64_t v = dV + c.slot * (C::kValB >> 4) + (kSpans == 1 ? h * 4 * (2048 >> 4) : 0);
#pragma unroll
            for (int s = 0; s < 4; ++s) umma_f16_ta(tmem + 256 + w * 128, tmem + w * 128 + (h * 4 + s) * 8, v + ((s * 2048) >> 4), kIdO, !(fresh && h == 0 && s == 0));
            if (h == 1 || kSpans == 2) {
              if (last) mb::tc_commit(&v_empty[c.slot]);
              c.step();
            }
          }
          at.step(by * C::kVals);
          return true;
        };
        // rows are written, and the outputs of the part in front read
        ok = mb::mbar_wait(&q_full[0], part & 1, p.status, MB_ST_TIMEOUT_MMA) && mb::mbar_wait(&q_full[1], part & 1, p.status, MB_ST_TIMEOUT_MMA);
        if (ok) ok = scores(0, k0, !x.two);
        if (ok && n1 > 0) ok = scores(1, k1, true);
        for (int i = 0; i < n0 && ok; ++i) {
          ok = values(0, v0, !x.two, done0 + i, i == 0);
          if (!ok) break;
          if (i + 1 < n0) ok = scores(0, k0, !x.two);
          else mb::tc_commit(&o_full[0]);
          if (!ok || i >= n1) break;
          ok = values(1, v1, true, done1 + i, i == 0);
          if (!ok) break;
          if (i + 1 < n1) ok = scores(1, k1, true);
          else mb::tc_commit(&o_full[1]);
        }
        mb::tc_commit(&q_free);
        key.step(n * C::kKeys);
        val.step(n * C::kVals);
        done0 += n0;
        done1 += n1;
        ++part;
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

// Heads of 256 dims: one tile of 128 rows a CTA (its outputs are half of TMEM), tiles of 64 cached tokens, two tiles of scores in turn: the products of the
// next one run under the softmax of this one. Warps 0-3 softmax, 4-7 loader, 8 products. Short prefixes are latency: 33 sequences behind two of 2047 bf16
// tokens (16 / 2 heads, one to two tiles a CTA) 17 us, the tensor pipe 4 % busy, HBM 6 %.
template <bool FP8>
__global__ void __launch_bounds__(288, 1) shared_prefix256_kernel(const MbSharedArgs p, const Ws ws) {
  constexpr int D = 256, kT = 64, kQB = 128 * D * 2, kTileB = kT * D * 2, kSpans = D / 64;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  uint8_t* sQ = smem_raw + ((1024u - (mb::smem_u32(smem_raw) & 1023u)) & 1023u);   // 4 spans x [128 rows x 128 B]
  uint8_t* sK = sQ + kQB;                                 // 2 stages x 4 spans x [64 tokens x 128 B]
  uint8_t* sV = sK + 2 * kTileB;
  Plan& plan = *reinterpret_cast<Plan*>(sV + 2 * kTileB);
  __shared__ __align__(8) uint64_t q_full, k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_done, o_full;
  __shared__ uint32_t s_tmem;
  __shared__ float s_qscale[2][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = ws.G;
  mb::pdl_wait();
  if (warp == 0) {
    make_plan<D>(p, plan, ws.per_seq, lane);
  } else if (warp == 1 && lane == 0) {
    mb::mbar_init(&q_full, 4);
    mb::mbar_init(&o_done, 1);
    mb::mbar_init(&o_full, 1);
    for (int i = 0; i < 2; ++i) {
      mb::mbar_init(&k_full[i], 4);
      mb::mbar_init(&v_full[i], 4);
      mb::mbar_init(&k_empty[i], 1);
      mb::mbar_init(&v_empty[i], 1);
      mb::mbar_init(&s_full[i], 1);
      mb::mbar_init(&p_full[i], 4);
    }
    mb::mbar_fence_init();
  }
  if (warp == 8) mb::tmem_alloc(&s_tmem, 512);
  mb::tc_fence_before();
  __syncthreads();
  mb::tc_fence_after();
  mb::pdl_launch_dependents();
  const uint32_t tmem = s_tmem;                           // S0 0-63, S1 64-127, O 256-511
  const int W = plan.base[p.groups], used = used_ctas(W, ws.ctas);
  const Share share(W, used);
  const bool idle = (int)blockIdx.x >= used;
  const int begin = idle ? 0 : share.first(blockIdx.x), end = idle ? 0 : share.first(blockIdx.x + 1);

  if (warp < 4) {
    // ------------------------------------------------------------ softmax
    const uint32_t lanes = (uint32_t)(warp * 32) << 16;
    const uint32_t tO = tmem + lanes + 256;
    const float ks = FP8 ? *p.k_scale : 1.f, sign = ks < 0.f ? -1.f : 1.f, sc0 = p.scale * fabsf(ks) * 1.44269504088896f;
    uint32_t part = 0, base = 0;                          // parts, tiles that are done
    bool ok = true;
    int pos = begin;
    Part x;
    while (ok && next_part<D>(plan, p.groups, ws.per_seq, pos, end, x)) {
      const int n = x.t1 - x.t0, last = x.rows - 1;
      // 128 rows x 32 pieces of 8 dims, sixteen of a thread's loads in flight together (rows past the last one are zeros)
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint4 v[16];
        QueryRow at(p, x, G, plan.start[x.group] * p.q_len, min(warp + 64 * half, last), 4);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          v[i] = *(reinterpret_cast<const uint4*>(at.row(D)) + lane);
          if (warp + 4 * (half * 16 + i + 1) <= last) at.step();
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int qr = warp + 4 * (half * 16 + i);
          if (qr > last) v[i] = make_uint4(0, 0, 0, 0);
          float back = 1.f;
          v[i] = query_piece<D, FP8>(v[i], sign, back);
          if (FP8 && lane == 0) s_qscale[part & 1][qr] = back;
          *reinterpret_cast<uint4*>(sQ + (lane >> 3) * (128 * 128) + sw_off(qr, lane & 7)) = v[i];
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mb::mbar_arrive(&q_full);
      float sc = sc0;
      if constexpr (FP8) {
        ok = mb::mbar_wait(&q_full, part & 1, p.status, MB_ST_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        sc = score_factor(sc * s_qscale[part & 1][tid]);
      }
      const bool live = tid <= last, some = warp * 32 <= last;
      const int len = plan.len[x.group];
      float m_run = -INFINITY, l_run = 0.f;
      for (int i = 0; i < n; ++i) {
        const uint32_t j = base + i, tS = tmem + lanes + (j & 1) * kT;
        ok = mb::mbar_wait(&s_full[j & 1], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_MMA);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        mb::tc_fence_after();
        if (some) {
          float s[kT];
#pragma unroll
          for (int c = 0; c < kT; c += 32) mb::tmem_ld32_async(tS + c, s + c);
          mb::tmem_ld_wait(s);
          const int seen = len - (x.t0 + i) * kT;
          if (seen < kT) {
#pragma unroll
            for (int k = 0; k < kT; ++k)
              if (k >= seen) s[k] = -INFINITY;
          }
          float mx4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int k = 4; k < kT; ++k) mx4[k & 3] = fmaxf(mx4[k & 3], s[k]);
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc;
          float alpha = 1.f;
          const bool move = mx > m_run + 8.f;
          if (move) {
            alpha = ex2(m_run - mx);
            m_run = mx;
          }
          if (i > 0 && __any_sync(0xffffffffu, move)) {
            ok = mb::mbar_wait(&o_done, (j - 1) & 1, p.status, MB_ST_TIMEOUT_MMA);     // P V of the tile before: that of this one waits for this warp
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            mb::tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 16) {
              float ov[16];
              mb::tmem_ld16(tO + c, ov);
#pragma unroll
              for (int k = 0; k < 16; ++k) ov[k] *= alpha;
              mb::tmem_st16(tO + c, ov);
            }
          }
          const float nm = m_run == -INFINITY ? 0.f : (FP8 ? kLift : 0.f) - m_run;
          const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
          uint32_t pk[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float2 e = fma2(make_float2(s[2 * k], s[2 * k + 1]), sc2, nm2);
            e.x = ex2(e.x);
            e.y = ex2(e.y);
            sum[k & 1] = add2(sum[k & 1], e);
            pk[k] = pack2<FP8>(e.x, e.y);
          }
          tmem_st32(tS, pk);
          mb::tmem_st_wait();
          l_run = l_run * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
        }
        mb::tc_fence_before();
        __syncwarp();
        if (lane == 0) mb::mbar_arrive(&p_full[j & 1]);
      }
      if (!ok) break;
      ok = mb::mbar_wait(&o_full, part & 1, p.status, MB_ST_TIMEOUT_MMA);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      mb::tc_fence_after();
      const Place to = x.t0 == 0 ? place_first<D>(p, ws, plan, x.group, x.kvh, x.row0, 0) : place_rest<D>(p, ws, blockIdx.x, 0);
      if (some) {
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 64) {
          float o[64];
          mb::tmem_ld32_async(tO + c0, o);
          mb::tmem_ld32_async(tO + c0 + 32, o + 32);
          mb::tmem_ld_wait(o);
          if (live)
#pragma unroll
            for (int c = 0; c < 16; ++c) to.o[(c0 / 4 + c) * to.pitch + tid] = make_float4(o[4 * c], o[4 * c + 1], o[4 * c + 2], o[4 * c + 3]);
        }
      }
      if (live) to.ml[tid] = make_float2(m_run - (FP8 ? kLift : 0.f), l_run);
      mb::tc_fence_before();
      base += n;
      ++part;
    }
  } else if (warp < 8) {
    load_tiles<D, FP8, kT>(p, ws, plan, begin, end, sK, sV, k_full, k_empty, v_full, v_empty, tid - 128);
  } else {
    if (mb::elect_one()) {
      // ---------------------------------------------------------- products
      constexpr uint32_t kF = FP8 ? 0 : 1;
      constexpr uint32_t kIdS = mb::umma_idesc(kF, kF, 128, kT), kIdO = mb::umma_idesc(kF, kF, 128, D, 0, 1);
      const uint32_t aQ = mb::smem_u32(sQ), aK = mb::smem_u32(sK), aV = mb::smem_u32(sV);
      uint32_t part = 0, base = 0;
      bool ok = true;
      int pos = begin;
      Part x;
      auto scores = [&](uint32_t j) {
        if (!mb::mbar_wait(&k_full[j & 1], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_MMA)) return false;
        mb::tc_fence_after();
#pragma unroll
        for (int h = 0; h < kSpans; ++h)
#pragma unroll
          for (int s = 0; s < 4; ++s)
            mb::umma_f16(tmem + (j & 1) * kT, mb::umma_desc_sw128(aQ + h * (128 * 128) + s * 32),
                         mb::umma_desc_sw128(aK + (j & 1) * kTileB + h * (kT * 128) + s * 32), kIdS, (h | s) != 0);
        mb::tc_commit(&s_full[j & 1]);
        mb::tc_commit(&k_empty[j & 1]);
        return true;
      };
      while (ok && next_part<D>(plan, p.groups, ws.per_seq, pos, end, x)) {
        const int n = x.t1 - x.t0;
        ok = mb::mbar_wait(&q_full, part & 1, p.status, MB_ST_TIMEOUT_MMA) && scores(base);
        for (int i = 0; i < n && ok; ++i) {
          const uint32_t j = base + i, b = j & 1;
          if (i + 1 < n) {                                // over P of the tile before, whose product was issued in front
            ok = scores(j + 1);
            if (!ok) break;
          }
          ok = mb::mbar_wait(&v_full[b], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_MMA) && mb::mbar_wait(&p_full[b], (j >> 1) & 1, p.status, MB_ST_TIMEOUT_MMA);
          if (!ok) break;
          mb::tc_fence_after();
#pragma unroll
          for (int s = 0; s < kT / 16; ++s)
            umma_f16_ta(tmem + 256, tmem + b * kT + s * 8, mb::umma_desc_sw128_mn(aV + b * kTileB + s * 2048, kT * 128, 1024), kIdO, (i | s) != 0);
          mb::tc_commit(&v_empty[b]);
          mb::tc_commit(&o_done);
          if (i + 1 == n) mb::tc_commit(&o_full);
        }
        base += n;
        ++part;
      }
    }
    __syncwarp();
  }
  __syncthreads();
  if (warp == 8) {
    mb::tc_fence_after();
    mb::tmem_dealloc(tmem, 512);
  }
}

template <int D, bool FP8>
int launch_prefix(const MbSharedArgs& a, const Ws& ws, cudaStream_t stream) {
  static std::atomic<uint64_t> asked{0};
  if constexpr (D == 256) {
    auto kern = shared_prefix256_kernel<FP8>;
    constexpr int smem = 128 * D * 2 + 4 * 64 * D * 2 + 1024 + (int)sizeof(Plan);
    const cudaError_t e = mb::allow_smem(reinterpret_cast<const void*>(kern), smem, asked);
    if (e != cudaSuccess) return (int)e;
    return (int)mb::launch_kernel_ex(kern, dim3(ws.ctas), dim3(288), smem, stream, 1, mb_pdl_enabled() != 0, a, ws);
  } else {
    using C = PrefixCfg<D, FP8>;
    auto kern = shared_prefix_kernel<D, FP8>;
    Boxes boxes{0};
    while (a.block_size % (16 >> boxes.bits)) ++boxes.bits;
    constexpr uint32_t row = FP8 ? D : 2 * D, width = row < 128 ? row : 128;
    CUtensorMap tm[4];
    for (int i = 0; i < (FP8 ? 2 : 4); ++i) {
      const int rc = mbh::encode_3d(&tm[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, i & 1 ? a.v_cache : a.k_cache, row, a.Hkv, (uint64_t)a.num_blocks * a.block_size, row,
                                    (uint64_t)a.Hkv * row, width, 1, i < 2 ? 16 >> boxes.bits : 1,
                                    FP8 && i == 1 ? CU_TENSOR_MAP_SWIZZLE_NONE : width == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
      if (rc) return rc;
    }
    if (FP8) tm[2] = tm[3] = tm[0];                        // not used
    const cudaError_t e = mb::allow_smem(reinterpret_cast<const void*>(kern), C::kSmem, asked);
    if (e != cudaSuccess) return (int)e;
    return (int)mb::launch_kernel_ex(kern, dim3(ws.ctas), dim3(C::kThreads), C::kSmem, stream, 1, mb_pdl_enabled() != 0, tm[0], tm[1], tm[2], tm[3], boxes, a, ws);
  }
}

}  // namespace mbs
