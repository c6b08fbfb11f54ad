// A tile of 128 scores of a row in TMEM to weights, half by half: what shared_prefix.cuh makes of them. The running maximum moves only when a tile's is more than 2^8
// above it.
//
// What bounds it is the special function units, 16 exponentials a cycle of an SM. Exponentials of three pairs in eight by a polynomial on the multiply-add units
// (degree 5) were slower: 128 sequences behind 32768 e4m3 tokens 138 us in place of 123.
#pragma once
#include "attention_rows.cuh"

namespace mbr {

// The 128 scores of TMEM columns tS on become weights in the first 64 of these columns. The second half is read twice, for the maximum and for its
// weights: a whole row's scores in registers meant twice the code, and behind a short prefix much of a kernel's time is the fetching of its code.
// `seen`: columns from here on are masked. `lift`: log2 of what weights are held larger by. `first`: the row's first tile. `rescale(alpha)`: the outputs so far
// times alpha, called by whole warps, never on a first tile. `publish(half)`: 64 weights are there.
template <bool F16, typename Rescale, typename Publish>
__device__ __forceinline__ void softmax_tile(uint32_t tS, int seen, float sc, float lift, bool first, float& m_run, float& l_run, Rescale&& rescale, Publish&& publish) {
  const bool masked = !__all_sync(0xffffffffu, seen >= 128);
  float s[64];
  auto load = [&](int h) {
    mb::tmem_ld32_async(tS + h * 64, s);
    mb::tmem_ld32_async(tS + h * 64 + 32, s + 32);
    mb::tmem_ld_wait(s);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 64; ++i)
        if (h * 64 + i >= seen) s[i] = -INFINITY;
    }
  };
  float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
  for (int h = 1; h >= 0; --h) {
    load(h);
#pragma unroll
    for (int i = 0; i < 64; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
  }
  const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sc;
  float alpha = 1.f;
  const bool move = mx > m_run + 8.f;                     // also true on a row's first finite tile
  if (move) {
    alpha = ex2(m_run - mx);                              // 0 when the row had seen nothing yet
    m_run = mx;
  }
  if (!first && __any_sync(0xffffffffu, move)) rescale(alpha);
  const float nm = m_run == -INFINITY ? 0.f : lift - m_run;
  const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
  for (int h = 0; h < 2; ++h) {
    if (h > 0) load(h);
    uint32_t pk[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float2 t = fma2(make_float2(s[2 * i], s[2 * i + 1]), sc2, nm2);
      t.x = ex2(t.x);
      t.y = ex2(t.y);
      sum[i & 1] = add2(sum[i & 1], t);
      pk[i] = pack2<F16>(t.x, t.y);
    }
    tmem_st32(tS + h * 32, pk);
    mb::tmem_st_wait();
    publish(h);
  }
  l_run = l_run * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
}

}  // namespace mbr
