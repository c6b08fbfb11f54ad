// A tile of 128 scores of a row, in registers, to weights: what the kernels of mla_prompt.cu and shared_prefix.cuh share. The running maximum moves only when a
// tile's is more than 2^8 above it.
//
// What bounds it is the special function units, 16 exponentials a cycle of an SM: 2048 cycles for two rows tiles, as long as their products take. So three pairs of
// eight are made on the multiply-add units instead: 2^x = 2^n 2^f with n the integer next to x, found by adding 1.5 * 2^23 (whose sum has n in its low
// bits), 2^f by a polynomial on [-1/2, 1/2] of the smallest largest relative error (Remez exchange), and n added to the exponent. Two of four cost about as
// much there as they save here.
#pragma once
#include "attention_rows.cuh"

namespace mbr {

// DEG 4: off by 2.7e-6 at most, 5: by 2.4e-7, next to what ex2 is
template <int DEG>
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  constexpr float c4[5] = {0.9999992847442627f, 0.6931217908859253f, 0.240247443318367f, 0.05591785907745361f, 0.009570102207362652f};
  constexpr float c5[6] = {1.0000001192092896f, 0.6931469440460205f, 0.24022120237350464f, 0.05550713092088699f, 0.009675540961325169f, 0.0013276472454890609f};
  const float2 magic = make_float2(12582912.f, 12582912.f);
  x.x = fmaxf(x.x, -126.f);                               // smaller ones become 2^-126: nothing beside the row's largest, which is 2^-8 or more
  x.y = fmaxf(x.y, -126.f);
  const float2 t = add2(x, magic), n = add2(t, make_float2(-12582912.f, -12582912.f));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  auto c = [&](int i) { return DEG == 4 ? make_float2(c4[i], c4[i]) : make_float2(c5[i], c5[i]); };
  float2 y = c(DEG);
#pragma unroll
  for (int i = DEG - 1; i >= 0; --i) y = fma2(y, f, c(i));
  return make_float2(__int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23)), __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23)));
}

// Scores of one row -> the first or second 64 weights 2^(s sc + nm), packed as the product's operand; `sum` grows by them. DEG 0: all by ex2
template <bool F16, int DEG>
__device__ __forceinline__ void half_weights(const float* s, float sc, float nm, uint32_t (&pk)[32], float2 (&sum)[2]) {
  const float2 sc2 = make_float2(sc, sc), nm2 = make_float2(nm, nm);
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    float2 t = fma2(make_float2(s[2 * i], s[2 * i + 1]), sc2, nm2);
    if (DEG > 0 && ((i & 7) == 1 || (i & 7) == 4 || (i & 7) == 6)) {
      t = exp2_poly<DEG == 0 ? 4 : DEG>(t);
    } else {
      t.x = ex2(t.x);
      t.y = ex2(t.y);
    }
    sum[i & 1] = add2(sum[i & 1], t);
    pk[i] = pack2<F16>(t.x, t.y);
  }
}

// max that keeps what is no number
__device__ __forceinline__ float max_nan(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
  return c;
}

// `lift`: log2 of what weights are held larger by. `first`: the row's first tile; `masked`: some scores are -inf by a mask. `rescale(alpha)`: the outputs so far
// times alpha, called by whole warps, never on a first tile. `publish(half, pk)`: 64 weights are ready.
template <bool F16, int DEG, typename Rescale, typename Publish>
__device__ __forceinline__ void softmax_tile(const float (&s)[128], float sc, float lift, bool first, bool masked, float& m_run, float& l_run, Rescale&& rescale,
                                             Publish&& publish) {
  float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
  for (int i = 4; i < 128; ++i) top[i & 3] = max_nan(top[i & 3], s[i]);
  float mx = max_nan(max_nan(top[0], top[1]), max_nan(top[2], top[3])) * sc;
  // scores that are no numbers, infinite ones, and rows that have seen nothing go the plain way, in which they stay visible and zeros are zeros
  const bool finite = mx < INFINITY;
  if (!finite && mx != INFINITY) {                        // the others' maximum
    float num[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 128; ++i) num[i & 3] = fmaxf(num[i & 3], s[i]);
    mx = fmaxf(fmaxf(num[0], num[1]), fmaxf(num[2], num[3])) * sc;
  }
  float alpha = 1.f;
  const bool move = mx > m_run + 8.f;                     // also true on a row's first finite tile
  if (move) {
    alpha = ex2(m_run - mx);                              // 0 when the row had seen nothing yet
    m_run = mx;
  }
  if (!first && __any_sync(0xffffffffu, move)) rescale(alpha);
  const float nm = m_run == -INFINITY ? 0.f : lift - m_run;
  uint32_t pk[32];
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  if (!masked && __all_sync(0xffffffffu, finite && m_run > -INFINITY)) {
    half_weights<F16, DEG>(s, sc, nm, pk, sum);
    publish(0, pk);
    half_weights<F16, DEG>(s + 64, sc, nm, pk, sum);
    publish(1, pk);
  } else {
    half_weights<F16, 0>(s, sc, nm, pk, sum);
    publish(0, pk);
    half_weights<F16, 0>(s + 64, sc, nm, pk, sum);
    publish(1, pk);
  }
  l_run = l_run * alpha + ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y));
}

}  // namespace mbr
