// Attention that was computed in parts over disjoint keys, joined: lse = ln sum_i exp l_i, out = sum_i exp(l_i - lse) o_i. A part of weight zero (l_i = -inf)
// is not read, so what it holds does not matter; a row without weight gives zeros and -inf. One pass over the parts, a thread a vector of 16 bytes of a row.
#include "common.cuh"
#include "shared_attn.h"

namespace {

// V: elements a thread takes at once (16 bytes, or one where rows are no whole vectors)
template <typename T, int V>
__global__ void __launch_bounds__(256) merge_kernel(const MbMergeArgs p) {
  const int per = p.dim / V;
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  mb::pdl_wait();
  if (i >= p.rows * per) return;
  const long long row = i / per;
  const int c = (int)(i - row * per);
  float l[kMergeParts], top = -INFINITY;
#pragma unroll
  for (int k = 0; k < kMergeParts; ++k) {
    l[k] = k < p.parts ? p.lses[k][row] : -INFINITY;
    top = fmaxf(top, l[k]);
  }
  float acc[V], total = 0.f;
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll
  for (int k = 0; k < kMergeParts; ++k) {
    if (k >= p.parts || l[k] == -INFINITY) continue;
    const float w = expf(l[k] - top);
    total += w;
    T x[V];
    if constexpr (V > 1) *reinterpret_cast<uint4*>(x) = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p.outs[k]) + row * p.dim) + c);
    else x[0] = reinterpret_cast<const T*>(p.outs[k])[row * p.dim + c];
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] += w * (float)x[j];
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T y[V];
#pragma unroll
  for (int j = 0; j < V; ++j) y[j] = (T)(acc[j] * inv);
  if constexpr (V > 1) reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + row * p.dim)[c] = *reinterpret_cast<uint4*>(y);
  else reinterpret_cast<T*>(p.out)[row * p.dim + c] = y[0];
  if (c == 0) p.lse[row] = total == 0.f ? -INFINITY : top + logf(total);
}

template <typename T>
int run(const MbMergeArgs& a, cudaStream_t stream) {
  constexpr int kV = 16 / sizeof(T);
  uintptr_t low = reinterpret_cast<uintptr_t>(a.out) | (a.dim % kV ? 1 : 0);
  for (int k = 0; k < a.parts; ++k) low |= reinterpret_cast<uintptr_t>(a.outs[k]);
  const bool wide = !(low & 15);
  const long long n = (a.rows * (wide ? a.dim / kV : a.dim) + 255) / 256;
  if (n > 0x7fffffffll) return MB_ERR_TOO_LARGE;
  return wide ? (int)mb::launch_kernel(merge_kernel<T, kV>, dim3((unsigned)n), dim3(256), 0, stream, a)
              : (int)mb::launch_kernel(merge_kernel<T, 1>, dim3((unsigned)n), dim3(256), 0, stream, a);
}

}  // namespace

extern "C" int mb_merge_attn(const MbMergeArgs* a, cudaStream_t stream) {
  if (!a || a->rows <= 0 || a->dim <= 0 || a->parts < 1 || a->parts > kMergeParts || !a->out || !a->lse) return MB_ERR_BAD_ARG;
  return a->f32 ? run<float>(*a, stream) : run<__nv_bfloat16>(*a, stream);
}
