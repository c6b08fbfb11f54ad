// Attention that was computed in parts over disjoint keys, joined: lse = ln sum_i exp l_i, out = sum_i exp(l_i - lse) o_i. A part of weight zero (l_i = -inf)
// is not read, so what it holds does not matter; a row without weight gives zeros and -inf. One pass over the parts, bound by memory: a thread asks for the
// same 16 bytes of all parts, of ITEMS rows, before it uses any of them. Weights and sums are 32 bits. Five parts of 8191 x 32 rows of 128 fp32 dims
// (811 MB) take 125 us, 6.5 TB/s; 8 of 4096 x 40 bf16 58 us, 6.6 TB/s; 16 of 2048 x 40 bf16 77 us, 4.7 TB/s.
#include "common.cuh"
#include "shared_attn.h"
#include <type_traits>

namespace {

// V: elements a thread takes at once (16 bytes, or one where rows are no whole vectors); PARTS: most parts
template <typename T, int V, int PARTS, int ITEMS>
__global__ void __launch_bounds__(256) merge_kernel(const MbMergeArgs p) {
  using Vec = typename std::conditional<(V > 1), uint4, T>::type;
  const int per = p.dim / V;
  const long long total = p.rows * per, i0 = (long long)blockIdx.x * (256 * ITEMS) + threadIdx.x;
  mb::pdl_wait();
  float l[ITEMS][PARTS];
  Vec x[ITEMS][PARTS];
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const long long i = i0 + it * 256, row = i / per;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) l[it][k] = i < total && k < p.parts ? p.lses[k][row] : -INFINITY;
  }
#pragma unroll
  for (int it = 0; it < ITEMS; ++it)
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
      if (l[it][k] != -INFINITY) {
        const Vec* src = reinterpret_cast<const Vec*>(p.outs[k]) + i0 + it * 256;
        if constexpr (V > 1) x[it][k] = __ldcs(src);
        else x[it][k] = *src;
      }
#pragma unroll
  for (int it = 0; it < ITEMS; ++it) {
    const long long i = i0 + it * 256;
    if (i >= total) return;
    float top = -INFINITY, acc[V], sum = 0.f;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) top = fmaxf(top, l[it][k]);
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll
    for (int k = 0; k < PARTS; ++k) {
      if (l[it][k] == -INFINITY) continue;
      const float w = expf(l[it][k] - top);
      sum += w;
      const T* e = reinterpret_cast<const T*>(&x[it][k]);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += w * (float)e[j];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    Vec y;
    T* e = reinterpret_cast<T*>(&y);
#pragma unroll
    for (int j = 0; j < V; ++j) e[j] = (T)(acc[j] * inv);
    Vec* dst = reinterpret_cast<Vec*>(p.out) + i;
    if constexpr (V > 1) __stcs(dst, y);
    else *dst = y;
    const long long row = i / per;
    if (i == row * per) p.lse[row] = sum == 0.f ? -INFINITY : top + logf(sum);
  }
}

template <typename T, int V, int PARTS, int ITEMS>
int launch(const MbMergeArgs& a, cudaStream_t stream) {
  const long long n = (a.rows * (a.dim / V) + 256 * ITEMS - 1) / (256 * ITEMS);
  if (n > 0x7fffffffll) return MB_ERR_TOO_LARGE;
  return (int)mb::launch_kernel(merge_kernel<T, V, PARTS, ITEMS>, dim3((unsigned)n), dim3(256), 0, stream, a);
}

// What is in flight is a thread's loads times the threads, and registers bound the one by the other: five fp32 parts in the kernel of eight 135 us, of six 125,
// of six with two rows a thread 132; four parts with two rows 105, one 103; two parts of 8191 x 32 x 128 fp32 with one row 66, two 64; ten bf16 parts in a kernel
// of twelve 112, of sixteen 99.
template <typename T, int V>
int by_parts(const MbMergeArgs& a, cudaStream_t stream) {
  if (a.parts <= 2) return launch<T, V, 2, 2>(a, stream);
  if (a.parts <= 4) return launch<T, V, 4, 1>(a, stream);
  if (a.parts <= 6) return launch<T, V, 6, 1>(a, stream);
  if (a.parts <= 8) return launch<T, V, 8, 1>(a, stream);
  return launch<T, V, kMergeParts, 1>(a, stream);
}

template <typename T>
int run(const MbMergeArgs& a, cudaStream_t stream) {
  constexpr int kV = 16 / sizeof(T);
  uintptr_t low = reinterpret_cast<uintptr_t>(a.out) | (a.dim % kV ? 1 : 0);
  for (int k = 0; k < a.parts; ++k) low |= reinterpret_cast<uintptr_t>(a.outs[k]);
  return low & 15 ? by_parts<T, 1>(a, stream) : by_parts<T, kV>(a, stream);
}

}  // namespace

extern "C" int mb_merge_attn(const MbMergeArgs* a, cudaStream_t stream) {
  if (!a || a->rows <= 0 || a->dim <= 0 || a->parts < 1 || a->parts > kMergeParts || !a->out || !a->lse) return MB_ERR_BAD_ARG;
  return a->f32 ? run<float>(*a, stream) : run<__nv_bfloat16>(*a, stream);
}
