// The weight that a prompt's last tokens give to what is cached: mass[s, h, j] += sum over observed rows r of p[r, j], p = softmax of the
// causal logits of the group's queries. K is read, V is not; the prompt's outputs are the prefill kernels' business.
//
// Two passes over the logits: the first leaves every observed row's maximum and sum, the second adds up the weights of a tile of keys over all
// rows. Every output has one writer, and sums have one order.
#include "common.cuh"
#include "kv_mass.h"

namespace {

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// observed rows of a sequence, and its cached tokens; a length beyond what the call was sized for is reported and cut
struct Span {
  int n, q_len, rows, q0;      // cached tokens, tokens of the portion, observed rows (tokens x group), first observed token
};
__device__ __forceinline__ Span span_of(const MbMassArgs& a, int s, int G) {
  Span x;
  x.n = a.ctx_len[s];
  x.q_len = a.q_len[s];
  if (x.n > a.max_ctx || x.q_len > a.max_q_len) {
    if (a.status && threadIdx.x == 0) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
    x.n = min(x.n, a.max_ctx);
    x.q_len = min(x.q_len, a.max_q_len);
  }
  x.n = max(x.n, 0);
  x.q_len = max(x.q_len, 0);
  if (a.q_start[s] < 0 || a.q_start[s] + (long long)x.q_len > a.q_rows) {
    if (a.status && threadIdx.x == 0) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
    x.q_len = 0;
  }
  const int seen = min(a.last, x.q_len);
  x.q0 = x.q_len - seen;
  x.rows = seen * G;
  return x;
}

template <bool FP8>
__device__ __forceinline__ float logit(const MbMassArgs& a, const float* q, long long at) {
  float acc = 0.f;
  for (int d = 0; d < a.D; ++d)
    acc += q[d] * (FP8 ? mb::e4m3_to_float(reinterpret_cast<const uint8_t*>(a.k_cache)[at + d])
                       : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.k_cache)[at + d]));
  return acc;
}
__device__ __forceinline__ long long row_at(const MbMassArgs& a, int s, int h, int j) {
  const int bi = j / a.block_size;
  int b = __ldg(a.block_table + s * a.table_ld + bi);
  if ((unsigned)b >= (unsigned long long)a.num_blocks) {
    if (a.status) atomicCAS(a.status, 0u, MB_ST_BOUNDS);
    b = 0;
  }
  return (((long long)b * a.block_size + (j - bi * a.block_size)) * a.Hkv + h) * a.D;
}

// One warp an observed row: log2 of its sum, in the log2 domain. Row r is token r / G of the observed ones, head r % G of the group.
template <bool FP8>
__global__ void __launch_bounds__(256) observe_rows_kernel(const MbMassArgs a, int max_rows) {
  __shared__ float sq[8][256];
  const int G = a.Hq / a.Hkv, h = blockIdx.y, s = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.x * 8 + warp;
  const Span x = span_of(a, s, G);
  if (r >= x.rows) return;
  const int tok = x.q0 + r / G, limit = min(x.n, x.n - x.q_len + tok + 1);
  const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + ((size_t)(a.q_start[s] + tok) * a.Hq + h * G + r % G) * a.D;
  for (int d = lane; d < a.D; d += 32) sq[warp][d] = __bfloat162float(q[d]);
  __syncwarp();
  const float sc = a.scale * (FP8 ? *a.k_scale : 1.f) * 1.44269504088896f;
  float m = -INFINITY, l = 0.f;
  for (int j = lane; j < limit; j += 32) {
    const float z = logit<FP8>(a, sq[warp], row_at(a, s, h, j)) * sc, mx = fmaxf(m, z);
    const float use = mx == -INFINITY ? 0.f : mx;
    l = l * ex2(m - use) + ex2(z - use);
    m = mx;
  }
  const float top = mb::warp_max(m), use = top == -INFINITY ? 0.f : top;
  l = mb::warp_sum(l * ex2(m - use));
  if (lane == 0) reinterpret_cast<float*>(a.ws)[((size_t)s * a.Hkv + h) * max_rows + r] = l == 0.f ? INFINITY : top + log2f(l);
}

// One thread a cached token: its weights over all observed rows.
template <bool FP8>
__global__ void __launch_bounds__(128) observe_keys_kernel(const MbMassArgs a, int max_rows) {
  __shared__ float sq[256];
  const int G = a.Hq / a.Hkv, h = blockIdx.y, s = blockIdx.z, j = blockIdx.x * 128 + threadIdx.x;
  const Span x = span_of(a, s, G);
  if (blockIdx.x * 128 >= x.n) return;
  const float sc = a.scale * (FP8 ? *a.k_scale : 1.f) * 1.44269504088896f;
  const float* lse = reinterpret_cast<const float*>(a.ws) + ((size_t)s * a.Hkv + h) * max_rows;
  const long long at = j < x.n ? row_at(a, s, h, j) : 0;
  float sum = 0.f;
  for (int r = 0; r < x.rows; ++r) {
    const int tok = x.q0 + r / G, limit = x.n - x.q_len + tok + 1;
    const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + ((size_t)(a.q_start[s] + tok) * a.Hq + h * G + r % G) * a.D;
    __syncthreads();
    for (int d = threadIdx.x; d < a.D; d += 128) sq[d] = __bfloat162float(q[d]);
    __syncthreads();
    if (j < limit && j < x.n) sum += ex2(logit<FP8>(a, sq, at) * sc - lse[r]);
  }
  if (j < x.n) a.mass[s * a.mass_seq + h * a.mass_head + j] += sum;
}

template <bool FP8>
int launch(const MbMassArgs& a, int max_rows, cudaStream_t stream) {
  observe_rows_kernel<FP8><<<dim3((max_rows + 7) / 8, a.Hkv, a.num_seqs), 256, 0, stream>>>(a, max_rows);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return (int)e;
  observe_keys_kernel<FP8><<<dim3((a.max_ctx + 127) / 128, a.Hkv, a.num_seqs), 128, 0, stream>>>(a, max_rows);
  return (int)cudaGetLastError();
}

}  // namespace

extern "C" {

size_t mb_prompt_mass_ws(int num_seqs, int Hq, int seen) { return (size_t)num_seqs * Hq * seen * 4; }

int mb_prompt_mass(const MbMassArgs* a, cudaStream_t stream) {
  if (!a || a->num_seqs <= 0 || a->num_seqs > 65535 || a->Hkv <= 0 || a->Hkv > 65535 || a->Hq % a->Hkv || (a->D != 64 && a->D != 128 && a->D != 256) ||
      a->block_size <= 0 || a->num_blocks <= 0 || a->max_ctx <= 0 || a->last <= 0 || a->last > a->max_q_len || !a->q || !a->k_cache || !a->block_table ||
      !a->q_start || !a->q_len || !a->ctx_len || !a->mass || (a->fp8 && !a->k_scale))
    return MB_ERR_BAD_ARG;
  const size_t need = mb_prompt_mass_ws(a->num_seqs, a->Hq, a->last);
  if (!a->ws || a->ws_bytes < need) return MB_ERR_TOO_LARGE;
  const long long max_rows = (long long)a->last * (a->Hq / a->Hkv);
  if (max_rows > (1ll << 30)) return MB_ERR_TOO_LARGE;
  return a->fp8 ? launch<true>(*a, (int)max_rows, stream) : launch<false>(*a, (int)max_rows, stream);
}

}  // extern "C"
