// Decode and verify attention of a batch whose sequences share long prefixes:
// z[j] = scale <q, k[j]> over the rows of the sequence's prefix (all of them) and its own (up to the token itself), out = softmax(z) v, lse = ln sum exp z.
#include "common.cuh"
#include "shared_attn.h"
#include "smem_limit.h"

namespace {

constexpr int kTile = 32, kThreads = 128;

__device__ __forceinline__ float load(const void* cache, size_t i, bool fp8) {
  return fp8 ? mb::e4m3_to_float(reinterpret_cast<const uint8_t*>(cache)[i]) : __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(cache)[i]);
}

__global__ void __launch_bounds__(kThreads) shared_simple_kernel(const MbSharedArgs p) {
  extern __shared__ float smem[];
  const int tok = blockIdx.x, kvh = blockIdx.y, tid = threadIdx.x, D = p.D, G = p.Hq / p.Hkv;
  float *sK = smem, *sV = sK + kTile * (D + 1), *sQ = sV + kTile * D, *sO = sQ + G * D, *sS = sO + G * D, *sM = sS + G * kTile, *sL = sM + G, *sA = sL + G;
  mb::pdl_wait();
  const int seq = tok / p.q_len, at = tok - seq * p.q_len;
  int prefix = 0, group = -1;
  {
    int start = 0;
    for (int g = 0, next = 0; g < p.groups; ++g) {
      const int a = p.group_start[g], b = p.group_start[g + 1];
      start = max(next, min(max(a, 0), p.num_seqs));
      next = max(start, min(max(b, 0), p.num_seqs));
      if (tid == 0 && p.status && (a < 0 || a > b || b > p.num_seqs)) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
      if (seq >= start && seq < next) group = g;
    }
  }
  if (group >= 0) prefix = max(p.prefix_len[group], 0);
  int own = max(p.ctx_len[seq], 0);
  if (prefix > p.max_prefix || own > p.max_ctx) {
    if (tid == 0 && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
    prefix = min(prefix, p.max_prefix);
    own = min(own, p.max_ctx);
  }
  own = max(0, own - p.q_len + at + 1);
  const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(p.q) + ((size_t)tok * p.Hq + kvh * G) * D;
  for (int i = tid; i < G * D; i += kThreads) {
    sQ[i] = __bfloat162float(q[i]);
    sO[i] = 0.f;
  }
  for (int g = tid; g < G; g += kThreads) {
    sM[g] = -INFINITY;
    sL[g] = 0.f;
  }
  __syncthreads();
  const float sc = p.scale * (p.fp8 ? *p.k_scale : 1.f);
  for (int side = 0; side < 2; ++side) {
    const int n = side ? own : prefix;
    const int* table = side ? p.block_table + (size_t)seq * p.table_ld : p.prefix_table + (size_t)max(group, 0) * p.prefix_ld;
    for (int j0 = 0; j0 < n; j0 += kTile) {
      const int m = min(kTile, n - j0);
      for (int i = tid; i < m * D; i += kThreads) {
        const int j = i / D, d = i - j * D, bi = (j0 + j) / p.block_size;
        int b = table[bi];
        if (b < 0 || b >= p.num_blocks) {
          if (p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
          b = 0;
        }
        const size_t from = (((size_t)b * p.block_size + (j0 + j - bi * p.block_size)) * p.Hkv + kvh) * D + d;
        sK[j * (D + 1) + d] = load(p.k_cache, from, p.fp8);
        sV[i] = load(p.v_cache, from, p.fp8);
      }
      __syncthreads();
      for (int i = tid; i < G * m; i += kThreads) {
        const int g = i / m, j = i - g * m;
        float z = 0.f;
        for (int d = 0; d < D; ++d) z += sQ[g * D + d] * sK[j * (D + 1) + d];
        sS[g * kTile + j] = z * sc;
      }
      __syncthreads();
      for (int g = tid; g < G; g += kThreads) {
        float mx = sM[g], sum = 0.f;
        for (int j = 0; j < m; ++j) mx = fmaxf(mx, sS[g * kTile + j]);
        const float base = mx == -INFINITY ? 0.f : mx, alpha = sM[g] == -INFINITY ? 0.f : expf(sM[g] - base);
        for (int j = 0; j < m; ++j) sum += sS[g * kTile + j] = expf(sS[g * kTile + j] - base);
        sL[g] = sL[g] * alpha + sum;
        sM[g] = mx;
        sA[g] = alpha;
      }
      __syncthreads();
      for (int i = tid; i < G * D; i += kThreads) {
        const int g = i / D, d = i - g * D;
        float o = sO[i] * sA[g];
        for (int j = 0; j < m; ++j) o += sS[g * kTile + j] * sV[j * D + d];
        sO[i] = o;
      }
      __syncthreads();
    }
  }
  const float vs = p.fp8 ? *p.v_scale : 1.f;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(p.out) + ((size_t)tok * p.Hq + kvh * G) * D;
  for (int i = tid; i < G * D; i += kThreads) {
    const float l = sL[i / D];
    out[i] = __float2bfloat16(l == 0.f ? 0.f : sO[i] * vs / l);
  }
  if (p.lse)
    for (int g = tid; g < G; g += kThreads) p.lse[(size_t)tok * p.Hq + kvh * G + g] = sL[g] == 0.f ? -INFINITY : sM[g] + logf(sL[g]);
}

bool bad_shape(const MbSharedArgs& a) {
  return a.num_seqs <= 0 || a.q_len <= 0 || a.Hkv <= 0 || a.Hkv > 65535 || a.Hq % a.Hkv || a.Hq / a.Hkv > 64 || (a.D != 64 && a.D != 128 && a.D != 256) ||
         a.block_size <= 0 || a.num_blocks <= 0 || a.max_prefix < 0 || a.max_ctx < 0 || !a.q || !a.k_cache || !a.v_cache || !a.ctx_len || !a.out ||
         (a.fp8 && (!a.k_scale || !a.v_scale)) || a.groups < 0 || (a.groups > 0 && (!a.prefix_table || !a.prefix_len || !a.group_start));
}

}  // namespace

extern "C" {

size_t mb_shared_attn_args(int which) {
  return which == 0 ? sizeof(MbSharedArgs) : which == 1 ? sizeof(MbMergeArgs) : which == 2 ? sizeof(MbMlaPromptArgs) : 0;
}

int mb_shared_attn(const MbSharedArgs* a, cudaStream_t stream) {
  if (!a || bad_shape(*a)) return MB_ERR_BAD_ARG;
  const int G = a->Hq / a->Hkv;
  const size_t smem = 4 * ((size_t)kTile * (2 * a->D + 1) + (size_t)G * (2 * a->D + kTile + 3));
  static std::atomic<uint64_t> asked{0};
  const cudaError_t e = mb::allow_smem(reinterpret_cast<const void*>(shared_simple_kernel), 220 * 1024, asked);
  if (e != cudaSuccess) return (int)e;
  return (int)mb::launch_kernel(shared_simple_kernel, dim3(a->num_seqs * a->q_len, a->Hkv), dim3(kThreads), smem, stream, *a);
}

}  // extern "C"
