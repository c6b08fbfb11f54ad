// Prompts over a latent cache in expanded form: a cached row's keys and values are made for every head, k = [W_k c | rotated part], v = W_v c, and attended
// as usual. Per head and pair 192 + 128 multiply-adds instead of the 576 + 512 of the absorbed form, for 512 x 256 a cached row and head in front.
#include "common.cuh"
#include "shared_attn.h"
#include "smem_limit.h"

namespace {

constexpr int kRow = 576, kLat = 512, kQk = 192, kNope = 128, kV = 128;

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

__global__ void __launch_bounds__(256) gather_kernel(const GatherParams p) {
  mb::pdl_wait();
  __shared__ long long s_first[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long r0 = (long long)blockIdx.x * 128;
  if (tid == 0) {
    long long at = 0;
    int found = -1;
    for (int s = 0; s < p.num_seqs; ++s) {
      const int n = p.ctx_len[s], len = min(max(n, 0), p.max_ctx);
      const long long end = at + ((len + 127) & ~127);
      if (n > p.max_ctx || end > p.kv_rows)
        if (p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
      if (blockIdx.x == 0) p.first[s] = (int)min(at, p.kv_rows);
      if (r0 >= at && r0 < end) {
        found = s;
        s_first[1] = at;
      }
      at = end;
    }
    s_first[0] = found;
  }
  __syncthreads();
  const int s = (int)s_first[0];
  if (s < 0) return;
  const int j0 = (int)(r0 - s_first[1]), n = min(max(p.ctx_len[s], 0), p.max_ctx);
  int bad = 0x7fffffff;
  for (int r = warp; r < 128; r += 8) {
    const int j = j0 + r;
    uint4* dst = reinterpret_cast<uint4*>(p.lat + (r0 + r) * kRow);
    const uint4* src = nullptr;
    if (j < n) {
      int b = p.block_table[s * p.table_ld + j / p.block_size];
      if (b < 0 || b >= p.num_blocks) {
        if (lane == 0 && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
        b = 0;
      }
      src = reinterpret_cast<const uint4*>(p.cache + ((size_t)b * p.block_size + j % p.block_size) * kRow);
    }
    uint4 v[3];
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int c = lane + 32 * i;
      v[i] = src && c < kRow / 8 ? src[c] : make_uint4(0, 0, 0, 0);
      if (c < kLat / 8) {
        const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) odd |= (x[k] & 0x7f80u) == 0x7f80u || (x[k] & 0x7f800000u) == 0x7f800000u;
      }
    }
    odd = __any_sync(0xffffffffu, odd);
    if (odd) bad = min(bad, j);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int c = lane + 32 * i;
      if (c < kRow / 8) dst[c] = odd && c < kLat / 8 ? make_uint4(0, 0, 0, 0) : v[i];
    }
  }
  __shared__ int s_bad[8];
  if (lane == 0) s_bad[warp] = bad;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) bad = min(bad, s_bad[w]);
    p.bad[blockIdx.x] = bad;
  }
}

constexpr int kTile = 16, kRows = 16;

__global__ void __launch_bounds__(128) mla_simple_kernel(const MbMlaPromptArgs p) {
  __shared__ float sQ[kRows][kQk], sK[kTile][kQk + 1], sV[kTile][kV], sS[kRows][kTile], sM[kRows], sL[kRows], sA[kRows];
  const int s = blockIdx.z, h = blockIdx.y, tid = threadIdx.x;
  mb::pdl_wait();
  const int qlen = p.q_len[s], qs = p.q_start[s], ctx = min(max(p.ctx_len[s], 0), p.max_ctx), t0 = blockIdx.x * kRows;
  const long long first = p.first[s];
  if (t0 >= qlen) return;
  if (qlen > p.max_q_len || qs < 0 || (long long)qs + qlen > p.q_rows || first + ctx > p.kv_rows) {
    if (tid == 0 && p.status) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
    return;
  }
  const int rows = min(kRows, qlen - t0), past = ctx - qlen;
  for (int i = tid; i < rows * kQk; i += 128)
    sQ[i / kQk][i % kQk] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.q)[((size_t)(qs + t0 + i / kQk) * p.H + p.head0 + h) * kQk + i % kQk]) * p.scale;
  if (tid < kRows) {
    sM[tid] = -INFINITY;
    sL[tid] = 0.f;
  }
  float o[kRows];
#pragma unroll
  for (int r = 0; r < kRows; ++r) o[r] = 0.f;
  const int last = past + t0 + rows;
  int bad = 0x7fffffff;
  for (int j = 0; j < last; j += 128) bad = min(bad, p.bad[(first + j) / 128]);
  __syncthreads();
  for (int j0 = 0; j0 < last; j0 += kTile) {
    const int m = min(kTile, last - j0);
    for (int i = tid; i < m * 320; i += 128) {
      const int j = i / 320, d = i % 320;
      const size_t row = first + j0 + j;
      if (d < 64) sK[j][kNope + d] = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.lat)[row * kRow + kLat + d]);
      else {
        const float x = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.kv)[(row * p.heads + h) * 256 + d - 64]);
        if (d < 192) sK[j][d - 64] = x;
        else sV[j][d - 192] = x;
      }
    }
    __syncthreads();
    for (int i = tid; i < rows * m; i += 128) {
      const int r = i / m, j = i % m;
      float z = 0.f;
      for (int d = 0; d < kQk; ++d) z += sQ[r][d] * sK[j][d];
      sS[r][j] = j0 + j < past + t0 + r + 1 ? z : -INFINITY;
    }
    __syncthreads();
    if (tid < rows) {
      float mx = sM[tid], sum = 0.f;
      for (int j = 0; j < m; ++j) mx = fmaxf(mx, sS[tid][j]);
      const float base = mx == -INFINITY ? 0.f : mx;
      sA[tid] = sM[tid] == -INFINITY ? 0.f : expf(sM[tid] - base);
      for (int j = 0; j < m; ++j) sum += sS[tid][j] = expf(sS[tid][j] - base);
      sL[tid] = sL[tid] * sA[tid] + sum;
      sM[tid] = mx;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      if (r >= rows) break;
      o[r] *= sA[r];
      for (int j = 0; j < m; ++j) o[r] += sS[r][j] * sV[j][tid];
    }
    __syncthreads();
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
    if (r < rows)
      reinterpret_cast<__nv_bfloat16*>(p.out)[((size_t)(qs + t0 + r) * p.H + p.head0 + h) * kV + tid] =
          __float2bfloat16(past + t0 + r + 1 > bad ? __int_as_float(0x7fffffff) : sL[r] == 0.f ? 0.f : o[r] / sL[r]);
}

}  // namespace

extern "C" {

int mb_mla_gather(const void* cache, const int* block_table, long long table_ld, const int* ctx_len, void* lat, int* first, int* bad, uint32_t* status,
                  long long num_blocks, long long kv_rows, int num_seqs, int block_size, int max_ctx, cudaStream_t stream) {
  if (!cache || !block_table || !ctx_len || !lat || !first || !bad || num_blocks <= 0 || kv_rows <= 0 || kv_rows % 128 || num_seqs <= 0 || block_size <= 0 || max_ctx <= 0)
    return MB_ERR_BAD_ARG;
  GatherParams p{(const __nv_bfloat16*)cache, block_table, table_ld, ctx_len, (__nv_bfloat16*)lat, first, bad, status, num_blocks, kv_rows, num_seqs, block_size, max_ctx};
  return (int)mb::launch_kernel(gather_kernel, dim3((unsigned)(kv_rows / 128)), dim3(256), 0, stream, p);
}

int mb_mla_prompt(const MbMlaPromptArgs* a, cudaStream_t stream) {
  if (!a || !a->q || !a->kv || !a->lat || !a->q_start || !a->q_len || !a->ctx_len || !a->first || !a->bad || !a->out || a->num_seqs <= 0 || a->num_seqs > 65535 ||
      a->H <= 0 || a->heads <= 0 || a->heads > 65535 || a->head0 < 0 || a->head0 + a->heads > a->H || a->max_q_len <= 0 || a->max_ctx <= 0)
    return MB_ERR_BAD_ARG;
  return (int)mb::launch_kernel(mla_simple_kernel, dim3((a->max_q_len + kRows - 1) / kRows, a->heads, a->num_seqs), dim3(128), 0, stream, *a);
}

}  // extern "C"
