// Decode and verify attention of a batch whose sequences share long prefixes:
// z[j] = scale <q, k[j]> over the rows of the sequence's prefix (all of them) and its own (up to the token itself), out = softmax(z) v, lse = ln sum exp z.
//
// What has no need of the rest is computed on its own: all rows behind a prefix over that prefix, which is read once for all of them (shared_prefix.cuh),
// and every token over what its sequence has of its own (the decode kernel, attention_decode_parts.cu). Either leaves outputs relative to 2^m, m and sums,
// and the join here adds them up. The decode kernel comes up under the prefix kernel and does not wait for it until its end, so that the two share the GPU.
// No atomics on results: every partial one has one writer, and the join adds them in an order that follows from the plan (below).
#include "attention_decode_parts.h"
#include "shared_prefix.cuh"

namespace {

using namespace mbs;

constexpr size_t kOwnBytes = size_t(512) << 20;            // most bytes of own rows' partial results: more tokens go in several steps

Ws workspace(const MbSharedArgs& a) {
  Ws w{};
  const size_t rows = (size_t)a.num_seqs * a.q_len * (a.Hq / a.Hkv), all = rows * a.Hkv, tokens = (size_t)a.num_seqs * a.q_len;
  w.ctas = a.sm_count > 0 ? a.sm_count : 148;
  w.G = a.Hq / a.Hkv;
  w.per_seq = a.q_len * w.G;
  auto take = [&](size_t bytes) {
    const size_t at = w.bytes;
    w.bytes += (bytes + 255) & ~size_t(255);
    return at;
  };
  if (a.groups > 0 && a.max_prefix > 0) {
    const size_t sides = a.D == 256 ? 1 : 2;
    w.first = take(sides * all * a.D * 4);
    w.first_ml = take(sides * all * 8);
    w.rest = take((size_t)w.ctas * 2 * kRowTile * a.D * 4);
    w.rest_ml = take((size_t)w.ctas * 2 * kRowTile * 8);
  }
  if (a.max_ctx > 0) {
    const int part = part_tokens_of(a.Hkv, a.D);
    const long long n = ((long long)a.max_ctx + part - 1) / part;
    w.parts = n > kMaxOwnParts ? kMaxOwnParts : (int)n;
    const size_t each = (size_t)a.Hq * w.parts * (a.D * 4 + 8);
    size_t step = kOwnBytes / each;
    step = step < 1 ? 1 : step > (size_t)kMaxTokens ? (size_t)kMaxTokens : step;
    if (step > tokens) step = tokens;
    w.step = (int)step;
    w.own = take(step * a.Hq * w.parts * a.D * 4);
    w.own_ml = take(step * a.Hq * w.parts * 8);
  } else {
    w.step = tokens < size_t(1) << 20 ? (int)tokens : 1 << 20;
  }
  return w;
}

// 32 rows (tokens x heads of a group) of a kv head and 32 dims at a time, lane = row. A row's partial results (a prefix's, of single units all first sides in
// front of all second ones, then its own) are dealt out to the eight warps, each of which sums every eighth and asks for maximum, sum and dims together; the
// warps' sums are joined in shared memory from warp 0 to 7. Few rows have many parts, and their latencies do not add up.
// Bound by latency: 2 to 3 us a unit, of which the first begin before the kernels in front are through. As many CTAs as fit walk the units: with a CTA for
// each, many of them came up late to plan again (the whole call 89.2 us instead of 87.2 for 128 sequences, 53.3 instead of 50.1 for 64 tokens behind 5000).
constexpr int kJoinDims = 32, kJoinCtas = 3;

template <int D, bool FP8>
__global__ void __launch_bounds__(256, kJoinCtas) shared_join_kernel(const MbSharedArgs p, const Ws ws, int tok0, int tokens) {
  __shared__ Plan plan;
  __shared__ float4 s_o[8][kJoinDims / 4][32];
  __shared__ float2 s_ml[8][32];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = ws.G;
  constexpr int kC = kJoinDims / 4, kCuts = D / kJoinDims;
  // What is planned by stood before the kernels in front, which have waited for it before they let this one come up: only what they write is waited for
  const bool prefixes = p.groups > 0 && p.max_prefix > 0;
  if (prefixes) {
    if (warp == 0) make_plan<D>(p, plan, ws.per_seq, lane);
    __syncthreads();
  }
  const int part_tokens = part_tokens_of(p.Hkv, D), blocks = (tokens * G + 31) / 32, units = blocks * p.Hkv * kCuts;
  bool waited = false;
#pragma unroll 1
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int kvh = u / kCuts % p.Hkv, c0 = u % kCuts * kC;  // fours of dims
    const int R = u / (kCuts * p.Hkv) * 32 + lane;         // of the step's rows
    const bool live = R < tokens * G;
    const int step_tok = live ? R / G : 0, head = live ? R - step_tok * G : 0, tok = tok0 + step_tok, seq = tok / p.q_len;
    float m = -INFINITY, l = 0.f;
    float4 acc[kC];
#pragma unroll
    for (int c = 0; c < kC; ++c) acc[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float2* pml, const float4* px, size_t pitch) {
      const float2 ml = __ldcg(pml);
      float4 x[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) x[c] = __ldcg(px + c * pitch);
      const bool none = ml.y == 0.f;                       // nothing seen: what lies there does not count
      const float mn = none ? m : fmaxf(m, ml.x), base = mn == -INFINITY ? 0.f : mn;    // all scores NaN leave no maximum, but a sum that is NaN
      const float fa = m == -INFINITY ? 0.f : ex2(m - base), fb = ml.x == -INFINITY ? 1.f : ex2(ml.x - base);
      m = mn;
      if (none) return;
      l = l * fa + ml.y * fb;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        acc[c].x = acc[c].x * fa + x[c].x * fb;
        acc[c].y = acc[c].y * fa + x[c].y * fb;
        acc[c].z = acc[c].z * fa + x[c].z * fb;
        acc[c].w = acc[c].w * fa + x[c].w * fb;
      }
    };
    int own_parts = 0;                                     // asked for beside the prefix's parts
    if (live && p.max_ctx > 0) {
      const int own = max(0, min(max(p.ctx_len[seq], 0), p.max_ctx) - p.q_len + (tok - seq * p.q_len) + 1);
      own_parts = own > 0 ? own_part_count(own, part_tokens) : 0;
    }
    if (!waited) mb::pdl_wait();
    waited = true;
    int at_warp = warp;                                    // this warp's next part of those that come
    if (live && prefixes && seq >= plan.start[0] && seq < plan.start[p.groups]) {
      int lo = 0, hi = p.groups;                           // start[lo] <= seq < start[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (plan.start[mid] <= seq) lo = mid;
        else hi = mid;
      }
      const int rows = row_count(plan, lo, ws.per_seq), tiles = (plan.len[lo] + Shape<D>::kT - 1) / Shape<D>::kT;
      if (tiles > 0) {
        const int row = (tok - plan.start[lo] * p.q_len) * G + head;
        int doubles, singles;
        unit_count<D>(rows, doubles, singles);
        const int W = plan.base[p.groups];
        const Share share(W, used_ctas(W, ws.ctas));
        const int two = row < doubles * 256, v = two ? row >> 8 : (row - doubles * 256) >> 7;
        const int at = plan.base[lo] + kvh * line_of_head<D>(rows, tiles) + (two ? 2 * tiles * v : (2 * doubles + v) * tiles);
        const int side = two ? (row >> 7) & 1 : 0, sides = two || D == 256 ? 1 : 2;
        const int cta0 = share.owner(at), ctas = share.owner(at + ((tiles - 1) << two)) - cta0 + 1, n = ctas * sides;      // first sides in front
        for (; at_warp < n; at_warp += 8) {
          const int k = at_warp >= ctas, c = cta0 + at_warp - k * ctas;
          int t0, t1;
          tiles_in(at, tiles, two, share.first(c), share.first(c + 1), t0, t1);
          if (t1 - t0 <= k) continue;                        // of one tile the second side has nothing (8 rows behind 700: 16.9 us, 18.5 with it read)
          const Place from = t0 == 0 ? place_first<D>(p, ws, plan, lo, kvh, row, k) : place_rest<D>(p, ws, c, two ? side : k);
          const int r = t0 == 0 ? 0 : row & 127;
          add(from.ml + r, from.o + c0 * from.pitch + r, from.pitch);
        }
        at_warp -= n;
      }
    }
    const size_t own_at = ((size_t)step_tok * p.Hq + kvh * G + head) * ws.parts;
    for (; at_warp < own_parts; at_warp += 8) {
      const size_t at = own_at + at_warp;
      add(reinterpret_cast<const float2*>(reinterpret_cast<const uint8_t*>(p.ws) + ws.own_ml) + at,
          reinterpret_cast<const float4*>(reinterpret_cast<const uint8_t*>(p.ws) + ws.own) + at * (D / 4) + c0, 1);
    }
    s_ml[warp][lane] = make_float2(m, l);
#pragma unroll
    for (int c = 0; c < kC; ++c) s_o[warp][c][lane] = acc[c];
    __syncthreads();
    // warp w sums dims 4 w to 4 w + 3 of the 32 rows
    float mx = -INFINITY;
    float2 ml[8];
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      ml[w] = s_ml[w][lane];
      if (ml[w].y != 0.f) mx = fmaxf(mx, ml[w].x);
    }
    const float base = mx == -INFINITY ? 0.f : mx;
    float sum = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      if (ml[w].y == 0.f) continue;
      const float f = ml[w].x == -INFINITY ? 1.f : ex2(ml[w].x - base);
      const float4 x = s_o[w][warp][lane];
      sum += ml[w].y * f;
      y.x += x.x * f; y.y += x.y * f; y.z += x.z * f; y.w += x.w * f;
    }
    const float inv = sum == 0.f ? 0.f : (FP8 ? *p.v_scale : 1.f) / sum;
    const uint2 out = make_uint2(pack2<false>(y.x * inv, y.y * inv), pack2<false>(y.z * inv, y.w * inv));
    const float lse = sum == 0.f ? -INFINITY : (base + log2f(sum)) * 0.693147180559945f;
    if (live) {
      const size_t row = (size_t)tok * p.Hq + kvh * G + head;
      *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.out) + row * D + (c0 + warp) * 4) = out;
      if (p.lse && warp == 0 && c0 == 0) p.lse[row] = lse;
    }
    __syncthreads();                                       // the next unit's sums take these places
  }
  // Lengths and groups are looked at by the kernels in front, which a maximum of 0 leaves out: what is beyond that is reported here
  if (blockIdx.x == 0 && tok0 == 0 && p.status) {
    bool beyond = false;
    if (p.max_ctx == 0)
      for (int s = tid; s < p.num_seqs; s += 256) beyond |= p.ctx_len[s] > 0;
    if (p.max_prefix == 0)
      for (int g = tid; g < p.groups; g += 256) {
        const int a = p.group_start[g], b = p.group_start[g + 1];
        beyond |= a < 0 || b > p.num_seqs || b < a || (b > a && p.prefix_len[g] > 0);
      }
    if (beyond) atomicCAS(p.status, 0u, MB_ST_BOUNDS);
  }
}

bool bad_shape(const MbSharedArgs& a) {
  return a.num_seqs <= 0 || a.q_len <= 0 || a.Hkv <= 0 || a.Hkv > 65535 || a.Hq % a.Hkv || a.Hq / a.Hkv > 64 || (a.D != 64 && a.D != 128 && a.D != 256) ||
         a.block_size <= 0 || a.num_blocks < 0 || a.num_blocks * a.block_size >= (1ll << 31) || a.table_ld >= (1ll << 31) || a.max_prefix < 0 || a.max_ctx < 0 ||
         ((a.max_prefix > 0 || a.max_ctx > 0) && (a.num_blocks == 0 || !a.k_cache || !a.v_cache)) || !a.q || !a.ctx_len || !a.out ||
         (a.fp8 && (!a.k_scale || !a.v_scale)) || a.groups < 0 || a.groups > kMaxGroups || (a.groups > 0 && ((a.max_prefix > 0 && !a.prefix_table) || !a.prefix_len || !a.group_start)) ||
         ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k_cache) | reinterpret_cast<uintptr_t>(a.v_cache) | reinterpret_cast<uintptr_t>(a.out)) & 15);
}

template <int D, bool FP8>
int run(const MbSharedArgs& a, const Ws& w, cudaStream_t stream) {
  const int tokens = a.num_seqs * a.q_len, G = a.Hq / a.Hkv;
  const bool prefixes = a.groups > 0 && a.max_prefix > 0;
  if (prefixes)
    if (const int rc = launch_prefix<D, FP8>(a, w, stream)) return rc;
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.ws);
  for (int t = 0; t < tokens; t += w.step) {
    const int n = tokens - t < w.step ? tokens - t : w.step;
    // only the first step stands directly behind the prefix kernel; a later one's results take the place of what the join in front reads
    if (a.max_ctx > 0)
      if (const int rc = mb_decode_parts(a, t, n, reinterpret_cast<float*>(ws + w.own), reinterpret_cast<float*>(ws + w.own_ml), w.parts, prefixes && t == 0, stream)) return rc;
    // a CTA takes several units rather than to come up late and plan again
    const long long units = ((long long)n * G + 31) / 32 * a.Hkv * (D / kJoinDims), most = (long long)w.ctas * kJoinCtas;
    const cudaError_t e = mb::launch_kernel_ex(shared_join_kernel<D, FP8>, dim3((unsigned)(units < most ? units : most)), dim3(256), 0, stream, 1, mb_pdl_enabled() != 0, a, w, t, n);
    if (e != cudaSuccess) return (int)e;
  }
  return 0;
}

}  // namespace

extern "C" {

size_t mb_shared_attn_args(int which) {
  return which == 0 ? sizeof(MbSharedArgs) : which == 1 ? sizeof(MbMergeArgs) : which == 2 ? sizeof(MbMlaPromptArgs) : 0;
}

size_t mb_shared_attn_ws(int num_seqs, int q_len, int groups, int Hq, int Hkv, int D, int max_prefix, int max_ctx, int sm_count) {
  if (num_seqs <= 0 || q_len <= 0 || Hkv <= 0 || Hq < Hkv) return 0;
  MbSharedArgs a{};
  a.num_seqs = num_seqs; a.q_len = q_len; a.groups = groups; a.Hq = Hq; a.Hkv = Hkv; a.D = D; a.max_prefix = max_prefix; a.max_ctx = max_ctx; a.sm_count = sm_count;
  return workspace(a).bytes;
}

int mb_shared_attn(const MbSharedArgs* a, cudaStream_t stream) {
  if (!a || bad_shape(*a)) return MB_ERR_BAD_ARG;
  const long long G = a->Hq / a->Hkv, rows = (long long)a->num_seqs * a->q_len * G;
  if (rows * a->Hkv > (1ll << 26)) return MB_ERR_TOO_LARGE;
  // places of the line that prefixes are shared out along, at most (shared_plan.cuh)
  const long long units = rows / 128 + (a->groups < a->num_seqs ? a->groups : a->num_seqs);
  if (a->groups > 0 && (units + 1) * a->Hkv * (a->max_prefix / (a->D == 256 ? 64 : 128) + 1) >= (1ll << 31)) return MB_ERR_TOO_LARGE;
  const Ws w = workspace(*a);
  if (w.bytes > 0 && (!a->ws || a->ws_bytes < w.bytes)) return MB_ERR_TOO_LARGE;
  switch (a->D) {
    case 64: return a->fp8 ? run<64, true>(*a, w, stream) : run<64, false>(*a, w, stream);
    case 128: return a->fp8 ? run<128, true>(*a, w, stream) : run<128, false>(*a, w, stream);
    default: return a->fp8 ? run<256, true>(*a, w, stream) : run<256, false>(*a, w, stream);
  }
}

}  // extern "C"
