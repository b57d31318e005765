// Attention of a step's rows over the paged cache (sm_100a).
//
// Row r is token or drafted node j of request i (row_start[i] + j = r), at
// position pos[r].  It attends the request's lengths[i] cached tokens and, of
// the step's own rows (their K and V lie at tokens lengths[i] + c), those whose
// mask bit is set; without masks the nodes c <= j, a chain.  Scores are
// q.k * scale, the window W keeps keys at positions > pos[r] - W, and
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s).
// A row with nothing to attend, or with a negative position, gives zeros.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <string>

#include "common.h"
#include "kernels.cuh"
#include "pdl.cuh"

namespace wl {
namespace {

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// ---------------------------------------------------------------- one (row, head) per CTA
template <class Q, class C>
__global__ void __launch_bounds__(128) k_tree_attn_row(const TreeAttnArgs a) {
  __shared__ float s_q[256], s_p[128], s_red[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x, head = blockIdx.y, hd = a.head_dim, kvh = head / (a.heads / a.kv_heads);
  pdl_wait();
  pdl_trigger();
  if (r >= a.row_start[a.n]) return;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.row_start[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  const int i = lo, row0 = a.row_start[i], T = a.row_start[i + 1] - row0;
  const int pos = a.pos[r], len = max(a.lengths[i], 0);
  const Q* q = (const Q*)a.q + (size_t)r * a.ldq + (size_t)head * hd;
  for (int d = tid; d < hd; d += 128) s_q[d] = as_f32(q[d]);
  __syncthreads();
  const int keys = pos < 0 ? 0 : (int)min((long long)len + T, (long long)a.max_pages * kKvPage);
  float m = -INFINITY, l = 0.f, o[2] = {0.f, 0.f};
  for (int t0 = 0; t0 < keys; t0 += 128) {
    const int t = t0 + tid;
    float s = -INFINITY;
    if (t < keys) {
      bool ok = true;
      int at = t;
      if (t >= len) {
        const int c = t - len;
        ok = a.mask ? c < 32 * a.words && (a.mask[(size_t)r * a.words + (c >> 5)] >> (c & 31) & 1u) : c <= r - row0;
        at = a.pos[row0 + c];
      }
      if (a.window > 0) ok = ok && at > pos - a.window;
      const int page = ok ? a.tables[(size_t)i * a.ld_tables + t / kKvPage] : -1;
      if (page >= 0 && page < a.n_pages) {
        const C* k = (const C*)a.cache_k + (((size_t)page * a.kv_heads + kvh) * kKvPage + t % kKvPage) * hd;
        float acc = 0.f;
        for (int d = 0; d < hd; d++) acc += s_q[d] * as_f32(k[d]);
        s = acc * a.scale;
      }
    }
    float mx = s;
    for (int x = 16; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
    if (lane == 0) s_red[warp] = mx;
    __syncthreads();
    const float mn = fmaxf(fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3])), m);
    const float alpha = m == -INFINITY ? 0.f : expf(m - mn);
    const float p = s == -INFINITY ? 0.f : expf(s - mn);
    m = mn;
    s_p[tid] = p;
    float sum = p;
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    __syncthreads();
    if (lane == 0) s_red[warp] = sum;
    __syncthreads();
    l = l * alpha + s_red[0] + s_red[1] + s_red[2] + s_red[3];
    for (int e = 0, d = tid; d < hd; d += 128, e++) {
      float acc = o[e] * alpha;
      for (int t = 0; t < 128 && t0 + t < keys; t++) {
        if (s_p[t] == 0.f) continue;
        const int page = a.tables[(size_t)i * a.ld_tables + (t0 + t) / kKvPage];
        acc += s_p[t] * as_f32(((const C*)a.cache_v)[(((size_t)page * a.kv_heads + kvh) * kKvPage +
                                                      (t0 + t) % kKvPage) * hd + d]);
      }
      o[e] = acc;
    }
    __syncthreads();
  }
  Q* out = (Q*)a.out + ((size_t)r * a.heads + head) * hd;
  for (int e = 0, d = tid; d < hd; d += 128, e++) put(out + d, l > 0.f ? o[e] / l : 0.f);
}

}  // namespace

size_t tree_attention_workspace(int, int, int, int, int, int) { return 0; }

int launch_tree_attention(const TreeAttnArgs& a, cudaStream_t st) {
  const dim3 grid(a.rows, a.heads);
  if (a.q_type == WL_F32) return launch_k(k_tree_attn_row<float, __half>, grid, dim3(128), 0, st, a);
  if (a.q_type == WL_F16) return launch_k(k_tree_attn_row<__half, __half>, grid, dim3(128), 0, st, a);
  return launch_k(k_tree_attn_row<__nv_bfloat16, __nv_bfloat16>, grid, dim3(128), 0, st, a);
}

}  // namespace wl
