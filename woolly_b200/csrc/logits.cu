// Rules applied to logits before sampling (sm_100a): penalties for repeated
// tokens, biases, grammar masks.
//
// With n_v the times token v occurs among the row's produced tokens (those of
// its history past the prompt, and the drafted tokens on its path) and "seen"
// for a token that occurs there or in the prompt:
//   y = x > 0 ? x / repetition : x * repetition     if seen, else x
//   y -= frequency * n_v + presence * (n_v > 0)
//   y += bias of v                                   (the last entry naming v)
//   y = -inf                                         if the row's mask has bit v clear
// in f32, rounded once to the logits' type.
//
// One CTA holds a run of the vocabulary of one row: a word of shared memory per
// token counts its occurrences (the top bit: seen in the prompt), a second one
// holds the last bias entry that names it; then the run streams through.  The
// counts are integers and the entry a maximum, so atomics' order is not seen.
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

constexpr int kLT = 512;        // threads
constexpr int kLChunk = 4096;   // tokens of the vocabulary per CTA
constexpr unsigned kPrompt = 0x80000000u;

__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ float get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

template <class T>
__global__ void __launch_bounds__(kLT) k_logits(const LogitArgs a) {
  __shared__ unsigned seen[kLChunk];
  __shared__ int entry[kLChunk];
  const int tid = threadIdx.x, r = blockIdx.x, v0 = blockIdx.y * kLChunk;
  const int nv = min(kLChunk, a.vocab - v0);
  pdl_wait();
  pdl_trigger();
  const wl_logit_context& c = a.ctx;
  const wl_logit_params p = a.params[r];
  for (int v = tid; v < nv; v += kLT) seen[v] = 0, entry[v] = -1;
  __syncthreads();
  const int req = c.requests ? c.requests[r] : r;
  const bool has = req >= 0 && req < c.n_history;
  if (has && c.history_start) {
    const int h0 = min(max(c.history_start[req], 0), c.history_total);
    const int h1 = min(max(c.history_start[req + 1], 0), c.history_total);
    const int np = c.prompt_lens ? c.prompt_lens[req] : 0;
    for (int h = h0 + tid; h < h1; h += kLT) {
      const unsigned v = (unsigned)c.history[h] - (unsigned)v0;
      if (v >= (unsigned)nv) continue;
      if (h - h0 < np) atomicOr(&seen[v], kPrompt);
      else atomicAdd(&seen[v], 1u);
    }
  }
  if (has && c.draft_mask) {
    const int row0 = c.row_start[req];
    for (int d = tid; d < 32 * c.words; d += kLT) {
      if (!(c.draft_mask[(size_t)r * c.words + (d >> 5)] >> (d & 31) & 1u)) continue;
      if (row0 < 0 || row0 + d >= a.rows) continue;
      const unsigned v = (unsigned)c.draft_tokens[row0 + d] - (unsigned)v0;
      if (v < (unsigned)nv) atomicAdd(&seen[v], 1u);
    }
  }
  if (c.bias_start) {
    const int b0 = min(max(c.bias_start[r], 0), c.bias_total), b1 = min(max(c.bias_start[r + 1], 0), c.bias_total);
    for (int b = b0 + tid; b < b1; b += kLT) {
      const unsigned v = (unsigned)c.bias_tokens[b] - (unsigned)v0;
      if (v < (unsigned)nv) atomicMax(&entry[v], b);
    }
  }
  __syncthreads();
  const unsigned* open = nullptr;
  if (c.allowed && p.allowed_row >= 0 && p.allowed_row < c.n_allowed)
    open = c.allowed + (size_t)p.allowed_row * c.allowed_words;
  const T* x = (const T*)a.logits + (size_t)r * a.ld;
  T* y = (T*)a.out + (size_t)r * a.ldo;
  for (int v = tid; v < nv; v += kLT) {
    float f = get(x + v0 + v);
    const unsigned s = seen[v];
    if (s) {
      f = f > 0.f ? f / p.repetition : f * p.repetition;
      const unsigned made = s & ~kPrompt;
      if (made) f -= p.frequency * (float)made + p.presence;
    }
    if (entry[v] >= 0) f += c.bias_values[entry[v]];
    if (open && !(open[(v0 + v) >> 5] >> ((v0 + v) & 31) & 1u)) f = -INFINITY;
    put(y + v0 + v, f);
  }
}

}  // namespace

int launch_logits(const LogitArgs& a, cudaStream_t st) {
  const dim3 grid(a.rows, (a.vocab + kLChunk - 1) / kLChunk);
  if (a.type == WL_F32) return launch_k(k_logits<float>, grid, dim3(kLT), 0, st, a);
  if (a.type == WL_F16) return launch_k(k_logits<__half>, grid, dim3(kLT), 0, st, a);
  return launch_k(k_logits<__nv_bfloat16>, grid, dim3(kLT), 0, st, a);
}

}  // namespace wl
