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
// One CTA takes a run of the vocabulary of one row or, when the rows are drafts
// of the same requests, of several: a word of shared memory per token counts its
// occurrences (top bits: seen in the prompt, has a bias), a second one holds the
// last bias entry that names it.  The history is counted once for the rows that
// share it; a row's path and biases are put in before its run streams through,
// four tokens at a time, and taken out after it.  The counts are integers and the
// entry a maximum, so atomics' order is not seen.
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
constexpr unsigned kPrompt = 0x80000000u, kBias = 0x40000000u;

__device__ __forceinline__ float get(const float* p) { return *p; }
__device__ __forceinline__ float get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// four values, 16 or 8 bytes
__device__ __forceinline__ void get4(const float* p, float* f) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}
template <class T>
__device__ __forceinline__ void get4(const T* p, float* f) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int e = 0; e < 4; e++) f[e] = get(h + e);
}
__device__ __forceinline__ void put4(float* p, const float* f) {
  *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
}
template <class T>
__device__ __forceinline__ void put4(T* p, const float* f) {
  uint2 v;
  T* h = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int e = 0; e < 4; e++) put(h + e, f[e]);
  *reinterpret_cast<uint2*>(p) = v;
}

// VEC: every row of four values is aligned
template <class T, bool VEC>
__global__ void __launch_bounds__(kLT) k_logits(const LogitArgs a, int per) {
  __shared__ __align__(16) unsigned seen[kLChunk];
  __shared__ __align__(16) int entry[kLChunk];
  constexpr int NV = kLChunk / kLT;  // tokens per thread
  const int tid = threadIdx.x, v0 = blockIdx.y * kLChunk, nv = min(kLChunk, a.vocab - v0);
  const int r0 = blockIdx.x * per, r1 = min(a.rows, r0 + per);
  pdl_wait();
  pdl_trigger();
  const wl_logit_context& c = a.ctx;
  // first token of the thread's g-th group of four (VEC), or its g-th token
  auto at = [&](int g) { return VEC ? (g * kLT + tid) * 4 : g * kLT + tid; };
  for (int i = tid * 4; i < kLChunk; i += kLT * 4) {
    *reinterpret_cast<uint4*>(seen + i) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<int4*>(entry + i) = make_int4(-1, -1, -1, -1);
  }
  int counted = -1;  // the request whose history `seen` holds
  for (int r = r0; r < r1; r++) {
    const wl_logit_params p = a.params[r];
    const T* x = (const T*)a.logits + (size_t)r * a.ld + v0;
    T* y = (T*)a.out + (size_t)r * a.ldo + v0;
    float f[NV];  // the row's logits are on their way while the counts are made
    if constexpr (VEC) {
#pragma unroll
      for (int g = 0; g < NV / 4; g++)
        if (at(g) + 4 <= nv) get4(x + at(g), f + 4 * g);
        else
          for (int e = 0; e < 4; e++) f[4 * g + e] = at(g) + e < nv ? get(x + at(g) + e) : 0.f;
    } else {
#pragma unroll
      for (int g = 0; g < NV; g++) f[g] = at(g) < nv ? get(x + at(g)) : 0.f;
    }
    int b0 = 0, b1 = 0;
    if (c.bias_start) {
      b0 = min(max(c.bias_start[r], 0), c.bias_total);
      b1 = min(max(c.bias_start[r + 1], 0), c.bias_total);
    }
    const int req = c.requests ? c.requests[r] : r;
    const bool has = req >= 0 && req < c.n_history;
    if (r == r0 || req != counted) {
      if (r != r0)
        for (int i = tid * 4; i < kLChunk; i += kLT * 4) *reinterpret_cast<uint4*>(seen + i) = make_uint4(0, 0, 0, 0);
      __syncthreads();
      counted = req;
      if (has && c.history_start) {
        const int h0 = min(max(c.history_start[req], 0), c.history_total);
        const int h1 = min(max(c.history_start[req + 1], 0), c.history_total);
        const int np = c.prompt_lens ? c.prompt_lens[req] : 0;
#pragma unroll 4
        for (int h = h0 + tid; h < h1; h += kLT) {
          const unsigned v = (unsigned)c.history[h] - (unsigned)v0;
          if (v >= (unsigned)nv) continue;
          if (h - h0 < np) atomicOr(&seen[v], kPrompt);
          else atomicAdd(&seen[v], 1u);
        }
      }
    }
    // the row's own tokens and biases: put in (add = 1), or taken out again
    auto own = [&](bool add) {
      if (has && c.draft_mask) {
        const int row0 = c.row_start[req];
        for (int d = tid; d < 32 * c.words; d += kLT) {
          if (!(c.draft_mask[(size_t)r * c.words + (d >> 5)] >> (d & 31) & 1u)) continue;
          if (row0 < 0 || row0 + d >= a.rows) continue;
          const unsigned v = (unsigned)c.draft_tokens[row0 + d] - (unsigned)v0;
          if (v < (unsigned)nv) atomicAdd(&seen[v], add ? 1u : ~0u);
        }
      }
      for (int b = b0 + tid; b < b1; b += kLT) {
        const unsigned v = (unsigned)c.bias_tokens[b] - (unsigned)v0;
        if (v >= (unsigned)nv) continue;
        if (add) {
          atomicMax(&entry[v], b);
          atomicOr(&seen[v], kBias);
        } else {
          entry[v] = -1;
          atomicAnd(&seen[v], ~kBias);
        }
      }
    };
    own(true);
    const unsigned* open = nullptr;
    if (c.allowed && p.allowed_row >= 0 && p.allowed_row < c.n_allowed)
      open = c.allowed + (size_t)p.allowed_row * c.allowed_words;
    __syncthreads();
    auto rules = [&](float x, unsigned s, int v) {
      if (s & ~kBias) {
        x = x > 0.f ? x / p.repetition : x * p.repetition;
        const unsigned made = s & ~(kPrompt | kBias);
        if (made) x -= p.frequency * (float)made + p.presence;
      }
      if (s & kBias) x += c.bias_values[entry[v]];
      return x;
    };
    if constexpr (VEC) {
#pragma unroll
      for (int g = 0; g < NV / 4; g++) {
        const int v = at(g);
        if (v >= nv) continue;
        const uint4 s = *reinterpret_cast<const uint4*>(seen + v);
        float* q = f + 4 * g;
        if (s.x | s.y | s.z | s.w) {
          q[0] = rules(q[0], s.x, v), q[1] = rules(q[1], s.y, v + 1);
          q[2] = rules(q[2], s.z, v + 2), q[3] = rules(q[3], s.w, v + 3);
        }
        if (open) {
          const unsigned bits = open[(v0 + v) >> 5] >> ((v0 + v) & 31);
#pragma unroll
          for (int e = 0; e < 4; e++) q[e] = bits >> e & 1u ? q[e] : -INFINITY;
        }
        if (v + 4 <= nv) put4(y + v, q);
        else
          for (int e = 0; v + e < nv; e++) put(y + v + e, q[e]);
      }
    } else {
#pragma unroll
      for (int g = 0; g < NV; g++) {
        const int v = at(g);
        if (v >= nv) continue;
        const unsigned s = seen[v];
        float z = s ? rules(f[g], s, v) : f[g];
        if (open && !(open[(v0 + v) >> 5] >> ((v0 + v) & 31) & 1u)) z = -INFINITY;
        put(y + v, z);
      }
    }
    if (r + 1 < r1) {
      __syncthreads();
      own(false);
      __syncthreads();
    }
  }
}

template <class T>
int launch_t(const LogitArgs& a, cudaStream_t st) {
  // drafted rows share their request's history: eight at a time count it once
  const int per = a.ctx.draft_mask ? 8 : 1;
  const dim3 grid((a.rows + per - 1) / per, (a.vocab + kLChunk - 1) / kLChunk);
  const size_t step = 4 * sizeof(T);
  const bool vec = !((reinterpret_cast<uintptr_t>(a.logits) | reinterpret_cast<uintptr_t>(a.out) |
                      a.ld * sizeof(T) | a.ldo * sizeof(T)) % step);
  return vec ? launch_step(k_logits<T, true>, grid, dim3(kLT), 0, st, a, per)
             : launch_step(k_logits<T, false>, grid, dim3(kLT), 0, st, a, per);
}

}  // namespace

int launch_logits(const LogitArgs& a, cudaStream_t st) {
  if (a.type == WL_F32) return launch_t<float>(a, st);
  if (a.type == WL_F16) return launch_t<__half>(a, st);
  return launch_t<__nv_bfloat16>(a, st);
}

}  // namespace wl
