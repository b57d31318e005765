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
// Most tokens of a row are open and unseen: they are copied, or closed, in one
// pass over the row that asks for nothing but the mask.  The others are few.  One
// CTA takes a run of the vocabulary of one row or, when the rows are drafts of the
// same requests, of eight: a word of shared memory per token counts its
// occurrences in the history (top bit: seen in the prompt), once for the rows that
// share it, and whoever turns a token's word from zero puts the token on a list.
// The tokens of each row's path and its biases that fall into the run make a
// second, short list.  Then a thread per (row, listed token) works out its value
// from the logit that the copy left in place, adding what the row's short list has
// to say about it; all rows of a request at once, so that the few dependent loads
// are paid once and not row by row.  A row whose short list does not fit marks its
// tokens in shared memory instead, and goes by itself.
// Counts are integers and of a token's biases the last holds, so atomics' order is
// not seen.
//
// Bound by the copy: 384 drafted rows of 128,000 f32 logits (395 MB) take 119 us =
// 3.3 TB/s, 51% of the measured copy rate; with every token going through the
// rules' branches it was 195 us, row by row with the short lists as marks 187 us.
// What is left is the passes over the listed tokens, which follow the CTA's whole
// copy, at two CTAs per SM.  16 rows of 32,000 take 6.4 us.
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
constexpr int kLRows = 8;       // most rows per CTA
constexpr int kLOwn = 64;       // path and bias tokens of a row that its list holds
constexpr unsigned kPrompt = 0x80000000u;

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
__global__ void __launch_bounds__(kLT, 2) k_logits(const LogitArgs a, int per) {
  __shared__ __align__(16) unsigned seen[kLChunk];
  __shared__ __align__(16) int entry[kLChunk];
  __shared__ unsigned short list[kLChunk];
  __shared__ int s_req[kLRows], s_first[kLRows], s_b0[kLRows], s_b1[kLRows];
  __shared__ wl_logit_params s_prm[kLRows];
  __shared__ int2 own[kLRows][kLOwn];  // (token, bias entry, or -1 for a node of the path)
  __shared__ int s_own[kLRows];        // how many there are
  __shared__ int s_n;                  // listed tokens
  constexpr int NV = kLChunk / kLT;  // tokens per thread
  const int tid = threadIdx.x, v0 = blockIdx.y * kLChunk, nv = min(kLChunk, a.vocab - v0);
  const int r0 = blockIdx.x * per, nr = min(per, a.rows - r0);
  pdl_wait();
  pdl_trigger();
  const wl_logit_context& c = a.ctx;
  for (int i = tid * 4; i < kLChunk; i += kLT * 4) {
    *reinterpret_cast<uint4*>(seen + i) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<int4*>(entry + i) = make_int4(-1, -1, -1, -1);
  }
  if (tid == 0) s_n = 0;
  if (tid < nr) {
    const int r = r0 + tid, req = c.requests ? c.requests[r] : r;
    const bool has = req >= 0 && req < c.n_history;
    s_prm[tid] = a.params[r];
    s_req[tid] = has ? req : -1;
    s_own[tid] = 0;
    s_first[tid] = has && c.draft_mask ? c.row_start[req] : -1;
    s_b0[tid] = c.bias_start ? min(max(c.bias_start[r], 0), c.bias_total) : 0;
    s_b1[tid] = c.bias_start ? min(max(c.bias_start[r + 1], 0), c.bias_total) : 0;
  }
  __syncthreads();
  auto mask_of = [&](int k) {
    const int m = s_prm[k].allowed_row;
    return c.allowed && m >= 0 && m < c.n_allowed ? c.allowed + (size_t)m * c.allowed_words : nullptr;
  };

  // the copy; its loads run ahead of its stores by four rows
  if constexpr (VEC) {
    constexpr int G = NV / 4;
    const int at = tid * 4;
    float f0[NV], f1[NV], f2[NV], f3[NV];
    auto load = [&](int k, float (&q)[NV]) {
      if (k >= nr) return;
      const T* x = (const T*)a.logits + (size_t)(r0 + k) * a.ld + v0;
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int v = at + g * kLT * 4;
        if (v + 4 <= nv) {
          get4(x + v, q + 4 * g);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++) q[4 * g + e] = v + e < nv ? get(x + v + e) : 0.f;
        }
      }
    };
    auto store = [&](int k, float (&q)[NV]) {
      if (k >= nr) return;
      const unsigned* open = mask_of(k);
      T* y = (T*)a.out + (size_t)(r0 + k) * a.ldo + v0;
#pragma unroll
      for (int g = 0; g < G; g++) {
        const int v = at + g * kLT * 4;
        if (v >= nv) continue;
        if (open) {
          const unsigned bits = open[(v0 + v) >> 5] >> ((v0 + v) & 31);
#pragma unroll
          for (int e = 0; e < 4; e++) q[4 * g + e] = bits >> e & 1u ? q[4 * g + e] : -INFINITY;
        }
        if (v + 4 <= nv) {
          put4(y + v, q + 4 * g);
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (v + e < nv) put(y + v + e, q[4 * g + e]);
        }
      }
    };
    load(0, f0), load(1, f1), load(2, f2), load(3, f3);
#pragma unroll 1
    for (int k = 0; k < nr; k += 4) {
      store(k, f0), load(k + 4, f0);
      store(k + 1, f1), load(k + 5, f1);
      store(k + 2, f2), load(k + 6, f2);
      store(k + 3, f3), load(k + 7, f3);
    }
  } else {
    for (int k = 0; k < nr; k++) {
      const unsigned* open = mask_of(k);
      const T* x = (const T*)a.logits + (size_t)(r0 + k) * a.ld + v0;
      T* y = (T*)a.out + (size_t)(r0 + k) * a.ldo + v0;
      float f[NV];
#pragma unroll
      for (int g = 0; g < NV; g++) f[g] = g * kLT + tid < nv ? get(x + g * kLT + tid) : 0.f;
#pragma unroll
      for (int g = 0; g < NV; g++) {
        const int v = g * kLT + tid;
        if (v >= nv) continue;
        put(y + v, open && !(open[(v0 + v) >> 5] >> ((v0 + v) & 31) & 1u) ? -INFINITY : f[g]);
      }
    }
  }

  // the rows' own tokens that fall into this run, kLT / per threads to a row
  {
    const int k = tid / (kLT / per), t = tid % (kLT / per);
    auto note = [&](unsigned token, int b) {
      const unsigned v = token - (unsigned)v0;
      if (v >= (unsigned)nv) return;
      const int e = atomicAdd(&s_own[k], 1);
      if (e < kLOwn) own[k][e] = make_int2((int)v, b);
    };
    if (k < nr) {
      const int row0 = s_first[k];
      if (row0 >= 0)
        for (int d = t; d < 32 * c.words && d < a.rows - row0; d += kLT / per)
          if (c.draft_mask[(size_t)(r0 + k) * c.words + (d >> 5)] >> (d & 31) & 1u) note(c.draft_tokens[row0 + d], -1);
#pragma unroll 4
      for (int b = s_b0[k] + t; b < s_b1[k]; b += kLT / per) note(c.bias_tokens[b], b);
    }
  }
  // seen: word of the token, made: times on the row's path, b: its bias entry
  auto apply = [&](int k, int v, unsigned w, unsigned made, int b) {
    const wl_logit_params& p = s_prm[k];
    const unsigned* open = mask_of(k);
    if (open && !(open[(v0 + v) >> 5] >> ((v0 + v) & 31) & 1u)) return;
    T* y = (T*)a.out + (size_t)(r0 + k) * a.ldo + v0 + v;
    float z = get(y);
    made += w & ~kPrompt;
    if (w | made) z = z > 0.f ? z / p.repetition : z * p.repetition;
    if (made) z -= p.frequency * (float)made + p.presence;
    if (b >= 0) z += c.bias_values[b];
    put(y, z);
  };
  for (int k0 = 0, k1; k0 < nr; k0 = k1) {
    const int req = s_req[k0];
    for (k1 = k0 + 1; k1 < nr && s_req[k1] == req; k1++) {
    }
    if (k0 > 0) {  // another history
      __syncthreads();
      for (int i = tid * 4; i < kLChunk; i += kLT * 4) *reinterpret_cast<uint4*>(seen + i) = make_uint4(0, 0, 0, 0);
      if (tid == 0) s_n = 0;
      __syncthreads();
    }
    if (req >= 0 && c.history_start) {
      const int h0 = min(max(c.history_start[req], 0), c.history_total);
      const int h1 = min(max(c.history_start[req + 1], 0), c.history_total);
      const int np = c.prompt_lens ? c.prompt_lens[req] : 0;
#pragma unroll 4
      for (int h = h0 + tid; h < h1; h += kLT) {
        const unsigned v = (unsigned)c.history[h] - (unsigned)v0;
        if (v >= (unsigned)nv) continue;
        const unsigned was = h - h0 < np ? atomicOr(&seen[v], kPrompt) : atomicAdd(&seen[v], 1u);
        if (was == 0) list[atomicAdd(&s_n, 1)] = (unsigned short)v;
      }
    }
    __syncthreads();  // the list, the rows' own and their copies are complete
    const int n = s_n;
    for (int i = tid; i < n * (k1 - k0); i += kLT) {
      const int k = k0 + i / n, v = list[i % n], m = s_own[k];
      if (m > kLOwn) continue;
      unsigned made = 0;
      int b = -1;
      for (int e = 0; e < m; e++)
        if (own[k][e].x == v) {
          made += own[k][e].y < 0;
          b = max(b, own[k][e].y);
        }
      apply(k, v, seen[v], made, b);
    }
    // own tokens that the history does not have: the first of several speaks for the token
    for (int i = tid; i < kLOwn * (k1 - k0); i += kLT) {
      const int k = k0 + i / kLOwn, j = i % kLOwn, m = s_own[k];
      if (m > kLOwn || j >= m) continue;
      const int v = own[k][j].x;
      bool mine = seen[v] == 0;
      unsigned made = 0;
      int b = -1;
      for (int e = 0; e < m && mine; e++)
        if (own[k][e].x == v) {
          mine = e >= j;
          made += own[k][e].y < 0;
          b = max(b, own[k][e].y);
        }
      if (mine) apply(k, v, 0, made, b);
    }
    for (int k = k0; k < k1; k++) {
      if (s_own[k] <= kLOwn) continue;
      // marks: path counts go into the words, the last bias entry beside them
      const int row0 = s_first[k];
      auto marks = [&](bool add) {
        if (row0 >= 0)
          for (int d = tid; d < 32 * c.words && d < a.rows - row0; d += kLT) {
            if (!(c.draft_mask[(size_t)(r0 + k) * c.words + (d >> 5)] >> (d & 31) & 1u)) continue;
            const unsigned v = (unsigned)c.draft_tokens[row0 + d] - (unsigned)v0;
            if (v < (unsigned)nv) atomicAdd(&seen[v], add ? 1u : ~0u);
          }
        for (int b = s_b0[k] + tid; b < s_b1[k]; b += kLT) {
          const unsigned v = (unsigned)c.bias_tokens[b] - (unsigned)v0;
          if (v >= (unsigned)nv) continue;
          if (add) atomicMax(&entry[v], b);
          else entry[v] = -1;
        }
      };
      __syncthreads();  // every reader of the words is done
      marks(true);
      __syncthreads();
      for (int v = tid; v < nv; v += kLT)
        if (seen[v] || entry[v] >= 0) apply(k, v, seen[v], 0, entry[v]);
      __syncthreads();
      marks(false);
    }
  }
}

template <class T>
int launch_t(const LogitArgs& a, cudaStream_t st) {
  // drafted rows share their request's history: a CTA counts it once for up to
  // eight, as many as leave two CTAs per SM.  384 rows of 128,000 take 118 us with
  // eight, 304 with one; 128 of 32,000 take 27 us with two, 28 with one, 48 with eight.
  const int runs = (a.vocab + kLChunk - 1) / kLChunk;
  int per = a.ctx.draft_mask ? kLRows : 1;
  while (per > 1 && (long long)((a.rows + per - 1) / per) * runs < 2 * 148) per /= 2;
  const dim3 grid((a.rows + per - 1) / per, runs);
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
