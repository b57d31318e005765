// Block tables, slot maps and cache writes of a serving step (sm_100a).
//
// Pages hold 16 tokens; token p of a request lies in page table[p / 16] at
// offset p % 16, its slot being page * 16 + p % 16.  Free pages form a stack
// (its top at the end).  A step adds counts[i] tokens to request i, which holds
// lengths[i]: need_i = ceil((L + c) / 16) - ceil(L / 16) pages come off the
// stack in request order, page g of the step being free[top - 1 - g].  Giving
// pages back pushes page g of the call to free[top + total - 1 - g], so a step
// taken back leaves the stack as it was.
//
// Both are prefix sums over the requests (one CTA, 1024 requests a round, sums
// in 64 bits) and a scatter over the rows, which starts from a binary search of
// the rows' prefix sums.  Latency is all there is to them: 64 requests of one
// token 4.2 us, 32 trees of up to 64 tokens 9.3 us, 1024 prompts of 314,000 rows
// 8.6 us (graph replays).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <string>

#include "common.h"
#include "kernels.cuh"
#include "pdl.cuh"

namespace wl {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kPlanRows = 2048;  // rows that the scan's CTA places itself

__device__ __forceinline__ long long pages_of(long long tokens) { return (tokens + kKvPage - 1) / kKvPage; }

// inclusive prefix sum over the CTA's threads; `total` is the sum of all
__device__ __forceinline__ long long block_scan(long long v, long long* red, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += y;
  }
  __syncthreads();  // red may still be read from the previous scan
  if (lane == 31) red[warp] = v;
  __syncthreads();
  long long w = red[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const long long before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
  return v + (warp ? before : 0);
}

__device__ __forceinline__ long long block_min(long long v, long long* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const long long y = __shfl_xor_sync(0xffffffffu, v, o);
    v = y < v ? y : v;
  }
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = red[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const long long y = __shfl_xor_sync(0xffffffffu, v, o);
    v = y < v ? y : v;
  }
  return v;
}

// What a row needs of the requests: in global memory, or in shared memory where
// the CTA that made it places the rows too.
struct PlanView {
  const int* row_start;   // [n + 1]
  const int* page_start;  // [n]
  const int* held;        // [n] tokens before the step
  const int* status;      // [n]
  const int* parents;     // [rows]
};

// One row of the step: its request, position and slot, the page it is the
// first on, and the mask of its node's path.
__device__ __forceinline__ void plan_row(const PlanArgs& a, const PlanView& q, int r, int total, int top) {
  int req = -1, pos = -1, slot = -1;
  bool walk = false;
  int i = 0, j = 0;
  if (r < total) {
    int lo = 0, hi = a.n - 1;  // the request whose rows hold r: the first with row_start[i + 1] > r
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (q.row_start[mid + 1] > r) hi = mid;
      else lo = mid + 1;
    }
    i = req = lo;
    j = r - q.row_start[i];
    if (q.status[i] == 0) {
      const int len = q.held ? q.held[i] : a.out.lengths[i] - a.counts[i];
      const int p = len + j, idx = p / kKvPage, held = (int)pages_of(len);
      int* entry = a.tables + (size_t)i * a.ld_tables + idx;
      int page;
      if (idx >= held) {
        page = a.free_pages[top - 1 - (q.page_start[i] + idx - held)];
        if (p % kKvPage == 0) *entry = page;
      } else {
        page = *entry;
      }
      pos = p;
      if (page >= 0 && page < INT_MAX / kKvPage) slot = page * kKvPage + p % kKvPage;
      walk = q.parents != nullptr;
    }
  }
  if (a.words > 0) {
    // the path from the row's node to the root; indices fall strictly, so each
    // word of the mask is written once, highest first
    unsigned* m = a.out.mask + (size_t)r * a.words;
    int w = a.words - 1;
    unsigned acc = 0;
    if (walk) {
      const int* parents = q.parents + (r - j);
      int node = j, depth = 0;
      while (true) {
        const int nw = node >> 5;
        while (w > nw) m[w--] = acc, acc = 0;
        acc |= 1u << (node & 31);
        depth++;
        const int up = parents[node];
        if (up < -1 || up >= node) {  // not an earlier node: the row is left out
          walk = false;
          break;
        }
        if (up < 0) break;
        node = up;
      }
      if (walk) {
        pos += depth - 1 - j;
      } else {
        pos = slot = -1;
        acc = 0;
        w = a.words - 1;
      }
    }
    while (w >= 0) m[w--] = acc, acc = 0;
  }
  a.out.requests[r] = req;
  a.out.positions[r] = pos;
  a.out.slots[r] = slot;
}

// with_rows: the rows too (a.n <= kPlanThreads, a.rows <= kPlanRows)
__global__ void __launch_bounds__(kPlanThreads) k_plan(const PlanArgs a, int with_rows) {
  __shared__ long long red[kPlanWarps];
  __shared__ int s_row[kPlanThreads + 1], s_page[kPlanThreads], s_held[kPlanThreads], s_status[kPlanThreads];
  __shared__ int s_parents[kPlanRows];
  const int tid = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  const int top = max(0, min(*a.free_count, a.free_cap));
  const long long limit = (long long)a.max_pages * kKvPage;
  long long rows_done = 0, pages_done = 0, cut = LLONG_MAX;
  for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const bool in = i < a.n;
    const int len = in ? a.lengths[i] : 0, cnt = in ? a.counts[i] : 0;
    const int ext = max(cnt, 0);
    long long sum;
    const long long row_end = rows_done + block_scan(ext, red, sum);
    rows_done += sum;
    int status = 0;
    if (len < 0 || cnt < 0 || (a.words > 0 && cnt > 32 * a.words)) status = WL_STEP_BAD_REQUEST;
    else if ((long long)len + cnt > limit) status = WL_STEP_TABLE_FULL;
    else if (row_end > a.rows) status = WL_STEP_NO_ROWS;
    const int need = in && status == 0 ? (int)(pages_of((long long)len + cnt) - pages_of(len)) : 0;
    const long long page_end = pages_done + block_scan(need, red, sum);
    pages_done += sum;
    const bool out_of_pages = need > 0 && page_end > top;
    if (out_of_pages) status = WL_STEP_NO_PAGES;
    // the pool is handed out up to the first request that it cannot serve
    const long long first = block_min(out_of_pages ? page_end - need : LLONG_MAX, red);
    cut = first < cut ? first : cut;
    if (in) {
      const long long row0 = row_end - ext, page0 = page_end - need;
      if (with_rows) {
        s_row[tid] = (int)(row0 < a.rows ? row0 : a.rows);
        s_page[tid] = (int)(page0 < cut ? page0 : cut);
        s_held[tid] = len;
        s_status[tid] = status;
      }
      a.out.row_start[i] = (int)(row0 < a.rows ? row0 : a.rows);
      a.out.page_start[i] = (int)(page0 < cut ? page0 : cut);
      a.out.status[i] = status;
      a.out.lengths[i] = status == 0 ? len + cnt : len;
    }
  }
  const int taken = (int)(pages_done < cut ? pages_done : cut);
  const int total = (int)(rows_done < a.rows ? rows_done : a.rows);
  __syncthreads();  // every thread has read free_count, which free_left may be
  if (tid == 0) {
    a.out.row_start[a.n] = total;
    a.out.page_start[a.n] = taken;
    *a.out.free_count = top - taken;
  }
  if (!with_rows) return;
  if (tid == 0) s_row[a.n] = total;
  if (a.parents)
    for (int r = tid; r < a.rows; r += kPlanThreads) s_parents[r] = a.parents[r];
  __syncthreads();
  const PlanView q = {s_row, s_page, s_held, s_status, a.parents ? s_parents : nullptr};
  for (int r = tid; r < a.rows; r += kPlanThreads) plan_row(a, q, r, total, top);
}

__global__ void __launch_bounds__(256) k_plan_rows(const PlanArgs a) {
  pdl_wait();
  pdl_trigger();
  const int total = a.out.row_start[a.n];
  const int top = *a.out.free_count + a.out.page_start[a.n];
  const int r = blockIdx.x * 256 + threadIdx.x;
  const PlanView q = {a.out.row_start, a.out.page_start, nullptr, a.out.status, a.parents};
  if (r < a.rows) plan_row(a, q, r, total, top);
}

constexpr int kOwnPages = 8;

__global__ void __launch_bounds__(kPlanThreads) k_release(const ReleaseArgs a) {
  __shared__ long long red[kPlanWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  const int top = max(0, min(*a.free_count, a.free_cap));
  const long long limit = (long long)a.max_pages * kKvPage;
  long long done = 0, cut = LLONG_MAX;
  for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int i = i0 + tid;
    const bool in = i < a.n;
    const int len = in ? a.lengths[i] : 0, keep = in ? min(a.keep[i], len) : 0;
    int status = len < 0 || keep < 0 || len > limit ? WL_STEP_BAD_REQUEST : 0;
    const int p0 = status ? 0 : (int)pages_of(keep), p1 = status ? 0 : (int)pages_of(len);
    // a thread looks at its request's first pages, a warp together at the rest
    {
      const int* row = a.tables + (size_t)i * a.ld_tables;
      bool hole = false;
#pragma unroll
      for (int q = 0; q < kOwnPages; q++)
        if (p0 + q < p1) hole |= row[p0 + q] < 0;
      if (hole) status = WL_STEP_TABLE_FULL;
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, p1 > p0 + kOwnPages); todo; todo &= todo - 1) {
      const int src = __ffs(todo) - 1;
      const int q0 = __shfl_sync(0xffffffffu, p0, src) + kOwnPages, q1 = __shfl_sync(0xffffffffu, p1, src);
      const int* row = a.tables + (size_t)(i0 + warp * 32 + src) * a.ld_tables;
      bool hole = false;
      for (int q = q0 + lane; q < q1; q += 32) hole |= row[q] < 0;
      if (__any_sync(0xffffffffu, hole) && lane == src) status = WL_STEP_TABLE_FULL;
    }
    const int give = status == 0 ? p1 - p0 : 0;
    long long sum;
    const long long end = done + block_scan(give, red, sum);
    done += sum;
    const bool full = give > 0 && end > (long long)a.free_cap - top;
    if (full) status = WL_STEP_NO_PAGES;
    const long long first = block_min(full ? end - give : LLONG_MAX, red);
    cut = first < cut ? first : cut;
    if (in) {
      const long long at = end - give;
      a.out.page_start[i] = (int)(at < cut ? at : cut);
      a.out.status[i] = status;
    }
  }
  const int total = (int)(done < cut ? done : cut);
  __syncthreads();
  if (tid == 0) {
    a.out.page_start[a.n] = total;
    *a.out.free_count = top + total;
  }
  for (int i = warp; i < a.n; i += kPlanWarps) {
    const int len = a.lengths[i], at = a.out.page_start[i];
    int kept = len;
    if (a.out.status[i] == 0) {
      kept = min(a.keep[i], len);
      const int p0 = (int)pages_of(kept), give = (int)pages_of(len) - p0;
      int* row = a.tables + (size_t)i * a.ld_tables + p0;
      for (int g = lane; g < give; g += 32) {
        a.free_pages[top + total - 1 - (at + g)] = row[g];
        row[g] = -1;
      }
    }
    __syncwarp();  // every lane has read lengths[i], which out.lengths may be
    if (lane == 0) a.out.lengths[i] = kept;
  }
}

// ---------------------------------------------------------------- cache writes
template <class T>
struct Eight;  // eight values as loaded from memory
template <>
struct Eight<float> {
  float4 a, b;
  __device__ void load(const float* p) {
    a = __ldcs(reinterpret_cast<const float4*>(p));
    b = __ldcs(reinterpret_cast<const float4*>(p) + 1);
  }
};
template <>
struct Eight<__half> {
  uint4 a;
  __device__ void load(const __half* p) { a = __ldcs(reinterpret_cast<const uint4*>(p)); }
};
template <>
struct Eight<__nv_bfloat16> {
  uint4 a;
  __device__ void load(const __nv_bfloat16* p) { a = __ldcs(reinterpret_cast<const uint4*>(p)); }
};

__device__ __forceinline__ uint32_t pack(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// f32 values are rounded to the cache's type, as the runtime's own appends do
template <class C>
__device__ __forceinline__ uint4 to_cache(const Eight<float>& e) {
  return make_uint4(pack(e.a.x, e.a.y, C()), pack(e.a.z, e.a.w, C()), pack(e.b.x, e.b.y, C()),
                    pack(e.b.z, e.b.w, C()));
}
template <class C>
__device__ __forceinline__ uint4 to_cache(const Eight<C>& e) {
  return e.a;
}

// One thread moves eight values of K and of V.  Bound by memory: 16 rows of 32
// heads of 128 take 1.8 us in a graph (latency), 16 prompts of up to 512 rows of 8
// heads (50 MB) 9.1 us a call = 5.5 TB/s, 85% of the measured copy rate.
template <class S, class C>
__global__ void __launch_bounds__(256) k_kv_append(const S* k, const S* v, size_t ldk, size_t ldv,
                                                   const int* slots, int rows, int kvh, int hd, int n_slots,
                                                   C* ck, C* cv) {
  pdl_wait();
  pdl_trigger();
  const int per_row = kvh * (hd / 8), hc = hd / 8;
  const size_t all = (size_t)rows * per_row;
  for (size_t e = (size_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (size_t)gridDim.x * 256) {
    const int r = (int)(e / per_row), rem = (int)(e - (size_t)r * per_row);
    const int slot = slots[r];
    if (slot < 0 || slot >= n_slots) continue;
    const int h = rem / hc, c = rem - h * hc;
    Eight<S> ek, ev;
    ek.load(k + (size_t)r * ldk + (size_t)rem * 8);
    ev.load(v + (size_t)r * ldv + (size_t)rem * 8);
    const size_t o = (((size_t)(slot / kKvPage) * kvh + h) * kKvPage + slot % kKvPage) * hd + c * 8;
    *reinterpret_cast<uint4*>(ck + o) = to_cache<C>(ek);
    *reinterpret_cast<uint4*>(cv + o) = to_cache<C>(ev);
  }
}

// Accepted nodes a_0 < a_1 < ... of request i move from tokens L + a_j to
// L + j.  One CTA holds a (request, head): it reads a run of nodes before it
// writes any of them, and since a_j >= j a later run reads nothing written.
__global__ void __launch_bounds__(128) k_kv_commit(const int* tables, int ld_tables, int max_pages,
                                                   const int* lengths, const int* accepted,
                                                   const int* accepted_start, int total, int kvh, int hc,
                                                   int n_pages, uint4* ck, uint4* cv) {
  pdl_wait();
  pdl_trigger();
  const int i = blockIdx.x, h = blockIdx.y;
  const int s0 = min(max(accepted_start[i], 0), total), s1 = min(max(accepted_start[i + 1], 0), total);
  const int len = lengths[i];
  if (len < 0) return;
  const int run = 128 / hc, t = threadIdx.x / hc, c = threadIdx.x % hc;
  auto chunk = [&](long long p, size_t& o) {  // offset of this thread's 16 bytes of token p
    if (p < 0 || p >= (long long)max_pages * kKvPage) return false;
    const int page = tables[(size_t)i * ld_tables + p / kKvPage];
    if (page < 0 || page >= n_pages) return false;
    o = (((size_t)page * kvh + h) * kKvPage + p % kKvPage) * hc + c;
    return true;
  };
  for (int j0 = s0; j0 < s1; j0 += run) {
    const int j = j0 + t;
    size_t from = 0, to = 0;
    bool ok = false;
    uint4 k, v;
    if (t < run && j < s1) {
      const int node = accepted[j];
      ok = node > j - s0 && chunk((long long)len + node, from) && chunk((long long)len + (j - s0), to);
      if (ok) k = ck[from], v = cv[from];
    }
    __syncthreads();
    if (ok) ck[to] = k, cv[to] = v;
    __syncthreads();
  }
}

template <class S, class C>
int append_t(const void* k, const void* v, size_t ldk, size_t ldv, const int* slots, int rows, int kvh, int hd,
             int n_slots, void* ck, void* cv, cudaStream_t st) {
  const size_t all = (size_t)rows * kvh * (hd / 8);
  const size_t blocks = ceil_div(all, 256);
  const int grid = (int)(blocks < 148 * 32 ? blocks : 148 * 32);
  return launch_step(k_kv_append<S, C>, dim3(grid), dim3(256), 0, st, (const S*)k, (const S*)v, ldk, ldv, slots,
                  rows, kvh, hd, n_slots, (C*)ck, (C*)cv);
}

}  // namespace

// The rows join the scan's CTA while there are few of them; past that the scatter
// takes a launch of its own over the whole GPU.  Graph replays, one launch and two:
// 64 rows 4.2 and 6.2 us, 1,024 7.2 and 8.0, 2,048 9.9 and 8.5 (but a second launch
// costs the host 2 us), 4,096 12.5 and 9.3.
int launch_block_tables(const PlanArgs& a, cudaStream_t st) {
  const bool one = a.rows <= kPlanRows && a.n <= kPlanThreads;
  WL_TRY(launch_step(k_plan, dim3(1), dim3(kPlanThreads), 0, st, a, one ? 1 : 0));
  if (!one && a.rows > 0) WL_TRY(launch_step(k_plan_rows, dim3((a.rows + 255) / 256), dim3(256), 0, st, a));
  return WL_OK;
}

int launch_release_pages(const ReleaseArgs& a, cudaStream_t st) {
  return launch_step(k_release, dim3(1), dim3(kPlanThreads), 0, st, a);
}

int launch_kv_append(int src, int cache, const void* k, const void* v, size_t ldk, size_t ldv, const int* slots,
                     int rows, int kvh, int hd, int n_slots, void* ck, void* cv, cudaStream_t st) {
  if (src == WL_F32 && cache == WL_F16)
    return append_t<float, __half>(k, v, ldk, ldv, slots, rows, kvh, hd, n_slots, ck, cv, st);
  if (src == WL_F32 && cache == WL_BF16)
    return append_t<float, __nv_bfloat16>(k, v, ldk, ldv, slots, rows, kvh, hd, n_slots, ck, cv, st);
  if (src == WL_F16 && cache == WL_F16)
    return append_t<__half, __half>(k, v, ldk, ldv, slots, rows, kvh, hd, n_slots, ck, cv, st);
  if (src == WL_BF16 && cache == WL_BF16)
    return append_t<__nv_bfloat16, __nv_bfloat16>(k, v, ldk, ldv, slots, rows, kvh, hd, n_slots, ck, cv, st);
  return fail(WL_ERR_UNSUPPORTED, "kv_append: f32 rows into an f16 or bf16 cache, or rows of the cache's type");
}

int launch_kv_commit(const int* tables, int ld_tables, int max_pages, const int* lengths, int n,
                     const int* accepted, const int* accepted_start, int total, int kvh, int hd, int n_pages,
                     void* ck, void* cv, cudaStream_t st) {
  return launch_step(k_kv_commit, dim3(n, kvh), dim3(128), 0, st, tables, ld_tables, max_pages, lengths, accepted,
                  accepted_start, total, kvh, hd / 8, n_pages, (uint4*)ck, (uint4*)cv);
}

}  // namespace wl
