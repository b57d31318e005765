// Attention of a step's rows over the paged cache (sm_100a).
//
// Row r is token or drafted node j of request i (row_start[i] + j = r), at
// position pos[r].  It attends the request's lengths[i] cached tokens and, of
// the step's own rows (their K and V lie at tokens lengths[i] + c), those whose
// mask bit is set; without masks the nodes c <= j, a chain.  Scores are
// q.k * scale, the window W keeps keys at positions > pos[r] - W, and
//   out = sum_j p_j v_j / sum_j p_j,   p_j = exp(s_j - max s).
// A row with nothing to attend, or with a negative position, gives zeros.
//
// k_tree_attn, tcgen05.  The (row, head of the group) pairs of a request and a
// KV head are the rows of 128-row query tiles, so a K / V tile is read once for
// all of them.  A work item is a run of key tiles for one or two query tiles;
// the key tiles of all (request, KV head, query tiles) are laid end to end and
// cut evenly over one CTA per SM, whatever the lengths, each CTA finding its
// share from a prefix sum over the requests (where it costs little, so that no
// CTA has parts of two groups).  A run that is not a whole group leaves
// unnormalised parts (o, m, l), which k_tree_combine merges.
//   a warp     brings K and V tiles in with TMA, a 16-token page at a time
//              (its 64-column halves land in 128-byte-swizzled rows);
//   a warp     issues S = Q K^T into TMEM and O += P V (P from TMEM, V as the
//              MN-major operand straight from its rows);
//   others     softmax, two threads per query row (half of a key tile's columns
//              each): S from TMEM into registers, mask, running maximum and sum,
//              P back over S.
// They work on two streams, so that one's softmax runs under the other's
// products: the two query tiles of a pair over the same keys or, for a single
// query tile, even and odd key tiles, merged at the end.  head_dim 256 has room
// in TMEM for one O only: one stream, with two S buffers.
// The maximum that P is taken against follows the true one with a lag of up to
// 2^6 (O is rescaled only past that), and P is scaled by 2^8 where it is f16, so
// that it stays clear of both ends of the type; both factors cancel in o / l.
// f32 queries enter as two f16 words, their rows scaled by a power of two that the
// score factor takes back: 22 bits of each element, or 2^-39 of the row's largest
// where that is more.  P too is two words (22 bits), two products each against the
// f16 cache; f16 and bf16 queries take P in their own type.
// Tensor products cut their sums off instead of rounding them, so O loses up to
// 2^-23 of itself, always towards zero, with each one added.  After 32 of them
// (f32; 512 for the 16-bit types) it is added, in f32 with rounding, to a copy in
// the workspace and starts again from zero, while the next scores are on their way:
// the error does not grow with the context.  f32, 27 requests of 3 tokens over
// 19,360 keys: 1.3e-6 of the result in 237 us, 1.8e-6 in 226 with 64, 1.2e-5 in 219
// without.  f16 and bf16 round P once, which takes the error, the output's own rounding
// included, from 2.1e-4 to 2.7e-4 of the result (f16) and from 1.7e-3 to 2.2e-3 (bf16);
// a second word would double the P V products.
// V rows of keys that no row may see (the end of the last page, a drafted node
// that is left out, cached tokens below the window) are zeroed in shared memory,
// since 0 * NaN is not 0.
//
// Measured (graph replays): 8 requests of one token over 32,768 keys, 8 KV heads of
// 128: 1.07 GB in 209 us = 5.1 TB/s, 79% of the measured copy rate; a ring of three or
// four tiles instead of five takes as long.  32 trees of up to 64 tokens over 8,192
// keys, 64 / 8 heads of 128, bf16: 414 GFLOP in 740 to 850 us by box and power = 490
// to 560 TFLOP/s, 28 to 32% of the measured GEMM rate.  That is bound by latency: a
// stream goes scores -> registers -> P -> product -> next scores one after the other
// (TMEM's 512 columns, two S and two O, leave no room for scores ahead), so a pair of
// 128 x 128 tiles takes about 5,000 cycles, of which the tensor pipe works 2,050 and
// the special-function unit (two exponentials per score pair) 2,100.  Tried and
// slower: 64-key tiles with two S buffers per stream (the products of 64 columns cost
// as much as those of 128), a thread per row with its 128 scores in registers, P taken
// before the maximum is known, a product warp per stream (both streams' exponentials
// then fall together), and a third of the exponentials as polynomials on the FMA pipe.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <cstring>
#include <string>
#include <type_traits>

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
// head_dim 32, whose rows are half as wide as the tiles of the tensor kernel: a thread
// per key for the scores, in f32, then 32 of the 128 threads for V, a column each, key
// after key; K and V read anew by every (row, head).  Bound by that serial pass: 16
// single tokens over 2,048 keys, 8 heads, 553 us (head_dim 64 on the tensor cores: 36).
template <class Q, class C>
__global__ void __launch_bounds__(128) k_tree_attn_row(const TreeAttnArgs a) {
  __shared__ float s_q[256], s_p[128], s_red[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int r = blockIdx.x, head = blockIdx.y, hd = a.head_dim, kvh = head / (a.heads / a.kv_heads);
  pdl_wait();
  pdl_trigger();
  if (r >= min(a.row_start[a.n], a.rows)) return;
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.row_start[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  const int i = lo, row0 = max(a.row_start[i], 0), T = min(a.row_start[i + 1], a.rows) - row0;
  const int len = (int)min((long long)max(a.lengths[i], 0), (long long)a.max_pages * kKvPage);
  const int pos = a.pos[r] < 0 ? -1 : max(a.pos[r], len);
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
        at = max(a.pos[row0 + c], len);
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
  for (int e = 0, d = tid; d < hd; d += 128, e++) put(out + d, l == 0.f ? 0.f : o[e] / l);
}


// ---------------------------------------------------------------- tcgen05
constexpr int kTaSoft = 16;          // softmax warps: 2 streams x 2 halves of the key tile x 4 lane quarters
constexpr int kTaLoad = 2;           // TMA warps, each with half of a tile's pages
constexpr int kTaThreads = (kTaSoft + kTaLoad + 1) * 32;
constexpr int kTaSmem = 232448;      // a CTA's shared memory: query tiles, the ring of K / V tiles, Small
constexpr int kTaLag = 6;             // log2 of the lag of the maximum

template <int HD, class Q>
struct Shape {
  static constexpr bool kSplit = sizeof(Q) == 4;       // f32 queries as two f16 words
  static constexpr int KT = HD == 256 ? 64 : 128;      // keys per tile
  static constexpr int NS = HD == 256 ? 1 : 2;         // streams
  static constexpr int NB = 2;                         // S buffers
  static constexpr int kQTile = 128 * HD * 2;          // bytes of a query tile (one word)
  static constexpr int kQBytes = kQTile * NS * (kSplit ? 2 : 1);
  static constexpr int kSlot = KT * HD * 2;            // bytes of a K or V tile
  static constexpr int kFit = (kTaSmem - kQBytes - 3 * 1024) / kSlot;
  static constexpr int kSlots = kFit < 12 ? kFit : 12;
  static constexpr int kTiles = kQBytes + kSlots * kSlot;
  // tiles after which O moves out of TMEM: 32 or 512 products
  static constexpr int kFlush = (kSplit ? 32 : 512) / (KT / 16 * (kSplit ? 2 : 1));
  static constexpr int kO = 256;                       // TMEM column of O; S buffers from 0
  static constexpr bool kBf16 = std::is_same<Q, __nv_bfloat16>::value;
  static constexpr float kShift = kBf16 ? 0.f : 8.f;   // log2 of P's scale
  static constexpr uint32_t kType = kBf16 ? (1u << 7) | (1u << 10) : 0u;
  // D f32; N at bit 17 (/8), M at bit 24 (/16), bit 16: B is MN-major
  static constexpr uint32_t kIdescS = (1u << 4) | kType | ((uint32_t)(KT >> 3) << 17) | (8u << 24);
  static constexpr uint32_t kIdescO = (1u << 4) | kType | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | (8u << 24);
};

__device__ __forceinline__ uint32_t sptr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// bounded wait; gives up at once when another role has
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* failed) {
  for (int it = 0; it < (1 << 22); it++) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 63) == 63 && *failed) return false;
  }
  *failed = 1;
  return false;
}
// Shared-memory operands: the descriptor's low word is the address (in 16-byte
// units, with the leading offset above it), the high word fixed for a layout
// (stride between 8-row groups 1024 bytes, version 1, 128-byte swizzle).
constexpr uint32_t kDescHi = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lead) { return (addr >> 4) | (lead >> 4) << 16; }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.b32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.b32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(acc), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar)
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

#define WL_R8(v, o) "=r"(v[o]), "=r"(v[o + 1]), "=r"(v[o + 2]), "=r"(v[o + 3]), "=r"(v[o + 4]), "=r"(v[o + 5]), "=r"(v[o + 6]), "=r"(v[o + 7])
#define WL_I8(v, o) "r"(v[o]), "r"(v[o + 1]), "r"(v[o + 2]), "r"(v[o + 3]), "r"(v[o + 4]), "r"(v[o + 5]), "r"(v[o + 6]), "r"(v[o + 7])
// 32 columns of this thread's TMEM lane (no wait)
__device__ __forceinline__ void tm_ld32(uint32_t a, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      : WL_R8(v, 0), WL_R8(v, 8), WL_R8(v, 16), WL_R8(v, 24)
      : "r"(a));
}
__device__ __forceinline__ void tm_ld16(uint32_t a, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n"
      : WL_R8(v, 0), WL_R8(v, 8)
      : "r"(a));
}
__device__ __forceinline__ void tm_st8(uint32_t a, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};\n" ::WL_I8(v, 0), "r"(a)
               : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t a, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15};\n" ::WL_I8(v, 0),
      WL_I8(v, 8), "r"(a)
      : "memory");
}
// the loads into v have arrived: v passes through, so that no use moves before the wait
#define WL_P8(v, o) "+r"(v[o]), "+r"(v[o + 1]), "+r"(v[o + 2]), "+r"(v[o + 3]), "+r"(v[o + 4]), "+r"(v[o + 5]), "+r"(v[o + 6]), "+r"(v[o + 7])
__device__ __forceinline__ void tm_wait_ld(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : WL_P8(v, 0), WL_P8(v, 8), WL_P8(v, 16), WL_P8(v, 24)::"memory");
}
__device__ __forceinline__ void tm_wait_ld16(uint32_t* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : WL_P8(v, 0), WL_P8(v, 8)::"memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
  float m;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(m) : "f"(x), "f"(y), "f"(z));
  return m;
}
using f2 = unsigned long long;  // two f32 values, for the paired instructions
__device__ __forceinline__ f2 make_f2(float x, float y) {
  f2 v;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(x), "f"(y));
  return v;
}
__device__ __forceinline__ float lo_of(f2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi_of(f2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f2 fma2(f2 x, f2 y, f2 z) {
  f2 v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(v) : "l"(x), "l"(y), "l"(z));
  return v;
}
__device__ __forceinline__ f2 add2(f2 x, f2 y) {
  f2 v;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(x), "l"(y));
  return v;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __half) {
  const __half2 h = __floats2half2_rn(x, y);
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}
__device__ __forceinline__ uint32_t pack2(float x, float y, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  uint32_t u;
  memcpy(&u, &h, 4);
  return u;
}

// A request as the attention sees it, and its share of the work: per KV head,
// qt query tiles times kt key tiles.
struct Req {
  int row0, T, len, keys;  // keys: end of the tokens that exist
  int tile0;               // first key tile (window)
  int kt, qt;
};
template <int KT>
__device__ __forceinline__ Req request(const TreeAttnArgs& a, int i) {
  Req q;
  q.row0 = max(a.row_start[i], 0);
  q.T = min(a.row_start[i + 1], a.rows) - q.row0;
  if (q.T < 0) q.T = 0;
  const long long cap = (long long)a.max_pages * kKvPage;
  q.len = (int)min((long long)max(a.lengths[i], 0), cap);
  q.keys = (int)min((long long)q.len + q.T, cap);
  q.tile0 = a.window > 0 && q.len >= a.window ? (q.len - a.window + 1) / KT : 0;
  q.kt = max(1, (q.keys + KT - 1) / KT - q.tile0);
  q.qt = (int)(((long long)q.T * (a.heads / a.kv_heads) + 127) / 128);
  return q;
}
__device__ __forceinline__ long long quot(long long a, long long b) {  // a >= 0, b > 0
  return ((a | b) >> 32) == 0 ? (long long)((unsigned)a / (unsigned)b) : a / b;
}

// How the work is cut: CTA c takes units [c * per, (c + 1) * per), a unit being a
// key tile times a query tile.  whole: every group starts at such a border (its
// units are rounded up to a multiple of per), so that no CTA has two.
struct Cut {
  long long per;
  bool whole;
  __device__ long long pad(long long u) const { return whole ? quot(u + per - 1, per) * per : u; }
};
// Groups of a request and KV head: pairs of query tiles, then single ones.
template <int NS>
struct Groups {
  int pairs, singles;
  long long pair, single, all;  // units of one, and of them together
  __device__ Groups(const Req& q, const Cut& cut) {
    pairs = NS == 2 ? q.qt / 2 : 0;
    singles = NS == 2 ? q.qt & 1 : q.qt;
    pair = cut.pad(2LL * q.kt);
    single = cut.pad(q.kt);
    all = pairs * pair + singles * single;
  }
};
template <int NS>
__device__ __forceinline__ long long units(const TreeAttnArgs& a, const Req& q, const Cut& cut) {
  return a.kv_heads * Groups<NS>(q, cut).all;
}

// Mask bits of nodes c0 .. c0 + 31 of a row (c0 > -32; nodes below 0: clear).
__device__ __forceinline__ uint32_t mask_bits(const TreeAttnArgs& a, int row, int c0) {
  const unsigned* m = a.mask + (size_t)row * a.words;
  if (c0 < 0) return m[0] << -c0;
  const int w = c0 >> 5;
  const uint32_t w0 = w < a.words ? m[w] : 0u, w1 = w + 1 < a.words ? m[w + 1] : 0u;
  return __funnelshift_r(w0, w1, c0 & 31);
}

// A run of key tiles of one group: KV head kvh, query tiles qt0 .. qt0 + w - 1.
// The TMA warp walks the CTA's share and hands the runs to the other warps
// through shared memory, which keeps that state out of their registers.
struct Run {
  int nt;             // key tiles; 0: no further run
  int key0;           // first key
  int w;              // query tiles: 2, or 1
  int len, keys;      // Req's
  int row0, T;
  int i, kvh, qt0;
  int first, whole;   // the CTA's first run; the whole group
};
// Runs in flight: the ring's 12 tiles are those of six runs at most, one more
// waits for a slot, and the softmax may still be at the end of the one before.
constexpr int kRuns = 9;

// Walks the CTA's share [x, x1) of the laid-out key tiles; all threads alike.
template <int HD, class Q>
struct Walk {
  using S = Shape<HD, Q>;
  long long x0, x, x1, base;  // base: start of request i
  Cut cut;
  int i;
  Req q;
  __device__ bool next(const TreeAttnArgs& args, Run& r) {
    while (x < x1) {
      for (long long u; x >= base + (u = units<S::NS>(args, q, cut)); q = request<S::KT>(args, ++i)) base += u;
      const Groups<S::NS> g(q, cut);
      const long long off = x - base;
      r.kvh = (int)quot(off, g.all);
      long long y = off - r.kvh * g.all, size = g.pair, g0 = base + r.kvh * g.all;
      const long long paired = g.pairs * g.pair;
      r.w = y < paired ? 2 : 1;
      r.qt0 = 0;
      if (r.w == 1) y -= paired, g0 += paired, r.qt0 = 2 * g.pairs, size = g.single;
      const int idx = (int)quot(y, size);
      r.qt0 += idx * r.w;
      g0 += idx * size;
      const long long e = min(x1, g0 + size);
      const int ta = (int)min((long long)q.kt, (x - g0) >> (r.w - 1));  // w is 1 or 2
      const int tb = (int)min((long long)q.kt, (e - g0) >> (r.w - 1));
      r.nt = tb - ta;
      r.key0 = (q.tile0 + ta) * S::KT;
      r.len = q.len, r.keys = q.keys, r.row0 = q.row0, r.T = q.T, r.i = i;
      r.first = x0 >= g0;
      r.whole = ta == 0 && tb == q.kt;
      x = e;
      if (tb > ta) return true;
    }
    return false;
  }
};

// Parts: [CTA][first / last run][stream][prow rows][HD] f32, then (m, l) of
// each; one status word per CTA and the requests' prefix sums before them.
constexpr int kGaveUp = 1, kOdd = 2;  // a wait ran out; some O is not finite
struct Parts {
  int* status;       // [ctas] bits
  long long* start;  // [n] prefix sums, then the total and a CTA's share (negative: whole groups)
  float* o;
  float* ml;
  int prow;          // rows kept of a 128-row tile
};
__host__ __device__ inline size_t round256(size_t x) { return (x + 255) / 256 * 256; }
__host__ inline int part_rows(int rows, int group) {
  const long long m = (long long)rows * group;
  return m < 128 ? (int)m : 128;
}
__host__ inline size_t part_bytes(int ctas, int n, int hd, int prow) {
  return round256((size_t)ctas * 4) + round256((size_t)(n + 2) * 8) + (size_t)ctas * 4 * prow * (hd + 2) * 4;
}
__host__ inline Parts parts_at(void* ws, int ctas, int n, int hd, int prow) {
  Parts p;
  uint8_t* b = (uint8_t*)ws;
  p.status = (int*)b;
  p.start = (long long*)(b + round256((size_t)ctas * 4));
  p.o = (float*)(b + round256((size_t)ctas * 4) + round256((size_t)(n + 2) * 8));
  p.ml = p.o + (size_t)ctas * 4 * prow * hd;
  p.prow = prow;
  return p;
}

__device__ __forceinline__ void st4(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
// O on its way out of TMEM, 16 columns of a row: a warp's rows side by side,
// four columns of each after another, in the place of their parts
__device__ __forceinline__ void put_kept(float* p, int rows, const float* v) {
#pragma unroll
  for (int e = 0; e < 4; e++) st4(p + e * 4 * rows, v + 4 * e);
}
__device__ __forceinline__ void add_kept(float* v, const float* p, int rows, float x) {
  float4 y[4];
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = *reinterpret_cast<const float4*>(p + e * 4 * rows);
#pragma unroll
  for (int e = 0; e < 4; e++)
    v[4 * e] += y[e].x * x, v[4 * e + 1] += y[e].y * x, v[4 * e + 2] += y[e].z * x, v[4 * e + 3] += y[e].w * x;
}

template <int HD, class Q>
struct Small {  // behind the tiles in shared memory
  static constexpr int NSLOT = Shape<HD, Q>::kSlots;
  uint64_t bars[2 * NSLOT + 26 + kRuns];
  Run runs[kRuns];
  union {
    float half[2][2][128];  // [stream][half][row]; one stream: [parity of the exchange]
    long long scan[kTaThreads / 32];  // at the start
  };
  long long base;
  Req q;
  int req, fail, odd, need[8];
  uint32_t tmem;
};

template <int HD, class Q>
__global__ void __launch_bounds__(kTaThreads, 1)
    k_tree_attn(const TreeAttnArgs a, const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                const Parts parts) {
  using S = Shape<HD, Q>;
  using C = typename std::conditional<S::kSplit, __half, Q>::type;
  constexpr int KT = S::KT, NS = S::NS, NB = S::NB, NSLOT = S::kSlots, ATOMS = HD / 64, PAGES = KT / kKvPage;
  // everything lies in one dynamic block, which starts at the CTA's first byte
  // of shared memory: 1024-byte aligned, as the swizzled tiles need it
  extern __shared__ __align__(1024) uint8_t sm[];
  Small<HD, Q>& sh = *reinterpret_cast<Small<HD, Q>*>(sm + S::kTiles);
  static_assert(S::kTiles + sizeof(Small<HD, Q>) <= kTaSmem, "more than a CTA's shared memory");
  if (sptr(sm) & 1023u) {
    if (threadIdx.x == 0) parts.status[blockIdx.x] = 1;
    return;
  }
  const uint32_t full = sptr(sh.bars), empty = full + 8 * NSLOT, qbar = empty + 8 * NSLOT, sbar = qbar + 8,
                 pbar = sbar + 32, dbar = pbar + 32, obar = dbar + 8, endbar = obar + 16, xfull = endbar + 8,
                 xempty = xfull + 16, hbar = xempty + 16, rbar = hbar + 64, mbar = rbar + 8 * kRuns;
  const uint32_t qs = sptr(sm), ring = qs + S::kQBytes;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = a.heads / a.kv_heads;

  if (warp == kTaSoft + kTaLoad) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(sptr(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  if (tid == 0) {
    for (int k = 0; k < NSLOT; k++) bar_init(full + 8 * k, kTaLoad), bar_init(empty + 8 * k, 1);
    bar_init(qbar, kTaSoft);
    for (int k = 0; k < NB; k++) bar_init(sbar + 8 * k, 1), bar_init(pbar + 8 * k, 8);
    for (int k = 0; k < 2; k++) bar_init(obar + 8 * k, 1), bar_init(xfull + 8 * k, 4), bar_init(xempty + 8 * k, 4);
    for (int k = 0; k < 8; k++) bar_init(hbar + 8 * k, 2);
    for (int k = 0; k < kRuns; k++) bar_init(rbar + 8 * k, 1);
    bar_init(dbar, 1);
    bar_init(endbar, 1);
    bar_init(mbar, kTaSoft);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    sh.fail = sh.odd = 0;
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];\n" ::"l"(&mv) : "memory");
  }
  pdl_wait();
  pdl_trigger();

  // this CTA's share of the key tiles: the total, then the request it starts in
  long long share0, share1;
  Cut cut;
  {
    auto block_sum = [&](long long v, long long& before) {  // the sum, and that of the threads before this one
      long long x = v;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      __syncthreads();
      if (lane == 31) sh.scan[warp] = x;
      __syncthreads();
      long long w = lane < kTaThreads / 32 ? sh.scan[lane] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
      }
      const long long upto = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
      before = (warp ? upto : 0) + x - v;
      return __shfl_sync(0xffffffffu, w, 31);
    };
    long long total = 0, before, u = 0;
    Req q{};
    cut = Cut{1, false};
    for (int i0 = 0; i0 < a.n; i0 += kTaThreads) {
      if (i0 + tid < a.n) q = request<KT>(a, i0 + tid);
      u = i0 + tid < a.n ? units<NS>(a, q, cut) : 0;
      total += block_sum(u, before);
    }
    cut.per = total > 0 ? quot(total + gridDim.x - 1, gridDim.x) : 1;
    // A CTA that gets the end of one group and the start of the next pays a run's
    // fixed latency twice (about 6 us, as much as six units).  If there is a share
    // up to seven units larger with which every group has CTAs of its own, it is
    // taken (5 drafted tokens over 640 keys, 32 KV heads: last CTA done after 12.4
    // instead of 15.7 us; 16 trees of 13 over 2048 keys: 30 instead of 33 us a call).
    if (a.n <= kTaThreads && cut.per < 4096) {
      // a warp per candidate, over the requests' groups (in the query tiles' place)
      int4* req = reinterpret_cast<int4*>(sm);
      const Groups<NS> g(q, cut);
      if (tid < a.n) req[tid] = u > 0 ? make_int4(g.pairs, g.singles, (int)g.pair, (int)g.single) : make_int4(0, 0, 0, 0);
      __syncthreads();
      if (warp < 8) {
        const unsigned p = (unsigned)cut.per + warp;
        long long ctas = 0;
        for (int i = lane; i < a.n; i += 32) {
          const int4 v = req[i];
          ctas += (long long)v.x * (((unsigned)v.z + p - 1) / p) + (long long)v.y * (((unsigned)v.w + p - 1) / p);
        }
        const int need = __reduce_add_sync(0xffffffffu, (int)min(ctas * a.kv_heads, 1LL << 20));
        if (lane == 0) sh.need[warp] = need;
      }
      __syncthreads();
      int k = 0;
      while (k < 8 && sh.need[k] > (int)gridDim.x) k++;
      if (k < 8) {
        cut.per += k;
        cut.whole = true;
        u = u > 0 ? units<NS>(a, q, cut) : 0;
        total = block_sum(u, before);
      }
    }
    share0 = min(total, cut.per * blockIdx.x);
    share1 = min(total, share0 + cut.per);
    long long sum = 0;
    for (int i0 = 0; i0 < a.n; i0 += kTaThreads) {
      const int i = i0 + tid;
      long long all = total;
      if (a.n > kTaThreads) {  // otherwise the sums above stand
        if (i < a.n) q = request<KT>(a, i);
        u = i < a.n ? units<NS>(a, q, cut) : 0;
        all = block_sum(u, before);
      }
      before += sum;
      if (share0 >= before && share0 < before + u) sh.req = i, sh.base = before, sh.q = q;
      if (blockIdx.x == 0 && i < a.n) parts.start[i] = before;
      sum += all;
    }
    if (blockIdx.x == 0 && tid == 0) parts.start[a.n] = total, parts.start[a.n + 1] = cut.whole ? -cut.per : cut.per;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  // run r of the CTA, once the TMA warp has put it down; null when a wait gave up
  auto get_run = [&](uint32_t r) -> const Run* {
    const uint32_t k = r % kRuns;
    return bar_wait(rbar + 8 * k, (r / kRuns) & 1, &sh.fail) ? &sh.runs[k] : nullptr;
  };

  if (warp >= kTaSoft && warp < kTaSoft + kTaLoad) {
    // ------------------------------------------------------------ TMA
    const int part = warp - kTaSoft;
    const bool lead = elect_one();
    uint32_t seq = 0, nr = 0;
    Walk<HD, Q> walk;
    walk.x0 = walk.x = share0;
    walk.x1 = share1;
    walk.cut = cut;
    if (share0 < share1) walk.i = sh.req, walk.base = sh.base, walk.q = sh.q;
    Run run;
    auto hand_over = [&]() {
      if (part == 0 && lane == 0) {
        sh.runs[nr % kRuns] = run;
        bar_arrive(rbar + 8 * (nr % kRuns));
      }
      nr++;
    };
    const int rows_end = a.n_pages * a.kv_heads * kKvPage;  // past the cache: read as zeros
    bool ok = true;
    while (ok && walk.next(a, run)) {
      hand_over();
      const int nt = run.nt;
      const int* table = a.tables + (size_t)run.i * a.ld_tables;
      // first rows of the pages of 32 / PAGES tiles, a page per lane; the next
      // batch is on its way while this one is used
      auto fetch = [&](int batch) {
        const int pg = run.key0 / kKvPage + batch * 32 + lane;
        int row = rows_end;
        if (pg < a.max_pages && pg * kKvPage < run.keys) {
          const int id = table[pg];
          if (id >= 0 && id < a.n_pages) row = (id * a.kv_heads + run.kvh) * kKvPage;
        }
        return row;
      };
      int before = rows_end, now = fetch(0), after = nt > 32 / PAGES ? fetch(1) : rows_end, at = 0;
      auto load = [&](const CUtensorMap* map, int tile) {
        if (!ok) return;
        const int batch = tile / (32 / PAGES);
        if (batch > at) before = now, now = after, after = fetch(batch + 1), at = batch;
        const int rows = batch == at ? now : before;  // V follows K by fewer tiles than a batch has
        const uint32_t slot = seq % NSLOT, bar = full + 8 * slot;
        if (seq >= NSLOT) ok = __all_sync(0xffffffffu, bar_wait(empty + 8 * slot, (seq / NSLOT - 1) & 1, &sh.fail));
        if (!ok) return;
        if (lead)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar),
                       "r"((uint32_t)(S::kSlot / kTaLoad))
                       : "memory");
#pragma unroll
        for (int p = 0; p < PAGES / kTaLoad; p++) {
          const int page = part * (PAGES / kTaLoad) + p;
          const int row = __shfl_sync(0xffffffffu, rows, tile % (32 / PAGES) * PAGES + page);
          if (lead) {
#pragma unroll
            for (int h = 0; h < ATOMS; h++)
              asm volatile(
                  "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
                  "[%4];\n" ::"r"(ring + slot * S::kSlot + h * KT * 128 + page * kKvPage * 128),
                  "l"(map), "r"(h * 64), "r"(row), "r"(bar)
                  : "memory");
          }
        }
        seq++;
      };
      // in the order the products use them: the K tiles whose scores run ahead, then V and K in turn
      const int ahead = run.w == 2 ? NB / 2 : NB;
      for (int t = 0; t < ahead && t < nt; t++) load(&mk, t);
      for (int t = 0; t < nt; t++) {
        load(&mv, t);
        if (t + ahead < nt) load(&mk, t + ahead);
      }
    }
    run.nt = 0;
    hand_over();
    // every copy has landed before the CTA ends
    for (uint32_t k = seq > NSLOT ? seq - NSLOT : 0; k < seq; k++) {
      int dummy = 0;
      bar_wait(full + 8 * (k % NSLOT), (k / NSLOT) & 1, &dummy);
    }
  } else if (warp == kTaSoft + kTaLoad) {
    // ------------------------------------------------------------ products
    // The whole warp follows the schedule, so that operands are formed in
    // uniform registers; one elected lane issues.  (With the loop run by a
    // single lane a product took about 90 cycles to issue.)
    const bool lead = elect_one();
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    uint32_t seq = 0;          // tiles of the ring used up by earlier runs
    uint32_t np = 0;           // parity of the P tiles taken from each buffer
    uint32_t runs = 0;
    bool ok = true;
    auto wait = [&](uint32_t bar, uint32_t parity) {
      return ok = ok && __all_sync(0xffffffffu, bar_wait(bar, parity, &sh.fail));
    };
    while (true) {
      const Run* run = get_run(runs);
      ok = __all_sync(0xffffffffu, run != nullptr);
      if (!ok) break;
      const int nt = __shfl_sync(0xffffffffu, run->nt, 0);
      const bool pair = __shfl_sync(0xffffffffu, run->w, 0) == 2;
      if (nt == 0) break;
      const int nu = pair ? 2 * nt : nt;
      // place in the ring's order of the K and V tile t
      const int ahead = pair ? NB / 2 : NB;
      auto k_at = [&](int t) { return (uint32_t)(t < ahead ? t : 2 * t - ahead + 1); };
      auto v_at = [&](int t) { return (uint32_t)(min(nt, t + ahead) + t); };
      // S buffer of unit u: one for each of two streams, or two for one
      auto buf = [&](int u) { return u & 1; };
      auto scores = [&](int u) {  // S = Q K^T
        const uint32_t k = seq + k_at(pair ? u >> 1 : u), slot = k % NSLOT;
        if (!wait(full + 8 * slot, (k / NSLOT) & 1)) return;
        fence_after();
        const uint32_t kb = desc_lo(ring + slot * S::kSlot, 16);
        const uint32_t qb = desc_lo(qs + (pair ? (u & 1) * S::kQTile : 0), 16), d = tm + buf(u) * KT;
        if (lead) {
#pragma unroll
          for (int w = 0; w < (S::kSplit ? 2 : 1); w++)
#pragma unroll
            for (int ks = 0; ks < HD / 16; ks++)
              // the low words first: sums are cut off rather than rounded, and
              // that costs least while they are small
              mma_ss(d, qb + (((S::kSplit && !w ? NS * S::kQTile : 0) + (ks >> 2) * 128 * 128 + (ks & 3) * 32) >> 4),
                     kb + (((ks >> 2) * KT * 128 + (ks & 3) * 32) >> 4), S::kIdescS, w || ks ? 1u : 0u);
          mma_commit(sbar + 8 * buf(u));
          if (!pair || (u & 1)) mma_commit(empty + 8 * slot);
        }
      };
      if (!wait(qbar, runs & 1)) break;
      runs++;
      fence_after();
      for (int u = 0; u < NB && u < nu; u++) scores(u);
      for (int u = 0; ok && u < nu; u++) {
        const int b = buf(u), t = NS == 2 ? u & 1 : 0;
        const uint32_t k = seq + v_at(pair ? u >> 1 : u), slot = k % NSLOT, parity = np >> b & 1;
        np ^= 1u << b;
        if (!wait(full + 8 * slot, (k / NSLOT) & 1) || !wait(pbar + 8 * b, parity)) break;
        fence_after();
        const uint32_t vb = desc_lo(ring + slot * S::kSlot, KT * 128);
        const uint32_t d = tm + S::kO + t * HD, p = tm + b * KT;
        const uint32_t acc = u < NS ? 0u : 1u;
        if (lead) {
#pragma unroll
          for (int w = 0; w < (S::kSplit ? 2 : 1); w++)
#pragma unroll
            for (int ks = 0; ks < KT / 16; ks++)
              mma_ts(d, p + (ks >> 1) * 32 + (ks & 1) * 8 + (S::kSplit && !w ? 16 : 0), vb + (ks * 16 * 128 >> 4),
                     S::kIdescO, w || ks ? 1u : acc);
          if (!pair || t) mma_commit(empty + 8 * slot);
          mma_commit(obar + 8 * t);
        }
        if (u + NB < nu) scores(u + NB);
      }
      if (!ok) break;
      if (lead) mma_commit(dbar);
      seq += 2 * nt;
    }
    if (!ok && lead) {  // products in flight finish before TMEM is given back
      mma_commit(endbar);
      int dummy = 0;
      bar_wait(endbar, 0, &dummy);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax
    // stream t; half hf of the key tile's columns (and of O's); row wt of the query tile
    const int t = warp >> 3, hf = (warp >> 2) & 1, wt = (warp & 3) * 32 + lane;
    constexpr int CW = KT / 2, OW = HD / 2;  // columns of S and of O that a thread takes
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t oth = hbar + 8 * (t * 4 + (warp & 3));  // meets the other half's warp
    const uint32_t op = tmem + lanes + S::kO + (NS == 2 ? t * HD : 0) + hf * OW;
    float c = a.scale * 1.4426950408889634f;
    uint32_t ns = 0, runs = 0, no = 0, seq = 0;  // ns: parities of the stream's S buffers; no: its products so far
    uint32_t nx = 0;           // exchanges between the streams
    uint32_t nh = 0;           // and between the halves
    bool ok = true;
    auto wait_warp = [&](uint32_t bar, uint32_t parity) {  // the same answer for the whole warp
      return (bool)__all_sync(0xffffffffu, bar_wait(bar, parity, &sh.fail));
    };
    auto arrive_warp = [&](uint32_t bar) {
      __syncwarp();
      if (lane == 0) bar_arrive(bar);
    };
    auto meet_all = [&](uint32_t parity) {  // all softmax warps
      arrive_warp(mbar);
      return wait_warp(mbar, parity & 1);
    };
    auto meet = [&]() {
      arrive_warp(oth);
      ok = wait_warp(oth, nh++ & 1);
    };
    // this row's value of the other half.  It is written over by the next call
    // (two streams: a product or a meet() lies between) or the one after that
    // (one stream: whose readers the next call meets).
    auto swap_half = [&](float v) {
      const int k = NS == 2 ? t : nh & 1;
      sh.half[k][hf][wt] = v;
      meet();
      return sh.half[k][hf ^ 1][wt];
    };
    while (true) {
      const Run* rp = get_run(runs);
      if (!__all_sync(0xffffffffu, rp != nullptr) || rp->nt == 0) break;
      const Run& run = *rp;
      const int nt = run.nt, pair = run.w == 2, nu = pair ? 2 * nt : nt, len = run.len, first = run.key0;
      // f32: the rows' factors go through sh.half, which the run before may still be reading
      if (S::kSplit && runs > 0 && !(ok = meet_all(runs - 1))) break;
      // queries: the threads copy 16-byte pieces of the (row, head) pairs
      {
        const int m0 = run.qt0 * 128, mn = min(run.w * 128, run.T * group - m0);
        const Q* src = (const Q*)a.q + (size_t)run.kvh * group * HD;
        for (int e = tid; e < mn * (HD / 8); e += kTaSoft * 32) {
          const int m = e / (HD / 8), ch = e - m * (HD / 8);
          const int j = (m0 + m) / group, g = (m0 + m) - j * group;
          const Q* p = src + (size_t)(run.row0 + j) * a.ldq + (size_t)g * HD + ch * 8;
          const int row = m & 127;
          uint8_t* d = sm + (m >> 7) * S::kQTile + (ch >> 3) * 128 * 128 + row * 128 + (((ch & 7) ^ (row & 7)) << 4);
          if constexpr (S::kSplit) {
            const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
            float f[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
            // The row times a power of two that brings its largest value to 2^14 .. 2^15, clear
            // of both ends of f16; the HD / 8 lanes that copy the row find it together.
            uint32_t big = 0;
#pragma unroll
            for (int k = 0; k < 8; k++) big = max(big, __float_as_uint(f[k]) & 0x7fffffffu);
            constexpr int LR = HD / 8;
            big = __reduce_max_sync((LR == 32 ? 0xffffffffu : (1u << (LR & 31)) - 1) << (lane & ~(LR - 1)), big) >> 23;
            const int up = big == 255 ? 0 : min(141 - (int)big, 100);  // the power; inf and NaN stay
            const float factor = __uint_as_float((127 + up) << 23);
#pragma unroll
            for (int k = 0; k < 8; k++) f[k] *= factor;
            // and its inverse for the threads of the row, each of which has a place of its own
            if (ch < 4 && (!pair || ch >> 1 == m >> 7)) sh.half[ch >> 1][ch & 1][row] = __uint_as_float((127 - up) << 23);
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
              const __half h0 = __float2half_rn(f[2 * k]), h1 = __float2half_rn(f[2 * k + 1]);
              const __half2 h = __halves2half2(h0, h1);
              memcpy(&hi[k], &h, 4);
              lo[k] = pack2(f[2 * k] - __half2float(h0), f[2 * k + 1] - __half2float(h1), __half());
            }
            *reinterpret_cast<uint4*>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(d + NS * S::kQTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          } else {
            *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(p);
          }
        }
      }
      fence_async();
      fence_before();
      arrive_warp(qbar);
      if constexpr (S::kSplit) {
        if (!(ok = wait_warp(qbar, runs & 1))) break;
        c = fmaxf(a.scale * 1.4426950408889634f * sh.half[NS == 2 ? t : 0][hf][wt], 0x1p-126f);  // -inf * c stays -inf
      }

      const int m = (run.qt0 + (pair ? t : 0)) * 128 + wt;
      const int j = m / group, g = m - j * group;
      const bool live = m < run.T * group;
      const int row = run.row0 + (live ? j : 0);
      int pos = live ? a.pos[row] : -1;
      if (pos >= 0 && pos < len) pos = len;
      const bool warp_live = __any_sync(0xffffffffu, live);
      // a page outside the cache: then every tile looks at its pages
      const int* table = a.tables + (size_t)run.i * a.ld_tables;
      bool holes = false;
      {
        const int p1 = min((first + nt * KT) / kKvPage, (run.keys + kKvPage - 1) / kKvPage);
        for (int p = first / kKvPage + lane; p < p1; p += 32) {
          const int id = table[p];
          holes |= id < 0 || id >= a.n_pages;
        }
        holes = __any_sync(0xffffffffu, holes);
      }
      // bits of the keys k0 .. k0 + 31 that this thread's row attends
      auto visible = [&](int k0) {
        uint32_t see = 0;
        if (pos < 0) return see;
        // cached tokens: a range
        const int lo = a.window > 0 ? max(pos - a.window + 1 - k0, 0) : 0, hi = min(len - k0, 32);
        if (hi > lo) see = (hi >= 32 ? 0xffffffffu : (1u << hi) - 1u) & ~((1u << lo) - 1u);
        // the step's own: bits of the mask (c0: node of the word's first key)
        const int c0 = k0 - len, cn = run.keys - len;
        if (c0 > -32 && c0 < cn) {
          uint32_t own;
          if (!a.mask) {
            const int n = j + 1 - c0;
            own = n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u;
            if (c0 < 0) own &= 0xffffffffu << -c0;
          } else {
            own = mask_bits(a, row, c0);
          }
          if (cn - c0 < 32) own &= (1u << (cn - c0)) - 1u;
          if (a.window > 0)
            for (uint32_t left = own; left; left &= left - 1) {
              const int bit = __ffs(left) - 1;
              if (max(a.pos[run.row0 + c0 + bit], len) <= pos - a.window) own &= ~(1u << bit);
            }
          see |= own;
        }
        if (holes) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int pg = k0 / kKvPage + h, id = pg * kKvPage < run.keys ? table[pg] : -1;
            if (id < 0 || id >= a.n_pages) see &= ~(0xffffu << (16 * h));
          }
        }
        return see;
      };
      // keys [open0, open1) are seen by all of the warp's rows
      int open0 = live ? pos < 0 || holes ? INT_MAX : a.window > 0 ? pos - a.window + 1 : 0 : 0;
      open0 = __reduce_max_sync(0xffffffffu, open0);
      // the place of the row's part, and of what O leaves there before
      auto part = [&]() { return (((size_t)blockIdx.x * 2 + (run.first ? 0 : 1)) * 2 + t) * parts.prow + wt; };
      auto kept_rows = [&]() { return min(32, parts.prow - (wt & ~31)); };
      auto keep = [&](int k) {
        return parts.o + (part() - lane) * HD + ((hf * OW / 4 + 4 * k) * kept_rows() + lane) * 4;
      };
      float mx = -INFINITY, l = 0.f, m_kept = 0.f;  // m_kept: the maximum that belongs to what lies there
      const int step = NS == 2 ? 2 : 1;
      for (int u = NS == 2 ? t : 0; u < nu && (NS == 2 || t == 0); u += step, no++) {
        const int b = u & 1, v = NS == 2 ? 0 : b;
        const int tile = pair ? u >> 1 : u, key0 = first + tile * KT;
        if (NS == 1 && !(ok = wait_warp(sbar + 8 * b, ns >> v & 1))) break;
        const int done = u / step;  // the stream's tiles before this one
        if (done > 0 && done % S::kFlush == 0 && warp_live) {
          // O leaves TMEM once it is at rest, while the next scores are on their way.  The
          // wait must be for the phase that may still be open: scores seen before came
          // after the product before the last.  With one stream that takes these scores.
          if (!(ok = wait_warp(obar + 8 * t, (no - 1) & 1))) break;
          fence_after();
          const float old = m_kept == mx ? 1.f : ex2(m_kept - mx);
          m_kept = mx;
#pragma unroll 1
          for (int k = 0; k < OW / 16; k++) {
            float v[16];
            tm_ld16(op + k * 16, reinterpret_cast<uint32_t*>(v));
            tm_wait_ld16(reinterpret_cast<uint32_t*>(v));
            if (live && wt < parts.prow) {
              if (done > S::kFlush) add_kept(v, keep(k), kept_rows(), old);
              put_kept(keep(k), kept_rows(), v);
            }
            __syncwarp();
            const uint32_t zero[16] = {};
            tm_st16(op + k * 16, zero);
          }
          tm_wait_st();  // a rescale of the same tile reads the zeros
        }
        if (NS == 2 && !(ok = wait_warp(sbar + 8 * b, ns >> v & 1))) break;
        ns ^= 1u << v;
        fence_after();
        const uint32_t sp = tmem + lanes + b * KT + hf * CW;
        if (warp_live) {
          // the scores, 32 at a time: for the maximum, and again for P (held in
          // between, 64 of them push the loop's state out of registers)
          const bool masked = key0 < open0 || key0 + KT > len;
          float s[32], top = -INFINITY;
          auto load = [&](int k) {
            tm_ld32(sp + k * 32, reinterpret_cast<uint32_t*>(s));
            tm_wait_ld(reinterpret_cast<uint32_t*>(s));
            if (masked) {
              const uint32_t see = visible(key0 + hf * CW + 32 * k);
#pragma unroll
              for (int e = 0; e < 32; e++) s[e] = see >> e & 1u ? s[e] : -INFINITY;
              __syncwarp();
            }
          };
#pragma unroll 1
          for (int k = 0; k < CW / 32; k++) {
            load(k);
            float t4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int e = 4; e < 32; e += 8)
#pragma unroll
              for (int x = 0; x < 4; x++) t4[x] = e + 4 < 32 ? max3(t4[x], s[e + x], s[e + 4 + x]) : fmaxf(t4[x], s[e + x]);
            top = max3(top, max3(t4[0], t4[1], t4[2]), t4[3]);
          }
          top = fmaxf(top, swap_half(top)) * c;
          if (!ok) break;
          // follow the maximum; O and l are rescaled only past the lag
          float scale = 1.f;
          if (mx == -INFINITY) {
            mx = top;
          } else if (live && top > mx + kTaLag) {
            scale = ex2(mx - top);
            mx = top;
            l *= scale;
          }
          if (__any_sync(0xffffffffu, scale != 1.f)) {
            // O is at rest once the stream's last product is done (the one before it is: these scores came after)
            if (!(ok = wait_warp(obar + 8 * t, (no - 1) & 1))) break;
            fence_after();
#pragma unroll 1
            for (int k = 0; k < OW / 16; k++) {
              uint32_t v[16];
              tm_ld16(op + k * 16, v);
              tm_wait_ld16(v);
#pragma unroll
              for (int e = 0; e < 16; e++) v[e] = __float_as_uint(__uint_as_float(v[e]) * scale);
              tm_st16(op + k * 16, v);
            }
          }
          const float off = (mx == -INFINITY ? 0.f : -mx) + S::kShift;
          const f2 c2 = make_f2(c, c), off2 = make_f2(off, off);
          f2 sum[2] = {make_f2(0.f, 0.f), make_f2(0.f, 0.f)};
#pragma unroll 1
          for (int k = 0; k < CW / 32; k++) {
            if (CW > 32) load(k);
            // over the scores they came from: 16 columns of high words, then low ones
#pragma unroll
            for (int h = 0; h < 2; h++) {
              uint32_t hi[8], lo[8];
#pragma unroll
              for (int e = 0; e < 8; e++) {
                const f2 x = fma2(make_f2(s[16 * h + 2 * e], s[16 * h + 2 * e + 1]), c2, off2);
                const float p0 = ex2(lo_of(x)), p1 = ex2(hi_of(x));
                sum[e & 1] = add2(sum[e & 1], make_f2(p0, p1));
                hi[e] = pack2(p0, p1, C());
                if constexpr (S::kSplit) {
                  __half2 y;
                  memcpy(&y, &hi[e], 4);
                  const float2 f = __half22float2(y);
                  lo[e] = pack2(p0 - f.x, p1 - f.y, __half());
                }
              }
              tm_st8(sp + k * 32 + h * 8, hi);
              if constexpr (S::kSplit) tm_st8(sp + k * 32 + 16 + h * 8, lo);
            }
          }
          sum[0] = add2(sum[0], sum[1]);
          l += lo_of(sum[0]) + hi_of(sum[0]);
          tm_wait_st();
        }
        if (hf == 0 && (key0 + KT > len || (a.window > 0 && key0 <= len - a.window))) {
          // V rows that no row sees: keys past the end, nodes in nobody's mask, cached
          // tokens below every row's window.  A warp takes 32 keys, its lanes the
          // request's rows.
          const int k0 = key0 + (wt & ~31);
          bool dead = false;
          if (wt < KT) {
            uint32_t seen = 0;
            if (!a.mask || k0 + 32 <= len) {
              seen = 0xffffffffu;
            } else if (k0 < run.keys) {
#pragma unroll 2
              for (int r = lane; r < run.T; r += 32) {
                const uint32_t bits = mask_bits(a, run.row0 + r, k0 - len);
                if (a.pos[run.row0 + r] >= 0) seen |= bits;
              }
              seen = __reduce_or_sync(0xffffffffu, seen);
              if (k0 < len) seen |= (1u << (len - k0)) - 1u;  // cached tokens of the word
            }
            dead = key0 + wt >= run.keys || !(seen >> lane & 1u) || (a.window > 0 && key0 + wt <= len - a.window);
          }
          const uint32_t k = seq + (uint32_t)(min(nt, tile + (pair ? NB / 2 : NB)) + tile);
          const uint32_t slot = k % NSLOT;
          ok = wait_warp(full + 8 * slot, (k / NSLOT) & 1);
          if (!ok) break;
          if (dead) {
            uint8_t* v = sm + S::kQBytes + slot * S::kSlot + wt * 128;
#pragma unroll 1
            for (int h = 0; h < ATOMS; h++)
#pragma unroll
              for (int e = 0; e < 8; e++)
                *reinterpret_cast<uint4*>(v + h * KT * 128 + e * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_async();
        }
        fence_before();
        arrive_warp(pbar + 8 * b);
      }
      seq += 2 * nt;
      if (!ok) break;
      ok = wait_warp(dbar, runs++ & 1);
      if (!ok) break;
      fence_after();
      if (!(NS == 2 ? t < nu : t == 0)) continue;  // no tile for this stream
      l += swap_half(l);
      if (!ok) break;
      const bool merge = NS == 2 && run.whole && !pair && nu > 1;  // two streams of one row, joined here
      float* xb = reinterpret_cast<float*>(sm + S::kQTile) + hf * 16 * 128;  // the second query tile's place is free
      float own = 1.f, other = 0.f;
      if (merge && t == 1) {  // (m, l) for the other stream
        meet();
        sh.half[1][hf][wt] = hf ? l : mx;
        if (ok) meet();
        if (!ok) break;
      }
      if (warp_live && (nu - 1 - (NS == 2 ? t : 0)) / step >= S::kFlush) {
        // O whole again; the halves' parts lie in one another's places
        const float old = m_kept == mx ? 1.f : ex2(m_kept - mx);
#pragma unroll 1
        for (int k = 0; k < OW / 16; k++) {
          float v[16];
          tm_ld16(op + k * 16, reinterpret_cast<uint32_t*>(v));
          tm_wait_ld16(reinterpret_cast<uint32_t*>(v));
          if (live && wt < parts.prow) add_kept(v, keep(k), kept_rows(), old);
          __syncwarp();
          tm_st16(op + k * 16, reinterpret_cast<const uint32_t*>(v));
        }
        tm_wait_st();
        meet();
        if (!ok) break;
      }
      float* po = nullptr;
      if (!run.whole && live && wt < parts.prow) {
        po = parts.o + part() * HD + hf * OW;
        if (hf == 0) *reinterpret_cast<float2*>(parts.ml + part() * 2) = make_float2(mx, l);
      }
      Q* out = (Q*)a.out + ((size_t)row * a.heads + (size_t)run.kvh * group + g) * HD + hf * OW;
      const bool write = run.whole && live && !(merge && t == 1);
      f2 odd[2] = {make_f2(0.f, 0.f), make_f2(0.f, 0.f)};  // 0 * O: NaN where O is not finite
#pragma unroll 1
      for (int k = 0; k < OW / 16; k++) {
        float v[16];
        __syncwarp();
        if (warp_live) {
          tm_ld16(op + k * 16, reinterpret_cast<uint32_t*>(v));
          tm_wait_ld16(reinterpret_cast<uint32_t*>(v));
        }
        if (merge) {
          if (t == 1) {
            if (nx > 0 && !(ok = wait_warp(xempty + 8 * hf, (nx - 1) & 1))) break;
#pragma unroll
            for (int e = 0; e < 16; e++) xb[e * 128 + wt] = v[e];
            arrive_warp(xfull + 8 * hf);
          } else {
            if (!(ok = wait_warp(xfull + 8 * hf, nx & 1))) break;
            if (k == 0) {
              const float2 ml = make_float2(sh.half[1][0][wt], sh.half[1][1][wt]);
              const float mn = fmaxf(mx, ml.x);
              own = l == 0.f ? 0.f : ex2(mx - mn);
              other = ml.y == 0.f ? 0.f : ex2(ml.x - mn);
              l = l * own + ml.y * other;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = v[e] * own + xb[e * 128 + wt] * other;
            arrive_warp(xempty + 8 * hf);
          }
          nx++;
        }
        if (po || write) {
#pragma unroll
          for (int e = 0; e < 8; e++) odd[e & 1] = fma2(make_f2(v[2 * e], v[2 * e + 1]), make_f2(0.f, 0.f), odd[e & 1]);
        }
        if (po) {
#pragma unroll
          for (int e = 0; e < 16; e += 4) st4(po + k * 16 + e, v + e);
        }
        if (write) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          if (l == 0.f) {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] = 0.f;
          }
          if constexpr (S::kSplit) {
#pragma unroll
            for (int e = 0; e < 16; e++) v[e] *= inv;
#pragma unroll
            for (int e = 0; e < 16; e += 4) st4((float*)out + k * 16 + e, v + e);
          } else {
            uint32_t w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = pack2(v[2 * e] * inv, v[2 * e + 1] * inv, C());
#pragma unroll
            for (int e = 0; e < 8; e += 4)
              *reinterpret_cast<uint4*>(out + k * 16 + 2 * e) = make_uint4(w[e], w[e + 1], w[e + 2], w[e + 3]);
          }
        }
      }
      odd[0] = add2(odd[0], odd[1]);
      if (lo_of(odd[0]) + hi_of(odd[0]) != 0.f) sh.odd = 1;  // NaN is unequal too
      // All warps have read the exchange's last round, and the other stream's (m, l),
      // before any of them copies the next run's queries: a pair's second query tile
      // takes the exchange's place.  (f32: they meet before every run.)
      if (!ok) break;
      if (!S::kSplit && merge && !(ok = meet_all(nx / (OW / 16) - 1))) break;  // nx: OW / 16 a merge
    }
  }
  fence_before();
  __syncthreads();
  if (warp == kTaSoft + kTaLoad) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
  if (tid == 0) parts.status[blockIdx.x] = (sh.fail ? kGaveUp : 0) | (sh.odd ? kOdd : 0);
}

// One (row, head) by the definition, a warp in f32, 32 keys at a time: the keys that
// the row does not attend are not touched.
template <int HD, class Q>
__device__ __noinline__ void row_again(const TreeAttnArgs& a, int i, int r, int head, float* s_q) {
  const Req q = request<Shape<HD, Q>::KT>(a, i);
  using C = typename std::conditional<Shape<HD, Q>::kSplit, __half, Q>::type;
  const int lane = threadIdx.x & 31, kvh = head / (a.heads / a.kv_heads);
  const int pos = a.pos[r] < 0 ? -1 : max(a.pos[r], q.len), end = pos < 0 ? 0 : q.keys;
  const Q* src = (const Q*)a.q + (size_t)r * a.ldq + (size_t)head * HD;
#pragma unroll
  for (int e = 0; e < HD / 32; e++) s_q[e * 32 + lane] = as_f32(src[e * 32 + lane]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, o[HD / 32] = {};
  for (int t0 = q.tile0 * Shape<HD, Q>::KT; t0 < end; t0 += 32) {
    const int t = t0 + lane, c = t - q.len;
    bool see = t < end;
    if (see && c >= 0)
      see = a.mask ? c < 32 * a.words && (a.mask[(size_t)r * a.words + (c >> 5)] >> (c & 31) & 1u) : c <= r - q.row0;
    if (see && a.window > 0) see = (c >= 0 ? max(a.pos[q.row0 + c], q.len) : t) > pos - a.window;
    const int page = see ? a.tables[(size_t)i * a.ld_tables + t / kKvPage] : -1;
    see = page >= 0 && page < a.n_pages;
    const size_t at = see ? (((size_t)page * a.kv_heads + kvh) * kKvPage + t % kKvPage) * HD : 0;
    float s = -INFINITY;
    if (see) {
      const uint4* k = reinterpret_cast<const uint4*>((const C*)a.cache_k + at);
      float acc = 0.f;
#pragma unroll 4
      for (int d = 0; d < HD / 8; d++) {
        const uint4 u = k[d];
        const C* x = reinterpret_cast<const C*>(&u);
#pragma unroll
        for (int e = 0; e < 8; e++) acc += s_q[d * 8 + e] * as_f32(x[e]);
      }
      s = acc * a.scale;
    }
    float mn = s;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, x));
    mn = fmaxf(m, mn);
    const float old = m == -INFINITY ? 0.f : expf(m - mn), p = s == -INFINITY ? 0.f : expf(s - mn);
    float sum = p, part[HD / 32] = {};
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    for (unsigned todo = __ballot_sync(0xffffffffu, p != 0.f); todo; todo &= todo - 1) {
      const float pk = __shfl_sync(0xffffffffu, p, __ffs(todo) - 1);
      const C* v = (const C*)a.cache_v + __shfl_sync(0xffffffffu, at, __ffs(todo) - 1) + lane;
#pragma unroll
      for (int e = 0; e < HD / 32; e++) part[e] += pk * as_f32(v[e * 32]);
    }
    l = l * old + sum;
    m = mn;
#pragma unroll
    for (int e = 0; e < HD / 32; e++) o[e] = o[e] * old + part[e];
  }
  Q* out = (Q*)a.out + ((size_t)r * a.heads + head) * HD + lane;
#pragma unroll
  for (int e = 0; e < HD / 32; e++) put(out + e * 32, l == 0.f ? 0.f : o[e] / l);
}

// Merges the parts of the groups that were cut: a warp per (row, head), its
// lanes a part each for the weights, then HD / 32 columns each.  A row of a call
// in which a CTA's wait gave up becomes NaN.
// A product takes every key of its tiles for every row, those that a row does not
// attend with P = 0.  inf or NaN in the V of one that another row does attend (a
// sibling in the tree, a later token of the chain, a token that only shallower rows
// have in their window) makes that 0 * NaN, so a row that comes out other than
// finite is worked out again without them (row_again).  That costs nothing where
// all is finite: the main kernel's CTAs say whether they saw anything else.
template <int HD, class Q>
__global__ void __launch_bounds__(128) k_tree_combine(const __grid_constant__ TreeAttnArgs a, const Parts parts, int ctas) {
  using S = Shape<HD, Q>;
  __shared__ float s_q[4][HD];
  const int lane = threadIdx.x & 31, r = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5);
  const int group = a.heads / a.kv_heads;
  pdl_wait();
  pdl_trigger();
  const int last = a.row_start[a.n];
  const long long signed_per = parts.start[a.n + 1], per = signed_per < 0 ? -signed_per : signed_per;
  if (head >= a.heads || r >= min(last, a.rows)) return;
  const Cut cut = {per, signed_per < 0};
  int lo = 0, hi = a.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a.row_start[mid + 1] > r) hi = mid;
    else lo = mid + 1;
  }
  const long long start = parts.start[lo];
  const Req q = request<S::KT>(a, lo);
  const int kvh = head / group, m = (r - q.row0) * group + head - kvh * group;
  const int qt0 = m / 128 / S::NS * S::NS, w = min(S::NS, q.qt - qt0), wt = m & 127;
  if (w < 1 || m < 0) return;
  const Groups<S::NS> g(q, cut);
  const long long g0 = start + kvh * g.all +
                       (w == 2 ? qt0 / 2 * g.pair : g.pairs * g.pair + (qt0 - 2 * g.pairs) * g.single);
  const long long g1 = g0 + (long long)w * q.kt;
  const int c0 = (int)quot(g0, per), c1 = (int)quot(g1 - 1, per);
  // parts: both streams of each CTA of the group, or the query tile's own
  const int nt = w == 2 ? 1 : S::NS, np = (c1 - c0 + 1) * nt;
  bool failed = false, odd = false, whole = false;
  float M = -INFINITY, L = 0.f, o[HD / 32];
#pragma unroll
  for (int e = 0; e < HD / 32; e++) o[e] = 0.f;
  for (int p0 = 0; p0 < np; p0 += 32) {
    const int p = p0 + lane, c = c0 + p / nt, t = w == 2 ? m / 128 - qt0 : p % nt;
    const long long s = max((long long)c * per, g0), e1 = min((long long)(c + 1) * per, g1);
    const int ta = (int)((s - g0) >> (w - 1)), tb = (int)((e1 - g0) >> (w - 1));
    const bool ok = p < np && tb > ta && (w == 2 || t < tb - ta);
    const size_t at = (((size_t)c * 2 + ((long long)c * per >= g0 ? 0 : 1)) * 2 + t) * parts.prow + wt;
    const int status = p < np ? parts.status[min(c, ctas - 1)] : 0;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (ok) ml = *reinterpret_cast<const float2*>(parts.ml + at * 2);
    failed |= __any_sync(0xffffffffu, status & kGaveUp);
    odd |= __any_sync(0xffffffffu, status & kOdd);
    if (__any_sync(0xffffffffu, ok && ta == 0 && tb == q.kt)) {  // one CTA had it all and wrote the row
      if (!failed && !odd) return;
      whole = true;
      break;
    }
    float top = ml.y == 0.f ? -INFINITY : ml.x;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float mn = fmaxf(M, top), old = M == -INFINITY ? 0.f : ex2(M - mn);
    const float f = ml.y == 0.f ? 0.f : ex2(ml.x - mn);
    float sum = ml.y * f;
    if (ml.y == 0.f) sum = 0.f;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    L = L * old + sum;
    M = mn;
#pragma unroll
    for (int e = 0; e < HD / 32; e++) o[e] *= old;
    const unsigned live = __ballot_sync(0xffffffffu, ml.y != 0.f);
#pragma unroll 4
    for (int k = 0; k < min(32, np - p0); k++) {
      const float fk = __shfl_sync(0xffffffffu, f, k);
      const size_t ak = __shfl_sync(0xffffffffu, at, k);
      if (live >> k & 1u) {
#pragma unroll
        for (int e = 0; e < HD / 32; e++) o[e] += parts.o[ak * HD + e * 32 + lane] * fk;
      }
    }
  }
  Q* out = (Q*)a.out + ((size_t)r * a.heads + head) * HD;
  if (odd && !failed) {
    bool again = false;
#pragma unroll
    for (int e = 0; e < HD / 32; e++) again |= !isfinite(whole ? as_f32(out[e * 32 + lane]) : L == 0.f ? 0.f : o[e]);
    if (__any_sync(0xffffffffu, again) && !(whole && a.q == a.out)) {  // in place the query is gone
      row_again<HD, Q>(a, lo, r, head, s_q[threadIdx.x >> 5]);
      return;
    }
    if (whole) return;
  }
#pragma unroll
  for (int e = 0; e < HD / 32; e++) put(out + e * 32 + lane, failed ? NAN : L == 0.f ? 0.f : o[e] / L);
}

int device_sms() {
  static int cache[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  int& n = cache[dev & 63];
  if (!n && (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)) n = 148;
  return n;
}

// the cache as rows of head_dim values, 16 rows of 64 columns a box
int cache_map(CUtensorMap* map, const void* base, bool bf16, int hd, size_t rows) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (Encode)f;
  }();
  if (!encode) return fail(WL_ERR_CUDA, "tree_attention: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)hd * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)kKvPage}, step[2] = {1, 1};
  const CUresult e = encode(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                            const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (e != CUDA_SUCCESS) return fail(WL_ERR_CUDA, "tree_attention: tensor map refused (" + std::to_string((int)e) + ")");
  return WL_OK;
}

template <int HD, class Q>
int launch_t(const TreeAttnArgs& a, cudaStream_t st) {
  using S = Shape<HD, Q>;
  CUtensorMap mk, mv;
  const size_t rows = (size_t)a.n_pages * a.kv_heads * kKvPage;
  WL_TRY(cache_map(&mk, a.cache_k, S::kBf16, HD, rows));
  WL_TRY(cache_map(&mv, a.cache_v, S::kBf16, HD, rows));
  const int ctas = device_sms();
  const Parts parts = parts_at(a.workspace, ctas, a.n, HD, part_rows(a.rows, a.heads / a.kv_heads));
  constexpr int smem = S::kTiles + (int)sizeof(Small<HD, Q>);
  WL_TRY(once_on_device((const void*)k_tree_attn<HD, Q>, []() -> int {
    WL_CUDA_TRY(cudaFuncSetAttribute(k_tree_attn<HD, Q>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    return WL_OK;
  }));
  WL_TRY(launch_step(k_tree_attn<HD, Q>, dim3(ctas), dim3(kTaThreads), smem, st, a, mk, mv, parts));
  return launch_step(k_tree_combine<HD, Q>, dim3(a.rows, (a.heads + 3) / 4), dim3(128), 0, st, a, parts, ctas);
}

template <class Q, class C>
int launch_hd(const TreeAttnArgs& a, cudaStream_t st) {
  switch (a.head_dim) {
    case 64: return launch_t<64, Q>(a, st);
    case 128: return launch_t<128, Q>(a, st);
    case 256: return launch_t<256, Q>(a, st);
  }
  return launch_step(k_tree_attn_row<Q, C>, dim3(a.rows, a.heads), dim3(128), 0, st, a);
}

}  // namespace

size_t tree_attention_workspace(int q_type, int n, int rows, int heads, int kv_heads, int head_dim) {
  (void)q_type;
  if (head_dim == 32) return 0;
  return part_bytes(device_sms(), n, head_dim, part_rows(rows, heads / kv_heads));
}

int launch_tree_attention(const TreeAttnArgs& a, cudaStream_t st) {
  if (a.q_type == WL_F32) return launch_hd<float, __half>(a, st);
  if (a.q_type == WL_F16) return launch_hd<__half, __half>(a, st);
  return launch_hd<__nv_bfloat16, __nv_bfloat16>(a, st);
}

}  // namespace wl
