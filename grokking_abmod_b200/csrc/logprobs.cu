// Log-probabilities of given tokens from rows of logits, with the rows'
// entropy and their k most likely tokens, and the gradient of the first two.
//
//   m = max_j x_j, d_j = x_j - m, s = sum_j e^d_j
//   lse = m + ln s, logprob = d_t - ln s, H = ln s - (sum_j e^d_j d_j) / s
//   dx_j = g (1[j = t] - p_j) - h p_j (ln p_j + H),  p_j = e^(x_j - lse)
//
// H is a sum of nonnegative terms, so nothing cancels where one token takes
// nearly all the probability.  The forward reads each logit once: every
// thread keeps a running (m, s, sum) of its own elements, rescaled when its
// maximum rises, and the triples are joined at the end in a fixed order.
//
// Top tokens order by (value descending, index ascending), a total order, so
// ties go to the lowest index whatever the launch shape.  The threads' maxima
// are known when the sums are: at least k elements reach the k-th largest of
// them, and few more do.  Only the threads whose maximum reaches it (k of
// them) look at their elements again; what they find is sorted in registers.
// Where fewer than k elements are not masked, the first masked ones follow
// them.  Rows where too many elements tie at the k-th, or with NaN, go through
// a slower list that is right for any row.

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.cuh"
#include "dtype.cuh"

namespace mb {
namespace logprobs {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kMaxTop = 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;      // 16-byte vectors a thread has in flight
constexpr int kAgain = 4;       // the same where it looks for top tokens
constexpr int kRowLanes = 1024; // vocabularies up to here take one warp per row, however few the rows
// So many top tokens of a row in registers are picked one by one, more are
// sorted: 4656 x 97 FP32, picked against sorted, 3.6 : 5.3 us for one, 5.4 : 5.4
// for 5, 6.0 : 5.5 for 6, 11.7 : 5.7 for 20.
constexpr int kFewTop = 6;
constexpr unsigned kFull = 0xFFFFFFFFu;

using u64 = unsigned long long;

// Running statistics in base-2 units: s = sum 2^t, a = sum 2^t t with
// t = (x - m) log2 e <= 0.
struct Stats {
  float m, s, a;
};

__device__ __forceinline__ Stats empty_stats() { return Stats{-INFINITY, 0.f, 0.f}; }

// Moves the statistics to a maximum m >= s.m.
__device__ __forceinline__ Stats rebase(Stats s, float m) {
  if (s.m == -INFINITY) return Stats{m, s.s, s.a};  // nothing counted (or only NaN terms)
  const float t = fmaxf((s.m - m) * kLog2e, -1e30f);
  const float c = ex2_ftz(t);
  return Stats{m, s.s * c, c * fmaf(t, s.s, s.a)};
}

__device__ __forceinline__ Stats join(Stats p, Stats q) {
  // a maximum of -inf on both sides: sums of empty sets, or NaN that stay NaN
  const float m = fmaxf(p.m, q.m);
  if (m == -INFINITY) return Stats{m, p.s + q.s, p.a + q.a};
  p = rebase(p, m);
  q = rebase(q, m);
  return Stats{m, p.s + q.s, p.a + q.a};
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}

__device__ __forceinline__ Stats warp_join(Stats v) {
  const float m = warp_max(v.m);
  if (m != -INFINITY) v = rebase(v, m);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    v.s += __shfl_xor_sync(kFull, v.s, o);
    v.a += __shfl_xor_sync(kFull, v.a, o);
  }
  return v;
}

// Adds N elements whose largest is mx.
template <int N>
__device__ __forceinline__ void accumulate(Stats& st, const float (&x)[N], float mx) {
  if (mx > st.m) st = rebase(st, mx);
  // all of them -inf so far: differences from 0 keep the terms at 2^-inf = 0
  const float2 less = splat2(st.m == -INFINITY ? 0.f : -st.m), scale = splat2(kLog2e);
  float2 s = make_float2(0.f, 0.f), a = make_float2(0.f, 0.f);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 t = mul2(add2(make_float2(x[i], x[i + 1]), less), scale);
    const float2 e = make_float2(ex2_ftz(t.x), ex2_ftz(t.y));
    s = add2(s, e);
    // a masked logit (-inf, or the type's lowest) may have t = -inf and has
    // e = 0: its term is 0, not NaN
    a = fma2(e, make_float2(fmaxf(t.x, -1e30f), fmaxf(t.y, -1e30f)), a);
  }
  st.s += s.x + s.y;
  st.a += a.x + a.y;
}

// The order of the top list: larger keys first.  -0 counts as +0, NaN above
// everything; 0 is below every element.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  if (x != x) return 0xFFFFFFFFu;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
constexpr uint32_t kUnmasked = 0x00800000u;  // the key above that of -inf: of the lowest finite value
__device__ __forceinline__ float unordered(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}
__device__ __forceinline__ u64 top_key(float x, uint32_t index) { return ((u64)ordered(x) << 32) | (uint32_t)~index; }

// Inserts a warp-uniform key into the warp's list (lane i holds the i-th
// largest).  The keys of a row are distinct.
__device__ __forceinline__ void insert(u64& mine, u64 key, int lane) {
  const int pos = __popc(__ballot_sync(kFull, mine > key));
  const u64 up = __shfl_up_sync(kFull, mine, 1);
  if (lane == pos) mine = key;
  if (lane > pos) mine = up;
}

// Offers each lane's key to the list; keys at or below `floor` are out.
__device__ __forceinline__ void offer(u64& mine, u64 key, u64 floor, int top, int lane) {
  u64 least = __shfl_sync(kFull, mine, top - 1);
  if (least < floor) least = floor;
  unsigned who = __ballot_sync(kFull, key > least);
  while (who) {
    const int src = __ffs(who) - 1;
    who &= who - 1;
    const u64 k = __shfl_sync(kFull, key, src);
    if (k > least) {
      insert(mine, k, lane);
      least = __shfl_sync(kFull, mine, top - 1);
      if (least < floor) least = floor;
    }
  }
}

// Sorting across a warp, largest in lane 0: a bitonic network.
template <class K>
__device__ __forceinline__ K merge_step(K v, int o, bool keep_larger) {
  const K w = __shfl_xor_sync(kFull, v, o);
  return (v > w) == keep_larger ? v : w;
}
template <class K>
__device__ __forceinline__ K warp_sort(K v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k *= 2)
#pragma unroll
    for (int o = k / 2; o; o /= 2) v = merge_step(v, o, ((lane & o) == 0) == ((lane & k) == 0));
  return v;
}
// The 32 largest of two sorted lists; `reversed`: the other list's lane 31 - lane.
template <class K>
__device__ __forceinline__ K warp_merge(K v, K reversed, int lane) {
  v = v > reversed ? v : reversed;  // a bitonic sequence
#pragma unroll
  for (int o = 16; o; o /= 2) v = merge_step(v, o, (lane & o) == 0);
  return v;
}
// The 32 largest of n keys in shared memory, sorted.
__device__ __forceinline__ u64 sort_found(const u64* at, int n, int lane) {
  u64 v = warp_sort(lane < n ? at[lane] : 0ull, lane);
  for (int b = 32; b < n; b += 32) {
    const u64 other = warp_sort(b + lane < n ? at[b + lane] : 0ull, lane);
    v = warp_merge(v, __shfl_sync(kFull, other, 31 - lane), lane);
  }
  return v;
}
// The same over sorted lists in shared memory, one a warp (n of them, a power
// of two): the result is warp 0's.  The lists are in place and synchronised.
template <class K>
__device__ __forceinline__ K tree_merge(K (*lists)[32], int n, int warp, int lane) {
  K v = warp < n ? lists[warp][lane] : 0;
  for (n /= 2; n; n /= 2) {
    if (warp < n) {
      v = warp_merge(v, lists[warp + n][31 - lane], lane);
      lists[warp][lane] = v;
    }
    __syncthreads();
  }
  return v;
}

struct Out {
  float *logprob, *entropy, *lse, *top_logprob;
  int* top_index;
  int* status;
};

// ln p of a logit x.  x - lse would carry the rounding of lse, as large as that of
// the logits, where ln p is small.
__device__ __forceinline__ float log_p(float x, Stats st, float log_s) {
  return (x - st.m) - log_s;
}

// A row's statistics; t its token, valid: inside the vocabulary, xt its logit.
// Returns ln s.
__device__ __forceinline__ float store_row(const Out& o, size_t row, Stats st, int t, bool valid, float xt) {
  const bool none = st.m == -INFINITY && st.s == 0.f;  // every token masked
  const float log_s = logf(st.s);
  o.lse[row] = none ? -INFINITY : (st.m == -INFINITY ? st.s : st.m + log_s);
  o.entropy[row] = none ? 0.f : log_s - st.a / st.s * kLn2;
  if (t != -1 && !valid && o.status) atomicOr(o.status, 2);
  o.logprob[row] = t == -1 ? 0.f : !valid ? NAN : none ? -INFINITY : log_p(xt, st, log_s);
  return log_s;
}

// Writes a row's results; one warp, with the joined statistics in every lane
// and the list in its lanes.
template <class T>
__device__ __forceinline__ void finish(const Out& o, size_t row, const T* x, int vocab, const int* tokens, int top,
                                       Stats st, u64 mine, int lane) {
  float log_s = 0.f;
  if (lane == 0) {
    const int t = tokens[row];
    const bool valid = (unsigned)t < (unsigned)vocab;
    log_s = store_row(o, row, st, t, valid, valid ? Element<T>::to(x[t]) : 0.f);
  }
  log_s = __shfl_sync(kFull, log_s, 0);
  if (lane < top) {
    const float v = unordered((uint32_t)(mine >> 32));
    o.top_logprob[row * top + lane] = v == -INFINITY ? v : log_p(v, st, log_s);
    o.top_index[row * top + lane] = (int)~(uint32_t)mine;
  }
}

// One warp per row, the whole row in registers (R elements a lane): small
// vocabularies, where a row is less work than a CTA's joining.  Bound by the
// latency of one row: 4656 x 97 FP32 with 5 top tokens 5.4 us, 0.3 of it bytes.
template <class T, int R>
__global__ void __launch_bounds__(kThreads)
    forward_small(const T* __restrict__ logits, size_t stride, size_t rows, int vocab, const int* __restrict__ tokens,
                  int top, Out o) {
  __shared__ u64 found[kWarps][32 * R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const size_t row = (size_t)blockIdx.x * kWarps + warp;
  if (row >= rows) return;
  const T* x = logits + row * stride;
  float v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = lane + 32 * r < vocab ? Element<T>::to(x[lane + 32 * r]) : -INFINITY;
  float mx = v[0];
#pragma unroll
  for (int r = 1; r < R; ++r) mx = fmaxf(mx, v[r]);
  mx = warp_max(mx);
  Stats st = empty_stats();
  accumulate(st, v, mx);
#pragma unroll
  for (int i = 16; i; i >>= 1) {
    st.s += __shfl_xor_sync(kFull, st.s, i);
    st.a += __shfl_xor_sync(kFull, st.a, i);
  }
  u64 mine = 0;
  if (top > kFewTop) {
    u64 key[R], best = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      key[r] = lane + 32 * r < vocab ? top_key(v[r], lane + 32 * r) : 0;
      best = key[r] > best ? key[r] : best;
    }
    if (R == 2) {
      const u64 other = warp_sort(key[1], lane);
      mine = warp_merge(warp_sort(key[0], lane), __shfl_sync(kFull, other, 31 - lane), lane);
    } else {
      // the k-th largest lane maximum (0 where fewer lanes hold elements) and what reaches it
      const u64 least = __shfl_sync(kFull, warp_sort(best, lane), top - 1);
      int count = 0;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool in = key[r] >= least && key[r] != 0;
        const unsigned who = __ballot_sync(kFull, in);
        const int at = count + __popc(who & ((1u << lane) - 1));
        if (in) found[warp][at] = key[r];
        count += __popc(who);
      }
      __syncwarp();
      mine = sort_found(found[warp], count, lane);
    }
  } else if (top) {
    // few: the largest key of all lanes, taken out of the lane it is in, k times
    uint32_t best = 0, at = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t k = lane + 32 * r < vocab ? ordered(v[r]) : 0u;
      if (k > best) best = k, at = r;
    }
    uint32_t taken = 0;  // bit r: v[r] is in the list
    for (int i = 0; i < top; ++i) {
      const uint32_t k = __reduce_max_sync(kFull, best);
      const uint32_t index = __reduce_min_sync(kFull, best == k ? lane + 32u * at : kFull);
      if (lane == i) mine = ((u64)k << 32) | (uint32_t)~index;
      if (lane == (int)(index & 31u)) {
        taken |= 1u << at;
        best = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint32_t c = lane + 32 * r < vocab && !((taken >> r) & 1u) ? ordered(v[r]) : 0u;
          if (c > best) best = c, at = r;
        }
      }
    }
  }
  finish(o, row, x, vocab, tokens, top, st, mine, lane);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// Reads 4 bytes at the address that `p` has in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t remote_u32(const void* p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), v;
  asm volatile(
      "{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.u32 %0, [r];\n\t}"
      : "=r"(v)
      : "r"(a), "r"(rank)
      : "memory");
  return v;
}

// Eight lanes per row, R elements a lane, without top tokens: the smallest
// vocabularies are all latency, and four rows a warp share it.  32768 x 64 FP32:
// 3.5 us against 7.5 with a warp a row (2.4 TB/s, from L2).
template <class T, int R>
__global__ void __launch_bounds__(kThreads)
    forward_narrow(const T* __restrict__ logits, size_t stride, size_t rows, int vocab, const int* __restrict__ tokens,
                   Out o) {
  constexpr int G = 8;
  const int id = threadIdx.x % G;
  const size_t at = (size_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  const size_t row = at < rows ? at : rows - 1;  // whole warps shuffle; rows past the last are not stored
  const T* x = logits + row * stride;
  const int t = tokens[row];
  const bool valid = (unsigned)t < (unsigned)vocab;
  const float xt = valid ? Element<T>::to(x[t]) : 0.f;
  float v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = id + G * r < vocab ? Element<T>::to(x[id + G * r]) : -INFINITY;
  float mx = v[0];
#pragma unroll
  for (int r = 1; r < R; ++r) mx = fmaxf(mx, v[r]);
#pragma unroll
  for (int i = G / 2; i; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, i));
  Stats st = empty_stats();
  accumulate(st, v, mx);
#pragma unroll
  for (int i = G / 2; i; i >>= 1) {
    st.s += __shfl_xor_sync(kFull, st.s, i);
    st.a += __shfl_xor_sync(kFull, st.a, i);
  }
  if (id == 0 && at < rows) store_row(o, row, st, t, valid, xt);
}

// The largest of a 16-byte vector's elements.
template <class T>
__device__ __forceinline__ float vector_max(uint4 raw) {
  if constexpr (sizeof(T) == 4) {
    return fmaxf(fmaxf(__uint_as_float(raw.x), __uint_as_float(raw.y)),
                 fmaxf(__uint_as_float(raw.z), __uint_as_float(raw.w)));
  } else {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* h = reinterpret_cast<const T2*>(&raw);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(Element<T>::to(m.x), Element<T>::to(m.y));
  }
}

// Rows of W warps each: 1 (kWarps rows a CTA), or kWarps with a cluster of
// CTAs per row, each on a contiguous share of it.  The ragged head and tail
// around the 16-byte aligned body (odd vocabularies leave rows unaligned) are
// fewer than 2 VEC elements, one more for the group's first threads.  Bound by
// exponentials and instruction issue in 16 bits, by HBM in FP32: 4096 x 32003
// without top tokens 53 us (4.9 TB/s) and 84 us (6.2 TB/s), with one 69 and 95.
template <class T, int W, bool TOP>
__global__ void __launch_bounds__(kThreads)
    forward_wide(const T* __restrict__ logits, size_t stride, size_t rows, int vocab, const int* __restrict__ tokens,
                 int top, Out o) {
  constexpr int VEC = Element<T>::kVec, N = kUnroll * VEC, GROUP = 32 * W;
  constexpr int kFound = 256;  // candidates of a group
  __shared__ Stats warp_stats[kWarps];
  __shared__ u64 lists[kWarps][32];
  __shared__ uint32_t maxima[kWarps][32];
  __shared__ u64 found[W == 1 ? kWarps : 1][kFound];
  __shared__ int counts[W == 1 ? kWarps : 1];
  __shared__ uint32_t limit;  // of one row, W > 1
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int id = W == 1 ? lane : threadIdx.x, group = W == 1 ? warp : 0;
  const uint32_t rank = W == 1 ? 0 : cluster_rank(), ranks = W == 1 ? 1 : cluster_size();
  const size_t row = W == 1 ? (size_t)blockIdx.x * kWarps + warp : blockIdx.x / ranks;
  if (W == 1 && row >= rows) return;
  const T* x = logits + row * stride;

  const int lead = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T));
  const int head = lead < vocab ? lead : vocab;
  const int vectors = (vocab - head) / VEC;
  const int tail = head + vectors * VEC;  // [tail, vocab) is left over
  const int share = (vectors + ranks - 1) / ranks;
  const int begin = min(vectors, (int)rank * share), end = min(vectors, begin + share);
  const uint4* body = reinterpret_cast<const uint4*>(x + head);
  const int left = rank == 0 ? head + vocab - tail : 0;
  const int left_at = id < head ? id : tail + id - head;

  Stats st = empty_stats();
  int best_at = begin + id;  // the step that raised the maximum last: the first with it
  for (int j = begin + id; j < end; j += GROUP * kUnroll) {
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (j + u * GROUP < end) raw[u] = __ldg(body + j + u * GROUP);
    if (j + (kUnroll - 1) * GROUP < end) {
      float v[N], mx = vector_max<T>(raw[0]);
#pragma unroll
      for (int u = 1; u < kUnroll; ++u) mx = fmaxf(mx, vector_max<T>(raw[u]));
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) Element<T>::unpack(raw[u], v + u * VEC);
      if (TOP && mx > st.m) best_at = j;
      accumulate(st, v, mx);
    } else {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * GROUP < end) {
          float v[VEC];
          Element<T>::unpack(raw[u], v);
          if (TOP && vector_max<T>(raw[u]) > st.m) best_at = j;
          accumulate(st, v, vector_max<T>(raw[u]));
        }
    }
  }
  if (id < left) {
    float v[2] = {Element<T>::to(x[left_at]), -INFINITY};
    accumulate(st, v, v[0]);
  }
  // this thread's largest element in the list's order; NaN, which a maximum
  // does not show, above all
  const uint32_t reach = st.s == st.s ? ordered(st.m) : 0xFFFFFFFFu;

  st = warp_join(st);
  u64 mine = 0;
  if constexpr (TOP) {
    // of one top token only the largest is needed
    uint32_t sorted = top > 1 ? warp_sort(reach, lane) : __reduce_max_sync(kFull, reach);
    if (id == 0) counts[group] = 0;
    if (W > 1) {
      maxima[warp][lane] = sorted;
      __syncthreads();
      if (top > 1) {
        sorted = tree_merge(maxima, kWarps, warp, lane);
      } else {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sorted = max(sorted, maxima[w][0]);
      }
      // NaN anywhere: no limit
      const bool nan = __shfl_sync(kFull, sorted, 0) == 0xFFFFFFFFu;
      if (warp == 0 && lane == top - 1) limit = nan ? 0 : max(sorted, kUnmasked);
      __syncthreads();
    } else {
      __syncwarp();
    }
    uint32_t least = limit;
    if (W == 1)
      least = __shfl_sync(kFull, sorted, 0) == 0xFFFFFFFFu ? 0 : max(__shfl_sync(kFull, sorted, top - 1), kUnmasked);
    const bool plain = least != 0;
    if (plain && reach >= least) {
      auto take = [&](float v, int index) {
        if (ordered(v) >= least) {
          const int at = atomicAdd(&counts[group], 1);
          if (at < kFound) found[group][at] = top_key(v, (uint32_t)index);
        }
      };
      // of one top token the step that holds the thread's first largest element is enough
      static_assert(kAgain == kUnroll, "steps");
      const int last = top == 1 ? min(end, best_at + GROUP * kAgain) : end;
      for (int j = top == 1 ? best_at : begin + id; j < last; j += GROUP * kAgain) {
        uint4 raw[kAgain];
#pragma unroll
        for (int u = 0; u < kAgain; ++u)
          if (j + u * GROUP < end) raw[u] = __ldg(body + j + u * GROUP);
        unsigned hits = 0;
#pragma unroll
        for (int u = 0; u < kAgain; ++u)
          if (j + u * GROUP < end && ordered(vector_max<T>(raw[u])) >= least) hits |= 1u << u;
        while (hits) {
          const int at = j + (__ffs(hits) - 1) * GROUP;
          hits &= hits - 1;
          float v[VEC];
          Element<T>::unpack(__ldg(body + at), v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) take(v[i], head + at * VEC + i);
        }
      }
      if (id < left) take(Element<T>::to(x[left_at]), left_at);
    }
    if (W > 1) __syncthreads();
    else __syncwarp();
    if (plain && least == kUnmasked && counts[group] < top) {
      // every element that is not masked is found: the first masked ones
      // follow, and the first 2 kMaxTop elements hold as many as are wanted
      if (W > 1) __syncthreads();
      else __syncwarp();
      const int begins = rank == 0 ? 0 : head + begin * VEC, ends = rank == 0 && ranks == 1 ? vocab : head + end * VEC;
      for (int i = id; i < 2 * kMaxTop; i += GROUP)
        if (begins + i < ends && ordered(Element<T>::to(x[begins + i])) < kUnmasked) {
          const int at = atomicAdd(&counts[group], 1);
          if (at < kFound) found[group][at] = top_key(-INFINITY, (uint32_t)(begins + i));
        }
      if (W > 1) __syncthreads();
      else __syncwarp();
    }
    const int count = counts[group];
    if (plain && count >= top && count <= kFound) {
      if (W == 1) mine = sort_found(found[group], count, lane);
      else if (32 * warp < count) mine = sort_found(found[group] + 32 * warp, min(32, count - 32 * warp), lane);
    } else {
      // any row: a sorted list a warp, every element offered to it
      for (int j = begin + (id & ~31); j < end; j += GROUP) {
        const bool there = j + lane < end;
        float v[VEC];
        Element<T>::unpack(there ? __ldg(body + j + lane) : make_uint4(0u, 0u, 0u, 0u), v);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          offer(mine, there ? top_key(v[i], (uint32_t)(head + (j + lane) * VEC + i)) : 0ull, 0, top, lane);
      }
      if (id < 32)
        offer(mine, id < left ? top_key(Element<T>::to(x[left_at]), (uint32_t)left_at) : 0ull, 0, top, lane);
    }
  }
  if (W > 1) {
    if (lane == 0) warp_stats[warp] = st;
    if (TOP) lists[warp][lane] = mine;
    __syncthreads();
    st = warp_stats[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) st = join(st, warp_stats[w]);
    if (TOP) mine = tree_merge(lists, kWarps, warp, lane);
    if (ranks > 1) {
      // the cluster's first CTA reads the others' results, a warp each
      __syncthreads();
      if (threadIdx.x == 0) warp_stats[0] = st;
      cluster_sync();
      Stats q = empty_stats();
      u64 theirs = 0;
      if (rank == 0 && warp < (int)ranks) {
        q.m = __uint_as_float(remote_u32(&warp_stats[0].m, warp));
        q.s = __uint_as_float(remote_u32(&warp_stats[0].s, warp));
        q.a = __uint_as_float(remote_u32(&warp_stats[0].a, warp));
        if (TOP) {
          const uint32_t* at = reinterpret_cast<const uint32_t*>(&lists[0][lane]);
          theirs = (u64)remote_u32(at + 1, warp) << 32 | remote_u32(at, warp);
        }
      }
      cluster_sync();  // read before any of it is written again
      if (rank != 0) return;
      if (lane == 0) warp_stats[warp] = q;
      lists[warp][lane] = theirs;
      __syncthreads();
      st = warp_stats[0];
      for (uint32_t r = 1; r < ranks; ++r) st = join(st, warp_stats[r]);
      if (TOP) mine = tree_merge(lists, (int)ranks, warp, lane);
    }
  }
  if (W == 1 || warp == 0) finish(o, row, x, vocab, tokens, TOP ? top : 0, st, mine, lane);
}

// ---------------------------------------------------------------- gradient
// Per row: the coefficients of dx_j = [j = t] g - p_j (g + h (ln p_j + H)).
struct RowGrad {
  float lse, g, h, gh;  // gh = g + h H
  int token;
  bool none;
};

struct GradIn {
  const int* tokens;
  const float *lse, *entropy, *dlogprob, *dentropy;
  int* status;
};

__device__ __forceinline__ RowGrad row_grad(const GradIn& in, size_t row, int vocab, bool report) {
  RowGrad r;
  r.lse = in.lse[row];
  r.token = in.tokens[row];
  r.none = r.lse == -INFINITY;  // nothing to move
  r.g = in.dlogprob && r.token != -1 ? in.dlogprob[row] : 0.f;
  r.h = in.dentropy ? in.dentropy[row] : 0.f;
  r.gh = r.h != 0.f ? fmaf(r.h, in.entropy[row], r.g) : r.g;
  if (r.token != -1 && (unsigned)r.token >= (unsigned)vocab) {
    r.g = r.gh = NAN;
    if (report && in.status) atomicOr(in.status, 2);
  }
  return r;
}

__device__ __forceinline__ float element_grad(const RowGrad& r, float x, int j) {
  const float logp = x - r.lse;
  const float p = ex2_ftz(logp * kLog2e);
  // p = 0 where the token is masked: its ln p is not looked at
  float d = -p * fmaf(r.h, fmaxf(logp, -1e30f), r.gh);
  if (j == r.token) d += r.g;
  return r.none ? 0.f : d;
}

// A group of G threads per row (8, a warp, or the CTA).  One read and one
// write of the logits, bound by HBM: 4096 x 32003 bfloat16 86 us (6.1 TB/s).
// Groups of 8 hold the smallest rows: 32768 x 64 FP32 4.0 us, 8.5 with a warp.
template <class T, int G>
__global__ void __launch_bounds__(kThreads)
    backward_rows(const T* __restrict__ logits, size_t stride, size_t rows, int vocab, GradIn in,
                  T* __restrict__ dlogits) {
  constexpr int VEC = Element<T>::kVec;
  const int id = threadIdx.x % G;
  const size_t row = (size_t)blockIdx.x * (kThreads / G) + threadIdx.x / G;
  if (row >= rows) return;
  const T* x = logits + row * stride;
  T* d = dlogits + row * vocab;
  const RowGrad r = row_grad(in, row, vocab, id == 0);
  const int part = G == kThreads ? blockIdx.y : 0, parts = G == kThreads ? gridDim.y : 1;
  if (((uintptr_t)x & 15) == ((uintptr_t)d & 15)) {
    const int lead = (int)(((16 - ((uintptr_t)x & 15)) & 15) / sizeof(T));
    const int head = lead < vocab ? lead : vocab;
    const int vectors = (vocab - head) / VEC, tail = head + vectors * VEC;
    const uint4* bx = reinterpret_cast<const uint4*>(x + head);
    uint4* bd = reinterpret_cast<uint4*>(d + head);
    for (int j = part * G * kUnroll + id; j < vectors; j += parts * G * kUnroll) {
      uint4 raw[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * G < vectors) raw[u] = __ldg(bx + j + u * G);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j + u * G < vectors) {
          float v[VEC];
          Element<T>::unpack(raw[u], v);
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[i] = element_grad(r, v[i], head + (j + u * G) * VEC + i);
          bd[j + u * G] = Element<T>::pack(v);
        }
    }
    // fewer than 2 VEC elements left over
#pragma unroll
    for (int i = id; i < 2 * VEC; i += G) {
      if (part != 0 || i >= head + vocab - tail) break;
      const int at = i < head ? i : tail + i - head;
      d[at] = Element<T>::from(element_grad(r, Element<T>::to(x[at]), at));
    }
  } else {
    for (int j = part * G + id; j < vocab; j += parts * G)
      d[j] = Element<T>::from(element_grad(r, Element<T>::to(x[j]), j));
  }
}

// CTAs per row: enough rows fill the GPU with one each; few rows are cut into
// up to 8 shares (the portable cluster size) of at least 4096 elements.
// Longer vocabularies than kRowLanes take a warp a row too where the rows are
// many: their joins cost a CTA more than its share of the row.  CTA : warp, us,
// bfloat16 without and with 20 top tokens: 600 x 2000 4.7 : 3.9, 9.4 : 10.7;
// 1184 x 2000 6.7 : 4.1, 14.7 : 11.1; 1184 x 4000 7.4 : 5.3, 16.5 : 22.5; 2400 x
// 4000 12.2 : 8.1, 28.8 : 25.1; 2400 x 8000 15.0 : 12.8, 32.3 : 37.3; 4096 x 8000
// 22.9 : 16.2, 50.5 : 42.8; 16384 x 16000 124 : 88, 256 : 233.  Up to kRowLanes
// always: 64 x 500 3.3 : 2.8, 4096 x 1000 14.2 : 5.4.
inline bool warp_rows(size_t rows, uint32_t vocab) {
  return vocab <= (uint32_t)kRowLanes || (vocab <= 16384 && rows * 2 >= vocab);
}

// The gradient has no join, so a CTA loses less: 16384 x 2000 47 : 25 us, 4096 x
// 4000 12.9 : 11.4 (FP32 21.4 : 20.7); 2400 x 4000 8.5 : 8.9 (FP32 8.9 : 10.8);
// 4096 x 8000 FP32 42.6 : 48.8; 64 x 4000 2.4 : 5.1.
inline bool warp_rows_backward(size_t rows, uint32_t vocab) {
  return vocab <= (uint32_t)kRowLanes || (vocab <= 4096 && rows >= vocab);
}

inline unsigned row_shares(size_t rows, int vocab) {
  const size_t want = (size_t)sm_count() * 4;
  unsigned n = 1;
  while (n < 8 && rows * n * 2 <= want && vocab / (int)(n * 2) >= 4096) n *= 2;
  return n;
}

inline void shape(size_t rows, uint32_t vocab, size_t stride) {
  require(rows >= 1 && rows <= (size_t)INT_MAX / 8, "rows must be in 1..2^28");
  require(vocab >= 1 && vocab <= (1u << 30), "vocab must be in 1..2^30");
  require(stride >= vocab || rows == 1, "the row stride must be at least vocab");
}

template <class T, int R>
void launch_small(const T* x, size_t stride, size_t rows, uint32_t vocab, const int* tokens, uint32_t top, const Out& o,
                  cudaStream_t st) {
  forward_small<T, R><<<(unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, st>>>(x, stride, rows, (int)vocab,
                                                                                    tokens, (int)top, o);
}

template <class T, bool TOP>
void launch_wide(const T* x, size_t stride, size_t rows, uint32_t vocab, const int* tokens, uint32_t top, const Out& o,
                 cudaStream_t st) {
  if (warp_rows(rows, vocab)) {
    forward_wide<T, 1, TOP><<<(unsigned)((rows + kWarps - 1) / kWarps), kThreads, 0, st>>>(
        x, stride, rows, (int)vocab, tokens, (int)top, o);
    return;
  }
  const unsigned shares = row_shares(rows, (int)vocab);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * shares));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = shares;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  launched("token log-probabilities",
           cudaLaunchKernelEx(&cfg, forward_wide<T, kWarps, TOP>, x, stride, rows, (int)vocab, tokens, (int)top, o));
}

template <class T>
void launch_forward(const T* x, size_t stride, size_t rows, uint32_t vocab, const int* tokens, uint32_t top,
                    const Out& o, cudaStream_t st) {
  if (vocab <= 128 && top == 0) {
    const unsigned blocks = (unsigned)((rows + kThreads / 8 - 1) / (kThreads / 8));
    if (vocab <= 64) forward_narrow<T, 8><<<blocks, kThreads, 0, st>>>(x, stride, rows, (int)vocab, tokens, o);
    else forward_narrow<T, 16><<<blocks, kThreads, 0, st>>>(x, stride, rows, (int)vocab, tokens, o);
    return;
  }
  if (vocab <= 64) return launch_small<T, 2>(x, stride, rows, vocab, tokens, top, o, st);
  if (vocab <= 128) return launch_small<T, 4>(x, stride, rows, vocab, tokens, top, o, st);
  if (top) launch_wide<T, true>(x, stride, rows, vocab, tokens, top, o, st);
  else launch_wide<T, false>(x, stride, rows, vocab, tokens, 0, o, st);
}

}  // namespace logprobs
}  // namespace mb

extern "C" {

int mb_op_token_logprobs(const mb_token_logprobs_args* a, void* stream) {
  using namespace mb::logprobs;
  return mb::guarded([&] {
    mb::need(a, "args");
    const uint32_t top = a->top;
    mb::need(a->logits, "logits");
    mb::need(a->tokens, "tokens");
    mb::need(a->logprob, "logprob");
    mb::need(a->entropy, "entropy");
    mb::need(a->lse, "lse");
    shape(a->rows, a->vocab, a->row_stride);
    mb::require(top <= (uint32_t)kMaxTop && top <= a->vocab, "top must be in 0..32 and at most vocab");
    if (top) {
      mb::need(a->top_logprob, "top_logprob");
      mb::need(a->top_index, "top_index");
    }
    const Out o{a->logprob, a->entropy, a->lse, a->top_logprob, a->top_index, a->d_status};
    mb::with_dtype(a->dtype, [&](auto tag) {
      using T = typename decltype(tag)::type;
      mb::aligned_to(a->logits, sizeof(T), "logits must be aligned to their elements");
      launch_forward<T>(static_cast<const T*>(a->logits), a->row_stride, a->rows, a->vocab, a->tokens, top, o,
                        (cudaStream_t)stream);
      mb::launched("token log-probabilities");
    });
  });
}

int mb_op_token_logprobs_backward(const mb_token_logprobs_backward_args* a, void* stream) {
  using namespace mb::logprobs;
  return mb::guarded([&] {
    mb::need(a, "args");
    mb::need(a->logits, "logits");
    mb::need(a->tokens, "tokens");
    mb::need(a->lse, "lse");
    mb::need(a->dlogits, "dlogits");
    if (a->dentropy) mb::need(a->entropy, "entropy");
    shape(a->rows, a->vocab, a->row_stride);
    const GradIn in{a->tokens, a->lse, a->entropy, a->dlogprob, a->dentropy, a->d_status};
    cudaStream_t st = (cudaStream_t)stream;
    mb::with_dtype(a->dtype, [&](auto tag) {
      using T = typename decltype(tag)::type;
      mb::aligned_to(a->logits, sizeof(T), "logits must be aligned to their elements");
      mb::aligned_to(a->dlogits, sizeof(T), "dlogits must be aligned to their elements");
      const T* x = static_cast<const T*>(a->logits);
      T* d = static_cast<T*>(a->dlogits);
      const size_t rows = a->rows;
      const uint32_t vocab = a->vocab;
      if (warp_rows_backward(rows, vocab)) {
        // 8 threads where they hold the row in their vectors in flight
        if (vocab * sizeof(T) <= 8 * kUnroll * 16) {
          const unsigned blocks = (unsigned)((rows + kThreads / 8 - 1) / (kThreads / 8));
          backward_rows<T, 8><<<blocks, kThreads, 0, st>>>(x, a->row_stride, rows, (int)vocab, in, d);
        } else {
          const unsigned blocks = (unsigned)((rows + kWarps - 1) / kWarps);
          backward_rows<T, 32><<<blocks, kThreads, 0, st>>>(x, a->row_stride, rows, (int)vocab, in, d);
        }
      } else {
        backward_rows<T, kThreads><<<dim3((unsigned)rows, row_shares(rows, (int)vocab)), kThreads, 0, st>>>(
            x, a->row_stride, rows, (int)vocab, in, d);
      }
      mb::launched("token log-probability gradient");
    });
  });
}

}  // extern "C"
