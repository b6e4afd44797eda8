// Writing new rows of K and V into the 8-bit paged cache, and reading a range
// of it back as floats.  Both move each byte once: the write reads a page's
// new rows into registers, reduces their largest magnitude, and stores the
// codes from the registers; the read loads codes and stores values.

#include <algorithm>
#include <climits>

#include "cache_host.h"
#include "dtype.cuh"

namespace mb {
namespace cache {

constexpr int kThreads = 256;

template <class T>
struct Rows {
  const T* p;
  size_t row_stride, head_stride;
  bool vector;  // base and strides allow 16-byte loads
};

// VEC channels [c, c + VEC) of a row; channels from head_dim on are 0.
template <class T>
__device__ __forceinline__ uint4 load_chunk(const Rows<T>& rows, size_t row, int head, int c, int head_dim) {
  constexpr int VEC = Element<T>::kVec;
  const T* p = rows.p + row * rows.row_stride + (size_t)head * rows.head_stride + c;
  if (rows.vector && c + VEC <= head_dim) return __ldg(reinterpret_cast<const uint4*>(p));
  union {
    uint4 v;
    T e[VEC];
  } u;
#pragma unroll
  for (int i = 0; i < VEC; ++i) u.e[i] = c + i < head_dim ? p[i] : Element<T>::from(0.f);
  return u.v;
}

template <class T>
__device__ __forceinline__ uint32_t magnitude(uint4 raw) {
  float x[Element<T>::kVec];
  Element<T>::unpack(raw, x);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < Element<T>::kVec; ++i) m = max(m, __float_as_uint(x[i]) & 0x7FFFFFFFu);
  return m;
}

__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  // a NaN scale gives code 0
  return (uint32_t)(__float2int_rn(a) & 0xFF) | (uint32_t)(__float2int_rn(b) & 0xFF) << 8 |
         (uint32_t)(__float2int_rn(c) & 0xFF) << 16 | (uint32_t)(__float2int_rn(d) & 0xFF) << 24;
}

template <class T>
__device__ __forceinline__ void store_codes(int8_t* at, uint4 raw, float inverse) {
  float x[Element<T>::kVec];
  Element<T>::unpack(raw, x);
#pragma unroll
  for (int i = 0; i < Element<T>::kVec; ++i) x[i] *= inverse;
  if constexpr (Element<T>::kVec == 4) {
    *reinterpret_cast<uint32_t*>(at) = pack_codes(x[0], x[1], x[2], x[3]);
  } else {
    *reinterpret_cast<uint2*>(at) = make_uint2(pack_codes(x[0], x[1], x[2], x[3]), pack_codes(x[4], x[5], x[6], x[7]));
  }
}

// A group of G threads (32: a warp, else the CTA) writes one page of one head,
// of K and of V.  A thread holds up to HELD 16-byte vectors of each between
// the reduction and the store; the two tensors' loads go out together, since a
// group begins with the chain length -> page -> rows.  16 x 2011 ragged tokens of
// 8 bfloat16 heads of 96, pages of 64: 29 us, 16 of them bytes; with 2048 tokens
// each the issue slots are 76% busy, mostly with magnitudes and codes.
template <class T, int G, int HELD>
__global__ void __launch_bounds__(G == 32 ? 128 : G, G == 256 && HELD == 4 ? 4 : 1)
    write_pages(View c, Batch t, Rows<T> k, Rows<T> v, int head_dim, int page_slots, unsigned units, int* status) {
  constexpr int VEC = Element<T>::kVec, GROUPS = G == 32 ? 4 : 1;
  const int id = threadIdx.x % G;
  const unsigned unit = blockIdx.x * GROUPS + threadIdx.x / G;
  if (unit >= units) return;
  const unsigned rest = unit / (unsigned)c.heads;
  const int head = (int)(unit - rest * c.heads);
  const int b = (int)(rest / (unsigned)page_slots), slot_page = (int)(rest - (unsigned)b * page_slots);
  const Span s = span_of(t, c, b);
  const bool report = status != nullptr && id == 0 && head == 0;
  if (report && slot_page == 0) {
    // pages past the announced number of new rows are not visited
    const bool missed = s.fresh && ((s.length - s.fresh) >> c.shift) + page_slots <= (s.length - 1) >> c.shift;
    const int flags = s.flags ? s.flags : missed ? kBadRows : 0;
    if (flags) atomicOr(status, flags);
  }
  if (s.flags || s.fresh == 0) return;  // nothing is written for a sequence whose numbers do not fit
  const int old = s.length - s.fresh;   // tokens before the new ones
  const int index = (old >> c.shift) + slot_page;
  if (index > (s.length - 1) >> c.shift) return;
  const int lo = index << c.shift;
  const int from = max(lo, old), to = lo + min(c.tokens, s.length - lo);
  const int page = page_of(t, c, b, index);
  if (page < 0) {
    if (report) atomicOr(status, kBadPage);
    return;
  }
  float* scale_at[2] = {c.k_scale + c.scale_at(page, head), c.v_scale + c.scale_at(page, head)};
  float before[2] = {0.f, 0.f};
  if (from > lo) {
    before[0] = *scale_at[0];
    before[1] = *scale_at[1];
  }
  const int per_row = c.width / VEC;  // width is a multiple of 32
  const int chunks = (to - from) * per_row;
  const size_t row0 = s.row + (from - old);
  uint4 raw[2][HELD];
  uint32_t most[2] = {0, 0};
  auto load = [&](int base) {
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int e = base + i * G + id;
      if (e < chunks) {
        const int r = e / per_row, ch = (e - r * per_row) * VEC;
        raw[0][i] = load_chunk(k, row0 + r, head, ch, head_dim);
        raw[1][i] = load_chunk(v, row0 + r, head, ch, head_dim);
      }
    }
  };
  for (int base = 0; base < chunks; base += G * HELD) {
    load(base);
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (base + i * G + id < chunks) {
        most[0] = max(most[0], magnitude<T>(raw[0][i]));
        most[1] = max(most[1], magnitude<T>(raw[1][i]));
      }
  }
  most[0] = __reduce_max_sync(0xFFFFFFFFu, most[0]);
  most[1] = __reduce_max_sync(0xFFFFFFFFu, most[1]);
  // The barriers also order all threads' reads of the scales before their store
  // below; a reduction alone orders no memory.
  if constexpr (G > 32) {
    __shared__ uint2 parts[G / 32];
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = make_uint2(most[0], most[1]);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < G / 32; ++w) {
      most[0] = max(most[0], parts[w].x);
      most[1] = max(most[1], parts[w].y);
    }
  } else {
    __syncwarp();
  }
  float inverse[2];
  const size_t page_at = c.row(page, head, 0);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float scale = scale_for(most[which]);
    if (from > lo) {
      // the page's earlier tokens: the scale never shrinks, NaN stays
      const float was = before[which];
      if (was != was || was > scale) scale = was;
      if (scale != was) {
        const float ratio = was / scale;
        uint32_t* w = reinterpret_cast<uint32_t*>((which ? c.v : c.k) + page_at);
        for (int e = id; e < (from - lo) * (c.width / 4); e += G) {
          const uint32_t q = w[e];
          w[e] = pack_codes(rintf((float)(int8_t)q * ratio), rintf((float)(int8_t)(q >> 8) * ratio),
                            rintf((float)(int8_t)(q >> 16) * ratio), rintf((float)(int8_t)(q >> 24) * ratio));
        }
      }
    }
    if (id == 0) *scale_at[which] = scale;
    inverse[which] = 1.0f / scale;
  }
  const size_t at = page_at + (size_t)(from - lo) * c.width;
  const bool held = chunks <= G * HELD;
  for (int base = 0; base < chunks; base += G * HELD) {
    if (!held) load(base);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const int e = base + i * G + id;
      if (e < chunks) {
        store_codes<T>(c.k + at + (size_t)e * VEC, raw[0][i], inverse[0]);
        store_codes<T>(c.v + at + (size_t)e * VEC, raw[1][i], inverse[1]);
      }
    }
  }
}

template <class T, int G, int HELD>
void launch_write(const View& c, const Batch& t, const Rows<T>& k, const Rows<T>& v, int head_dim, int page_slots,
                  unsigned units, int* status, cudaStream_t st) {
  constexpr unsigned GROUPS = G == 32 ? 4 : 1;
  write_pages<T, G, HELD><<<(units + GROUPS - 1) / GROUPS, G == 32 ? 128 : G, 0, st>>>(c, t, k, v, head_dim, page_slots,
                                                                                     units, status);
}

constexpr int kReadTokens = 8;  // tokens a thread has in flight

// out [batch][tokens][heads][head_dim]: blockIdx.x a run of tokens of one
// sequence, blockIdx.y a run of columns (head, chunk), blockIdx.z K or V.
// Bound by the writes: 8 x 4096 FP32 tokens of 8 heads of 64 27.7 us (87% of
// the copy rate), bfloat16 of 96, 16 x 2088 tokens, 28.7 (72%).
template <class T, int CHUNK>
__global__ void __launch_bounds__(kThreads)
    read_pages(View c, Batch t, const int32_t* __restrict__ first, int tokens, int head_dim, int columns,
               int columns_here, int runs, T* __restrict__ k_out, T* __restrict__ v_out, int* status) {
  const int b = blockIdx.x / runs, run = blockIdx.x % runs;
  const int lanes = kThreads / columns_here;  // tokens side by side
  const int column = blockIdx.y * columns_here + threadIdx.x % columns_here;
  const int lane = threadIdx.x / columns_here;
  if (lane >= lanes || column >= columns) return;
  const int chunks = head_dim / CHUNK;
  const int head = column / chunks, ch = (column - head * chunks) * CHUNK;
  const int8_t* codes = blockIdx.z ? c.v : c.k;
  const float* scales = blockIdx.z ? c.v_scale : c.k_scale;
  T* out = blockIdx.z ? v_out : k_out;
  const int n = t.lengths[b];
  const long long room = (long long)t.table_pages << c.shift;
  const int length = (int)(n < 0 ? 0 : n > room ? room : n);
  if (status && run == 0 && column == 0 && lane == 0 && blockIdx.z == 0 && length != n) atomicOr(status, kBadLength);
  const long long start = first ? first[b] : 0;
  uint2 q[kReadTokens];
  float scale[kReadTokens];
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u) {
    const int i = (run * kReadTokens + u) * lanes + lane;
    const long long pos = start + i;
    q[u] = make_uint2(0u, 0u);
    scale[u] = 0.f;
    if (i < tokens && pos >= 0 && pos < length) {
      const int page = page_of(t, c, b, (int)(pos >> c.shift));
      if (page >= 0) {
        const int8_t* at = codes + c.row(page, head, (int)pos & (c.tokens - 1)) + ch;
        if constexpr (CHUNK == 8) q[u] = __ldg(reinterpret_cast<const uint2*>(at));
        else if constexpr (CHUNK == 4) q[u].x = __ldg(reinterpret_cast<const uint32_t*>(at));
        else q[u].x = (uint8_t)*at;
        scale[u] = __ldg(scales + c.scale_at(page, head));
      } else {
        scale[u] = NAN;  // the tokens that should be there
        if (status) atomicOr(status, kBadPage);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kReadTokens; ++u) {
    const int i = (run * kReadTokens + u) * lanes + lane;
    if (i >= tokens) continue;
    T* o = out + (((size_t)b * tokens + i) * c.heads + head) * head_dim + ch;
    float x[8];
#pragma unroll
    for (int e = 0; e < CHUNK; ++e)
      x[e] = (float)(int8_t)((e < 4 ? q[u].x : q[u].y) >> (8 * (e & 3))) * scale[u];
    if constexpr (CHUNK == 1) *o = Element<T>::from(x[0]);
    else __stcs(reinterpret_cast<uint4*>(o), Element<T>::pack(x));  // not read again here
  }
}

template <class T>
Rows<T> make_rows(const void* p, size_t row_stride, size_t head_stride) {
  constexpr size_t VEC = Element<T>::kVec;
  aligned_to(p, sizeof(T), "rows must be aligned to their elements");
  return Rows<T>{static_cast<const T*>(p), row_stride, head_stride,
                 reinterpret_cast<uintptr_t>(p) % 16 == 0 && row_stride % VEC == 0 && head_stride % VEC == 0};
}

}  // namespace cache
}  // namespace mb

extern "C" {

int mb_op_cache_write(const mb_cache_write_args* a, void* stream) {
  using namespace mb::cache;
  return mb::guarded([&] {
    mb::need(a, "args");
    const View c = view_of(a->cache, a->head_dim);
    const Batch t = batch_of(a->where, a->max_new);
    const uint32_t max_new = a->max_new;
    if (t.rows == 0 || t.count == 0) return;
    mb::need(a->k, "k");
    mb::need(a->v, "v");
    const int page_slots = (int)(((size_t)max_new + c.tokens - 2) / c.tokens + 1);
    const size_t units = (size_t)t.count * page_slots * c.heads;
    mb::require(units <= (size_t)INT_MAX, "too many pages for one call");
    mb::with_dtype(a->dtype, [&](auto tag) {
      using T = typename decltype(tag)::type;
      const Rows<T> kr = make_rows<T>(a->k, a->k_row_stride, a->k_head_stride);
      const Rows<T> vr = make_rows<T>(a->v, a->v_row_stride, a->v_head_stride);
      // As few threads as hold a page's new rows in registers (16 x 2048 tokens of
      // 8 bfloat16 heads of 64, pages of 16: 27 us with a warp, 143 with 256
      // threads; of 96, pages of 64: 39 with 256, 51 with a warp that reads twice).
      // Eight vectors a lane pay where pages are many: a warp against 128 threads
      // 26 : 36 us with pages of 32, FP32 pages of 16 40 : 64, 6.2 : 8.4 for 2064
      // units; 5.3 : 4.7 for 1024.
      const size_t vectors = std::min<size_t>(max_new, c.tokens) * c.width / mb::Element<T>::kVec;
      const int hd = (int)a->head_dim;
      const unsigned n = (unsigned)units;
      const cudaStream_t st = (cudaStream_t)stream;
      if (vectors <= 32 * 4) launch_write<T, 32, 4>(c, t, kr, vr, hd, page_slots, n, a->d_status, st);
      else if (vectors <= 32 * 8 && units >= 12 * (size_t)mb::sm_count())
        launch_write<T, 32, 8>(c, t, kr, vr, hd, page_slots, n, a->d_status, st);
      else if (vectors <= 128 * 4) launch_write<T, 128, 4>(c, t, kr, vr, hd, page_slots, n, a->d_status, st);
      else if (vectors <= 256 * 4) launch_write<T, 256, 4>(c, t, kr, vr, hd, page_slots, n, a->d_status, st);
      else launch_write<T, 256, 8>(c, t, kr, vr, hd, page_slots, n, a->d_status, st);
      mb::launched("cache write");
    });
  });
}

int mb_op_cache_read(const mb_cache_read_args* a, void* stream) {
  using namespace mb::cache;
  return mb::guarded([&] {
    mb::need(a, "args");
    const uint32_t head_dim = a->head_dim, tokens = a->tokens;
    const View c = view_of(a->cache, head_dim);
    const Batch t = batch_of(a->where, 0);
    mb::require(tokens <= (1u << 30), "tokens must be at most 2^30");
    if (tokens == 0 || t.count == 0) return;
    void *k_out = a->k_out, *v_out = a->v_out;
    mb::need(k_out, "k_out");
    mb::need(v_out, "v_out");
    cudaStream_t st = (cudaStream_t)stream;
    mb::with_dtype(a->dtype, [&](auto tag) {
      using T = typename decltype(tag)::type;
      constexpr int VEC = mb::Element<T>::kVec;
      for (const void* p : {(const void*)k_out, (const void*)v_out})
        mb::aligned_to(p, sizeof(T), "outputs must be aligned to their elements");
      const bool vector = head_dim % VEC == 0 && reinterpret_cast<uintptr_t>(k_out) % 16 == 0 &&
                          reinterpret_cast<uintptr_t>(v_out) % 16 == 0;
      const int columns = c.heads * (int)(head_dim / (vector ? VEC : 1));
      const int here = std::min(columns, kThreads);
      const int per_block = kThreads / here * kReadTokens;
      const size_t runs = (tokens + (size_t)per_block - 1) / per_block;
      mb::require(runs * t.count <= (size_t)INT_MAX && (columns + here - 1) / here <= 65535,
                  "too many tokens for one call");
      const dim3 grid((unsigned)(runs * t.count), (unsigned)((columns + here - 1) / here), 2);
      if (vector)
        read_pages<T, VEC><<<grid, kThreads, 0, st>>>(c, t, a->first, (int)tokens, (int)head_dim, columns, here,
                                                      (int)runs, (T*)k_out, (T*)v_out, a->d_status);
      else
        read_pages<T, 1><<<grid, kThreads, 0, st>>>(c, t, a->first, (int)tokens, (int)head_dim, columns, here,
                                                    (int)runs, (T*)k_out, (T*)v_out, a->d_status);
      mb::launched("cache read");
    });
  });
}

}  // extern "C"
