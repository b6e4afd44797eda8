// Attention of new rows over the 8-bit paged cache.
//
// For row i of sequence b (n new rows, L tokens in the cache with them) and
// query head a of key head h = a / G, over the positions j that the row sees,
// first_b <= j <= L - n + i:
//
//   s_j = scale q . k_j,   p_j = e^(s_j - m),   o = sum_j p_j v_j / sum_j p_j
//
// A row that sees nothing gives 0, and -inf as its log-sum-exp.
//
// Codes are small integers, exact in FP16, so the products run on FP16
// tensor-core instructions with FP32 accumulation and the scales of K and V,
// powers of two, multiply scores and probabilities without rounding.  q and p
// enter as FP16 pairs hi + lo (22 bits) after an exact scaling by a power of
// two: q by its row's largest magnitude; p, times its V's scale, by the largest
// V scale that the row has seen so far, and 2^14 (2^11 in tiles).  So what a
// weight loses is 2^-22 of it, or 2^-39 (2^-36) of the largest |v| that the row
// sees, and nothing that it does not see moves that.
//
// The split kernel serves rows that share a key head and are few, one tile of
// 32 tokens after the other, bound by the bytes of the cache.  The tensor
// core's operand has 16 rows: 8 query rows' hi parts are its rows 0-7 and
// their lo parts its rows 8-15, so the second term costs nothing; of 16-bit
// rows, which need no second term (bfloat16's 8 bits fit into FP16, and a
// probability's rounding to 11 bits is below the output's own), up to 16 are
// served at once.  Every warp runs its own ring of bulk copies and its own
// running softmax (no barrier between warps until the end); the four warps'
// results, and the chunks that a long sequence is cut into, are joined by
// their maxima in a fixed order.

#include <algorithm>
#include <cmath>

#include "cache_host.h"
#include "common.cuh"
#include "dtype.cuh"
#include "tc05.cuh"

namespace mb {
namespace cache {

constexpr unsigned kFull = 0xFFFFFFFFu;
constexpr int kTile = 32;        // tokens a warp takes at a time
constexpr int kSplitWarps = 4;
constexpr int kSplitThreads = kSplitWarps * 32;

struct Queries {
  const void* q;
  size_t row_stride, head_stride;
  void* out;   // [rows][q_heads][head_dim]
  float* lse;  // [q_heads][rows] base 2, or null
  int heads, group, head_dim;
  float scale_log2;  // softmax scale times log2 e
  const int32_t* first;
  int* status;
};

// Partial results of the chunks: [unit][chunk][row] log-sum-exp and
// [unit][chunk][row][width] normalised outputs.
struct Partials {
  float* lse;
  float* o;
  int chunks;       // per unit
  int chunk_tiles;  // tiles of a chunk; the last one takes what is left
  float4* sums;     // [block][head][chunk][half][width / 4][row of the half], of wide FP32 rows in tiles
  bool packed;      // the blocks of the sums are packed_block's, else the units
};

// Numbers for the row blocks that hold rows, whatever the sequences' shares: the
// ceil(n G / 256) blocks of sequence b, which brings n rows from row r of the
// packed array on, begin at floor(r G / 256) + b and end before the next sequence's
// begin (floor(x + y) + 1 >= floor(x) + ceil(y)).  Units count a longest prompt
// for each sequence.
__host__ __device__ inline size_t packed_block(size_t first_row, int group, int block_rows, size_t b) {
  return first_row * group / block_rows + b;
}

template <int D, int ROWS>
struct SplitSmem {
  // Tiles a warp has in its ring, and CTAs of an SM that registers and shared
  // memory then allow: the warps that wait on latencies count more than a
  // deeper ring.  4 x 131071 tokens, 8 heads of 128, 4 query heads each: 192 us
  // (5.6 TB/s); about 290 with 3 stages, 2 CTAs and chunks of uneven waves, which
  // went together.
  static constexpr int kStages = D > 64 ? 2 : 3;
  static constexpr int kResident = D > 64 ? 3 : D > 32 ? 4 : 5;
  static constexpr int kTileBytes = kTile * D;
  static constexpr int kWarpBytes = kStages * 2 * kTileBytes;
  static constexpr int kBars = kSplitWarps * kWarpBytes;
  static constexpr int kMeta = kBars + kSplitWarps * kStages * 8;          // scales of each stage
  static constexpr int kJoin = kMeta + kSplitWarps * kStages * 16;         // m, l, exponent per warp and row
  static constexpr int kBytes = kJoin + kSplitWarps * ROWS * 12 + 16;
};

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two codes u = c + 128 (bytes of `biased` picked by `select`) as FP16: the
// byte under the exponent of 1024 is 1024 + u, and 1152 comes off exactly.
__device__ __forceinline__ uint32_t codes_to_f16(uint32_t biased, uint32_t select) {
  const uint32_t w = __byte_perm(biased, 0x64646464u, select);
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6480)));
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int WORDS>
__device__ __forceinline__ void load_words(const int8_t* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS % 4 == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
      w[i + 2] = v.z;
      w[i + 3] = v.w;
    }
  } else if constexpr (WORDS % 2 == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; i += 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
      w[i] = v.x;
      w[i + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
  }
}

__device__ __forceinline__ int exponent_of(float power) { return (int)(__float_as_uint(power) >> 23) - 127; }

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(kFull, v, 1));
  return fmaxf(v, __shfl_xor_sync(kFull, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(kFull, v, 1);
  return v + __shfl_xor_sync(kFull, v, 2);
}

// What a unit (sequence, 8 rows, key head) covers.
struct Unit {
  int b, row0, rows;     // rows of the group's row list: row r is token r / G, head r % G
  int length, fresh;
  size_t first_row;
  int lo;                // first visible position
  int hi;                // one past the last that any of its rows sees
  bool bad;
};

template <int ROWS>
__device__ __forceinline__ Unit unit_of(const View& c, const Batch& t, const Queries& q, int z, int blocks_per_seq) {
  Unit u;
  u.b = z / blocks_per_seq;
  u.row0 = (z % blocks_per_seq) * ROWS;
  const Span s = span_of(t, c, u.b);
  u.length = s.length;
  u.fresh = s.fresh;
  u.first_row = s.row;
  u.rows = (int)min((long long)ROWS, (long long)s.fresh * q.group - u.row0);
  u.bad = s.flags != 0;
  const int old = s.length - s.fresh;
  u.lo = q.first ? max(0, q.first[u.b]) : 0;
  u.hi = u.rows > 0 ? old + (u.row0 + u.rows - 1) / q.group + 1 : 0;
  return u;
}

// Rows past the announced number are not visited: the last block of a
// sequence gives them NaN; a sequence whose numbers do not fit, all its rows.
template <class T>
__device__ __forceinline__ void refuse_rows(const Batch& t, const Queries& q, int head, const Unit& u, int from_row,
                                            int threads) {
  const size_t count = (size_t)u.fresh * q.group;
  for (size_t r = from_row; r < count; ++r) {
    const size_t row = u.first_row + r / q.group;
    const int a = head * q.group + (int)(r % q.group);
    T* out = static_cast<T*>(q.out) + (row * q.heads + a) * q.head_dim;
    for (int ch = threadIdx.x; ch < q.head_dim; ch += threads) out[ch] = Element<T>::from(NAN);
    if (threadIdx.x == 0 && q.lse) q.lse[(size_t)a * t.rows + row] = NAN;
  }
}

// Rows in front of the first sequence's and behind the last one's, as of a batch
// padded to a fixed size, see nothing: 0 and -inf (NaN where that sequence's
// numbers do not fit).  The CTAs of those two sequences share them, this one the
// `part`-th of `parts`.
template <class T>
__device__ __forceinline__ void unowned_rows(const Batch& t, const Queries& q, int head, const Unit& u, unsigned part,
                                             unsigned parts, int threads) {
  const bool first = u.b == 0 && u.first_row > 0, last = u.b == t.count - 1 && u.first_row + u.fresh < t.rows;
  if (!first && !last) return;
  const size_t end = u.first_row + u.fresh, before = first ? u.first_row : 0;
  const size_t count = (before + (last ? t.rows - end : 0)) * q.group;
#pragma unroll 1
  for (size_t r = part; r < count; r += parts) {
    const size_t at = r / q.group, row = at < before ? at : end + at - before;
    const int a = head * q.group + (int)(r % q.group);
    T* out = static_cast<T*>(q.out) + (row * q.heads + a) * q.head_dim;
    for (int ch = threadIdx.x; ch < q.head_dim; ch += threads) out[ch] = Element<T>::from(u.bad ? NAN : 0.f);
    if (threadIdx.x == 0 && q.lse) q.lse[(size_t)a * t.rows + row] = u.bad ? NAN : -INFINITY;
  }
}

template <class T, int D, int ROWS>
__global__ void __launch_bounds__(kSplitThreads, SplitSmem<D, ROWS>::kResident)
    attend_split(View c, Batch t, Queries q, Partials part, int blocks_per_seq) {
  using S = SplitSmem<D, ROWS>;
  // 8 rows in two terms, or 16 in one: a lane has rows g (and g + 8), NB of them
  static_assert(ROWS == 8 || (ROWS == 16 && sizeof(T) == 2), "rows");
  constexpr int NB = ROWS / 8;
  constexpr int STAGES = S::kStages;
  constexpr int KW = D / 16;  // words of a K row that a thread reads: one K step of 16 channels each
  constexpr int VW = D / 32;  // words of a V row
  extern __shared__ __align__(128) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, tq = lane & 3;
  const int chunk = blockIdx.x % part.chunks, head = blockIdx.y, z = blockIdx.x / part.chunks;
  const Unit u = unit_of<ROWS>(c, t, q, z, blocks_per_seq);
  const bool last_block = z % blocks_per_seq == blocks_per_seq - 1;

  unowned_rows<T>(t, q, head, u, z % blocks_per_seq * part.chunks + chunk, blocks_per_seq * part.chunks, kSplitThreads);
  if (u.bad) {
    if (chunk == 0 && z % blocks_per_seq == 0) {
      refuse_rows<T>(t, q, head, u, 0, kSplitThreads);
      if (q.status && threadIdx.x == 0) atomicOr(q.status, span_of(t, c, u.b).flags);
    }
  } else if (last_block && chunk == 0 && (long long)u.fresh * q.group > u.row0 + ROWS) {
    refuse_rows<T>(t, q, head, u, u.row0 + ROWS, kSplitThreads);
    if (q.status && threadIdx.x == 0) atomicOr(q.status, kBadRows);
  }
  if (u.bad || u.rows <= 0) return;

  const int tile_lo = u.lo / kTile, tile_hi = u.hi > u.lo ? (u.hi + kTile - 1) / kTile : tile_lo;
  const int begin = (int)min((long long)tile_hi, tile_lo + (long long)chunk * part.chunk_tiles);
  const int end = chunk == part.chunks - 1 ? tile_hi : min(tile_hi, begin + part.chunk_tiles);
  const size_t slot = ((size_t)z * c.heads + head) * part.chunks + chunk;
  if (begin >= end && part.chunks > 1) {
    if (threadIdx.x < ROWS) part.lse[slot * ROWS + threadIdx.x] = -INFINITY;
    return;
  }

  int8_t* ring = reinterpret_cast<int8_t*>(smem) + warp * S::kWarpBytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars) + warp * STAGES;
  float4* meta = reinterpret_cast<float4*>(smem + S::kMeta) + warp * STAGES;
  float* join = reinterpret_cast<float*>(smem + S::kJoin);
  int* gave_up = reinterpret_cast<int*>(smem + S::kJoin + kSplitWarps * ROWS * 12);
  if (lane == 0)
    for (int s = 0; s < STAGES; ++s) tc::bar_init(&bars[s], 1);
  tc::bar_init_fence();
  if (threadIdx.x == 0) *gave_up = 0;
  __syncthreads();

  const int mine = end > begin + warp ? (end - begin - warp + kSplitWarps - 1) / kSplitWarps : 0;  // this warp's tiles
  const bool two = c.tokens == kTile / 2;  // a tile spans two pages

  // page numbers and scales of 32 tiles, one a lane
  int page0 = -1, page1 = -1;
  float ks0 = 0.f, ks1 = 0.f, vs0 = 0.f, vs1 = 0.f;
  auto look_up = [&](int n) {
    page0 = page1 = -1;
    ks0 = ks1 = vs0 = vs1 = 0.f;
    if (n + lane >= mine) return;
    const int pos = (begin + warp + (n + lane) * kSplitWarps) * kTile;
    // scales of pages that no row sees stay 0: theirs may be anything
    bool bad = false;
    if (!two || pos + kTile / 2 > u.lo) {
      page0 = page_of(t, c, u.b, pos >> c.shift);
      bad = page0 < 0;
      ks0 = bad ? NAN : __ldg(c.k_scale + c.scale_at(page0, head));
      vs0 = bad ? NAN : __ldg(c.v_scale + c.scale_at(page0, head));
    }
    if (!two) {
      ks1 = ks0;
      vs1 = vs0;
    } else if (pos + kTile / 2 < u.hi) {
      page1 = page_of(t, c, u.b, (pos >> c.shift) + 1);
      ks1 = page1 < 0 ? NAN : __ldg(c.k_scale + c.scale_at(page1, head));
      vs1 = page1 < 0 ? NAN : __ldg(c.v_scale + c.scale_at(page1, head));
      bad = bad || page1 < 0;
    }
    if (bad && q.status) atomicOr(q.status, kBadPage);
  };
  auto issue = [&](int n) {
    const int s = n % STAGES, from = n & 31;
    const int p0 = __shfl_sync(kFull, page0, from), p1 = __shfl_sync(kFull, page1, from);
    if (lane == 0) {
      int8_t* k_at = ring + s * 2 * S::kTileBytes;
      int8_t* v_at = k_at + S::kTileBytes;
      const int inside = ((begin + warp + n * kSplitWarps) * kTile) & (c.tokens - 1);
      const uint32_t bytes = two ? S::kTileBytes / 2 : S::kTileBytes;
      tc::bar_expect_tx(&bars[s], 2 * bytes * ((p0 >= 0) + (p1 >= 0)));
      if (p0 >= 0) {
        tc::bulk_g2s(k_at, c.k + c.row(p0, head, inside), bytes, &bars[s]);
        tc::bulk_g2s(v_at, c.v + c.row(p0, head, inside), bytes, &bars[s]);
      }
      if (p1 >= 0) {
        tc::bulk_g2s(k_at + bytes, c.k + c.row(p1, head, 0), bytes, &bars[s]);
        tc::bulk_g2s(v_at + bytes, c.v + c.row(p1, head, 0), bytes, &bars[s]);
      }
    }
    // behind the copies: the scales' loads may still be on their way
    const float4 m = make_float4(__shfl_sync(kFull, ks0, from), __shfl_sync(kFull, ks1, from),
                                 __shfl_sync(kFull, vs0, from), __shfl_sync(kFull, vs1, from));
    if (lane == 0) meta[s] = m;
  };

  look_up(0);
  int issued = 0;
  for (; issued < STAGES - 1 && issued < mine; ++issued) issue(issued);

  // This lane's query rows: hi parts as operand rows g; as rows g + 8 their
  // lo parts, or row g + 8.
  uint32_t qf[KW][4];
  float row_factor[NB];
  int limit[NB];  // last position the row sees
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = u.row0 + 8 * nb + g;
    const bool there = 8 * nb + g < u.rows;
    const int tok = r / q.group, a = head * q.group + r % q.group;
    limit[nb] = there ? u.length - u.fresh + tok : -1;
    const T* src = static_cast<const T*>(q.q) + (u.first_row + tok) * q.row_stride + (size_t)a * q.head_stride;
    float x[KW][4];
    float most = 0.f;
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int ch = tq * (D / 4) + 4 * w + e;
        x[w][e] = there && ch < q.head_dim ? Element<T>::to(src[ch]) : 0.f;
        most = fmaxf(most, fabsf(x[w][e]));
      }
    const float up = tc::f16_scale(quad_max(most));
#pragma unroll
    for (int w = 0; w < KW; ++w)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        uint32_t lo;
        tc::split_f16x2(x[w][2 * e] * up, x[w][2 * e + 1] * up, qf[w][2 * e + nb], lo);
        if (NB == 1) qf[w][2 * e + 1] = lo;
      }
    row_factor[nb] = q.scale_log2 / up;
  }
  const int sure = u.length - u.fresh + u.row0 / q.group;  // the last position that every row sees

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
  float m[NB], l[NB];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    m[nb] = -INFINITY;
    l[nb] = 0.f;
  }
  int ev[NB];  // o carries 2^(14 - ev)
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) ev[nb] = -126;

  // The first tiles' scales, which lane 0 wrote behind the copies' arrivals, are
  // there for every lane; those of later tiles by the end of each turn.
  __syncwarp();
  for (int n = 0; n < mine; ++n) {
    if (issued < mine) {
      if ((issued & 31) == 0) look_up(issued);
      issue(issued++);
    }
    const int s = n % STAGES;
    if (!__all_sync(kFull, tc::bar_wait(&bars[s], (n / STAGES) & 1))) {
      *gave_up = 1;
      // it and the copies behind it may still land: none is left when the CTA ends
      for (int k = n; k < issued; ++k) tc::bar_wait(&bars[k % STAGES], (k / STAGES) & 1);
      break;
    }
    const float4 sc = meta[s];
    const int8_t* kt = ring + s * 2 * S::kTileBytes;
    const int8_t* vt = kt + S::kTileBytes;
    const int pos = (begin + warp + n * kSplitWarps) * kTile;

    float x[4][2 * NB];  // [8 tokens][row, token 2 tq + e]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t w[KW];
      load_words<KW>(kt + (8 * j + g) * D + tq * (D / 4), w);
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        const uint32_t biased = w[k] ^ 0x80808080u;
        mma16816(acc, qf[k][0], qf[k][1], qf[k][2], qf[k][3], codes_to_f16(biased, 0x4140),
                 codes_to_f16(biased, 0x4342));
      }
      const float scale = j < 2 ? sc.x : sc.y;
      if constexpr (NB == 1) {
        x[j][0] = (acc[0] + acc[2]) * (scale * row_factor[0]);
        x[j][1] = (acc[1] + acc[3]) * (scale * row_factor[0]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j][e] = acc[e] * (scale * row_factor[e / 2]);
      }
    }
    // V's scales for this lane's rows: 0 where a row sees nothing of the 16
    // tokens, whose scale may be NaN or far from the seen ones
    float seen0[NB], seen1[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      seen0[nb] = sc.z;
      seen1[nb] = sc.w;
    }
    if (pos < u.lo || pos + kTile - 1 > sure) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2 * NB; ++e) {
          const int at = pos + 8 * j + 2 * tq + (e & 1);
          if (at < u.lo || at > limit[e / 2]) x[j][e] = -INFINITY;
        }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        if (pos + kTile / 2 <= u.lo || max(pos, u.lo) > limit[nb]) seen0[nb] = 0.f;
        if (pos + kTile <= u.lo || max(pos + kTile / 2, u.lo) > limit[nb]) seen1[nb] = 0.f;
      }
    }
    float base[NB], change[NB];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      // V's exponent: o is kept relative to the largest V scale that the row has seen
      int top = ev[nb];
      if (seen0[nb] == seen0[nb]) top = max(top, exponent_of(seen0[nb]));
      if (seen1[nb] == seen1[nb]) top = max(top, exponent_of(seen1[nb]));
      const float lower = top != ev[nb] ? power_of_two(max(ev[nb] - top, -126)) : 1.f;
      ev[nb] = top;
      float mx = fmaxf(x[0][2 * nb], x[0][2 * nb + 1]);
#pragma unroll
      for (int j = 1; j < 4; ++j) mx = fmaxf(mx, fmaxf(x[j][2 * nb], x[j][2 * nb + 1]));
      mx = fmaxf(m[nb], quad_max(mx));
      base[nb] = mx == -INFINITY ? 0.f : mx;
      const float shrink = ex2_ftz(m[nb] - base[nb]);
      m[nb] = mx;
      l[nb] *= shrink;
      change[nb] = shrink * lower;
    }
    if (__any_sync(kFull, change[0] != 1.0f || change[NB - 1] != 1.0f)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] *= change[NB == 1 ? 0 : e / 2];
    }
    uint32_t pf[4][2];  // [8 tokens][operand rows g, g + 8]
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const float f = (j < 2 ? seen0[nb] : seen1[nb]) * power_of_two(-ev[nb]) * 16384.f;
        const float p0 = ex2_ftz(x[j][2 * nb] - base[nb]), p1 = ex2_ftz(x[j][2 * nb + 1] - base[nb]);
        l[nb] += p0 + p1;
        if constexpr (NB == 1) {
          tc::split_f16x2(p0 * f, p1 * f, pf[j][0], pf[j][1]);
        } else {
          const __half2 h = __floats2half2_rn(p0 * f, p1 * f);
          pf[j][nb] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t v0[VW], v1[VW], v2[VW], v3[VW];
      const int8_t* vr = vt + (16 * k + 2 * tq) * D + g * (D / 8);
      load_words<VW>(vr, v0);
      load_words<VW>(vr + D, v1);
      load_words<VW>(vr + 8 * D, v2);
      load_words<VW>(vr + 9 * D, v3);
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        const uint32_t a = v0[w] ^ 0x80808080u, b = v1[w] ^ 0x80808080u;
        const uint32_t d = v2[w] ^ 0x80808080u, e = v3[w] ^ 0x80808080u;
        // bytes of the two rows side by side: channels 0, 1 and 2, 3
        const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
        const uint32_t de0 = __byte_perm(d, e, 0x5140), de1 = __byte_perm(d, e, 0x7362);
        mma16816(o[4 * w + 0], pf[2 * k][0], pf[2 * k][1], pf[2 * k + 1][0], pf[2 * k + 1][1], codes_to_f16(ab0, 0x4140),
                 codes_to_f16(de0, 0x4140));
        mma16816(o[4 * w + 1], pf[2 * k][0], pf[2 * k][1], pf[2 * k + 1][0], pf[2 * k + 1][1], codes_to_f16(ab0, 0x4342),
                 codes_to_f16(de0, 0x4342));
        mma16816(o[4 * w + 2], pf[2 * k][0], pf[2 * k][1], pf[2 * k + 1][0], pf[2 * k + 1][1], codes_to_f16(ab1, 0x4140),
                 codes_to_f16(de1, 0x4140));
        mma16816(o[4 * w + 3], pf[2 * k][0], pf[2 * k][1], pf[2 * k + 1][0], pf[2 * k + 1][1], codes_to_f16(ab1, 0x4342),
                 codes_to_f16(de1, 0x4342));
      }
    }
    __syncwarp();  // the stage is read: its next copy may be issued
  }

  // The four warps' results side by side; every copy issued has landed.
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const float sum = quad_sum(l[nb]);
    if (tq == 0) {
      float* w = join + (warp * ROWS + 8 * nb + g) * 3;
      w[0] = m[nb];
      w[1] = sum;
      w[2] = power_of_two(ev[nb]);
    }
  }
  __syncwarp();
  float* mine_o = reinterpret_cast<float*>(ring);  // [ROWS][D]
#pragma unroll
  for (int i = 0; i < D / 8; ++i) {
    // n-tile i, column n is channel n D/8 + i
    float* at = mine_o + g * D + 2 * tq * (D / 8) + i;
    if constexpr (NB == 1) {
      at[0] = o[i][0] + o[i][2];
      at[D / 8] = o[i][1] + o[i][3];
    } else {
      at[0] = o[i][0];
      at[D / 8] = o[i][1];
      at[8 * D] = o[i][2];
      at[8 * D + D / 8] = o[i][3];
    }
  }
  __syncthreads();
  const bool failed = *gave_up != 0;
  if (failed && threadIdx.x == 0 && q.status) atomicOr(q.status, kGaveUp);
  for (int e = threadIdx.x; e < u.rows * D; e += kSplitThreads) {
    const int r = e / D, ch = e % D;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, join[(w * ROWS + r) * 3]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, value = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const float* jw = join + (w * ROWS + r) * 3;
      const float f = ex2_ftz(jw[0] - base);
      const float ow = reinterpret_cast<const float*>(smem + w * S::kWarpBytes)[e];
      sum = fmaf(jw[1], f, sum);
      value = fmaf(ow * (1.0f / 16384.f) * jw[2], f, value);
    }
    float lse = sum == 0.f ? -INFINITY : base + log2f(sum);
    value = sum == 0.f ? 0.f : value / sum;
    if (failed) lse = value = NAN;
    if (part.chunks > 1) {
      part.o[(slot * ROWS + r) * D + ch] = value;
      if (ch == 0) part.lse[slot * ROWS + r] = lse;
    } else {
      const int row = u.row0 + r;
      const size_t at = u.first_row + row / q.group;
      const int a = head * q.group + row % q.group;
      if (ch < q.head_dim) static_cast<T*>(q.out)[(at * q.heads + a) * q.head_dim + ch] = Element<T>::from(value);
      if (ch == 0 && q.lse) q.lse[(size_t)a * t.rows + at] = lse;
    }
  }
}

// ---------------------------------------------------------------- tiles
// The tile kernel serves rows that are many (prompts): 256 query rows of a key
// head against tiles of 64 tokens, on the tcgen05 tensor cores.
//
//   warps 0-3, 4-7  one query row a thread, rows 0-127 and 128-255: softmax of
//                   S from tensor memory, P back over it as FP16, O rescaled
//                   where a maximum has grown
//   warps 8-11      converters: the tile's codes from global memory (loaded a
//                   tile ahead), as FP16 into shared memory, once for both halves
//   warps 12, 13    issue the products S = Q K^T and O += P V of a half each
//
// Each half has two score buffers (P goes over S in place), so that the next
// scores are there when a softmax ends and only softmax follows softmax in a
// half's chain.  K and V share one layout, rows = tokens: K-major for S,
// MN-major for O.  Queries and probabilities of FP32 rows are FP16 pairs
// (two products), those of 16-bit rows one FP16 (bfloat16's 8 bits fit; a
// probability's rounding to 11 bits is below the output's own).
//
// The tensor core cuts its accumulator's sums instead of rounding them, and the
// loss grows with the number of products added to O (1024 tokens of FP32 rows:
// 1.1e-6 of the result, 4096: 3.4e-6; rounded sums 0.7e-6 and 1.1e-6).  Of FP32
// rows O is therefore added to a sum, rounded, every 6 tiles and begun again:
// in shared memory where Q has gone to tensor memory, else in the workspace, by
// additions that nothing waits for, each address its own thread's.  (Every 4,
// 6 and 8 tiles: 0.81, 0.91 and 0.97e-6; 180, 177 and 173 us for 32 x 1024
// tokens of 8 heads of 64, 165 without.)
//
// O follows a row's maximum lazily: probabilities up to 2^4 are let through,
// so that after the first tiles O is hardly ever touched; they carry 2^11,
// 2^15 in all, inside FP16's range.
constexpr int kKeys = 64;
constexpr int kHalfRows = 128;
constexpr int kTileRows = 2 * kHalfRows;
constexpr int kTileThreads = 14 * 32;
constexpr int kConverters = 128;
constexpr int kStages = 3;
constexpr float kLazy = 4.f;
constexpr float kProbScale = 2048.f;
constexpr int kSumTiles = 6;     // FP32 rows: tiles whose products O holds at most
constexpr int kSumWidth = 64;    // widest rows with sums in shared memory

template <int D, int TERMS>
struct TileShape {
  // Two score buffers a half and O leave room for Q in tensor memory up to
  // head width 64; wider heads read it from shared memory.
  static constexpr bool kQInSmem = D > 64;
  static constexpr int kQ = kQInSmem ? 0 : TERMS * D / 2;  // columns of a half's Q
  static constexpr int kS = 2 * kQ;                        // [half][buffer]
  static constexpr int kO = kS + 4 * kKeys;
  static_assert(kO + 2 * D <= 512, "tensor memory");
  static constexpr int kOperand = kKeys * D * 2;           // bytes of a K or V tile
  static constexpr int kQTile = kHalfRows * D * 2;         // bytes of a half's Q, a term
  // Q's FP16 tiles [half][term], also on their way into tensor memory; at the
  // end the outputs' rows, which are as large
  static constexpr int kQueries = kStages * 2 * kOperand;
  static constexpr int kScales = kQueries + 2 * TERMS * kQTile;  // of Q's rows
  static constexpr int kMeta = kScales + kTileRows * 4;
  static constexpr int kSpoilt = kMeta + kStages * 32;
  static constexpr int kBars = kSpoilt + 32;
  static constexpr int kBytes = kBars + 192;
};

// D (tensor memory) (+)= A (tensor memory, or shared memory) * B (shared memory), FP16.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add));
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add));
}

__device__ __forceinline__ void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Sixteen columns of this thread's lane, asynchronously: the registers may be
// read after tmem_wait, which takes them so that no use moves before it.
__device__ __forceinline__ void tmem_ld16_async(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]),
                 "+r"(v[8]), "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
               :
               : "memory");
}

// *at += {a, b, c, d}, without waiting for it.
__device__ __forceinline__ void add_f32x4(float4* at, float a, float b, float c, float d) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// The largest of three (NaN only of three NaN).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// FP16 hi and lo parts of a pair.
__device__ __forceinline__ void pair_f16x2(float2 w, uint32_t& hi, uint32_t& lo) {
  const __half2 a = __floats2half2_rn(w.x, w.y);
  const float2 r = fma2(__half22float2(a), splat2(-1.0f), w);
  const __half2 b = __floats2half2_rn(r.x, r.y);
  hi = *reinterpret_cast<const uint32_t*>(&a);
  lo = *reinterpret_cast<const uint32_t*>(&b);
}

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

template <class T, int D>
__global__ void __launch_bounds__(kTileThreads, 1)
    attend_tiles(View c, Batch t, Queries q, Partials part, int blocks_per_seq) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  using S = TileShape<D, TERMS>;
  constexpr bool SUMS = TERMS == 2, FAR = SUMS && D > kSumWidth;  // sums of O; in the workspace
  extern __shared__ __align__(128) uint8_t smem[];
  // the shuffle makes the warp's number, and what follows from it, uniform
  const int warp = __shfl_sync(kFull, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int chunk = blockIdx.x % part.chunks, head = blockIdx.y;
  // the last rows see the most: they go first
  const int block = blockIdx.x / part.chunks;
  const int z = block / blocks_per_seq * blocks_per_seq + (blocks_per_seq - 1 - block % blocks_per_seq);
  const Unit u = unit_of<kTileRows>(c, t, q, z, blocks_per_seq);
  unowned_rows<T>(t, q, head, u, z % blocks_per_seq * part.chunks + chunk, blocks_per_seq * part.chunks, kTileThreads);
  if (u.bad) {
    if (chunk == 0 && z % blocks_per_seq == 0) {
      refuse_rows<T>(t, q, head, u, 0, kTileThreads);
      if (q.status && threadIdx.x == 0) atomicOr(q.status, span_of(t, c, u.b).flags);
    }
    return;
  }
  if (z % blocks_per_seq == blocks_per_seq - 1 && chunk == 0 && (long long)u.fresh * q.group > u.row0 + kTileRows) {
    refuse_rows<T>(t, q, head, u, u.row0 + kTileRows, kTileThreads);
    if (q.status && threadIdx.x == 0) atomicOr(q.status, kBadRows);
  }
  if (u.rows <= 0) return;

  const int old = u.length - u.fresh;
  // tiles of both halves, counted from the tile that holds the first visible position
  const int tile_lo = u.lo / kKeys;
  auto tiles_to = [&](int last_row) {
    const int hi = old + (u.row0 + last_row) / q.group + 1;
    return hi > u.lo ? (hi + kKeys - 1) / kKeys : tile_lo;
  };
  const bool both = u.rows > kHalfRows;
  const int end1 = tiles_to(u.rows - 1), end0 = both ? tiles_to(kHalfRows - 1) : end1;
  const int begin = (int)min((long long)end1, tile_lo + (long long)chunk * part.chunk_tiles);
  const int end = chunk == part.chunks - 1 ? end1 : min(end1, begin + part.chunk_tiles);
  // half h takes tiles begin .. begin + count[h]; the first half never more than the second
  const int count1 = end - begin, count0 = max(0, min(end0, end) - begin);
  const size_t slot = ((size_t)z * c.heads + head) * part.chunks + chunk;
  if (begin >= end && part.chunks > 1) {  // a chunk behind the block's last row
    for (int r = threadIdx.x; r < kTileRows; r += kTileThreads) part.lse[slot * kTileRows + r] = -INFINITY;
    return;
  }

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* kv_full = bars;               // [stage] converters -> products and softmax
  uint64_t* kv_free = bars + kStages;     // [stage] products -> converters
  uint64_t* s_full = bars + 2 * kStages;  // [half][buffer] scores -> softmax
  uint64_t* p_full = s_full + 4;          // [half][buffer] softmax -> products: a half may be two tiles ahead
  uint64_t* q_full = p_full + 4;          // [half]
  uint64_t* o_full = q_full + 2;          // [half][tile & 1] O += P V is done
  uint64_t* drained = o_full + 4;         // [half]
  uint32_t* tmem_at = reinterpret_cast<uint32_t*>(drained + 2);
  int* failed = reinterpret_cast<int*>(tmem_at + 1);
  float* meta = reinterpret_cast<float*>(smem + S::kMeta);  // [stage][4 K scales, 4 V scales] of 16 tokens each
  // meta holds numbers in the place of scales that are NaN, whose product with a
  // masked token's weight of 0 would reach every row.  A row sees positions from
  // the first visible one to its own, so it is spoilt if the first such token that
  // is visible at all is no later than that: [tokens 16 g of the tiles][K, V].
  // (Selecting scales by row where the weights are made takes 32 x 1024 FP32 tokens
  // of 8 heads of 64 from 143.7 to 149 us, this to 144.9.)
  int* spoilt = reinterpret_cast<int*>(smem + S::kSpoilt);
  if (threadIdx.x < 8) spoilt[threadIdx.x] = INT_MAX;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::bar_init(&kv_full[s], kConverters);
      tc::bar_init(&kv_free[s], both ? 2 : 1);
    }
    for (int h = 0; h < 2; ++h) {
      for (int k = 0; k < 2; ++k) {
        tc::bar_init(&o_full[2 * h + k], 1);
        tc::bar_init(&s_full[2 * h + k], 1);
        tc::bar_init(&p_full[2 * h + k], kHalfRows);
      }
      tc::bar_init(&q_full[h], kHalfRows);
      tc::bar_init(&drained[h], 1);
    }
    *failed = 0;
  }
  tc::bar_init_fence();
  if (warp == 12) tc::tmem_alloc(tmem_at, 512);
  // Barriers and tensor memory are there.  Every role passes this once, after
  // what it can do without them.
  auto ready = [&]() -> uint32_t {
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    return __shfl_sync(kFull, *tmem_at, 0);
  };
  // Rows of Q and of the output move between global and shared memory with
  // eight lanes on eight rows and four on a row's 16-byte chunks: whole sectors
  // there, all banks here.  A thread that read or wrote its own row would touch
  // 32 lines an instruction (12000 cycles for Q, 10000 for the output, of 65000
  // a CTA took for 1024 tokens of 64 channels).
  const int sub = lane & 7, quarter = lane >> 3;
  // Row r of the unit is token token0 + n / group of the sequence's new rows and
  // query head n % group of the key head, n = rest0 + r below 2048: exact in FP32.
  const int token0 = u.row0 / q.group, rest0 = u.row0 - token0 * q.group;
  const float per_group = 1.0f / (float)q.group;
  auto token_at = [&](int r) { return token0 + (int)(((float)(rest0 + r) + 0.5f) * per_group); };
  auto row_at = [&](int r) { return u.first_row + token_at(r); };
  auto head_at = [&](int r) { return head * q.group + rest0 + r - (token_at(r) - token0) * q.group; };

  if (warp < 8) {
    const int h = warp >> 2;
    const int count = h ? (both ? count1 : 0) : (both ? count0 : count1);
    const int r = h * kHalfRows + (warp & 3) * 32 + lane;  // row of the unit
    const bool there = r < u.rows;
    const int tok = token_at(r);
    const int limit = there ? old + tok : -1;
    // the last position that every row of the warp sees
    const int sure = old + token_at(r - lane);
    float factor = 0.f;
    float m = -INFINITY, l = 0.f;
    int ev = -126;
    bool alive = true;
    uint8_t* tile = smem + S::kQueries + h * TERMS * S::kQTile;
    float* scales = reinterpret_cast<float*>(smem + S::kScales);
    if (count > 0) {
      // 16-byte loads where every row is aligned for them
      const bool vector = ((reinterpret_cast<uintptr_t>(q.q) | q.row_stride * sizeof(T) | q.head_stride * sizeof(T)) & 15) == 0 &&
                          q.head_dim % Element<T>::kVec == 0;
      constexpr int AT_ONCE = D <= 64 ? 4 : 2;  // groups of eight rows whose loads go out together
#pragma unroll 1
      for (int rg = 0; rg < 4; rg += AT_ONCE) {
        float x[AT_ONCE][D / 32][8];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
          const int r8 = r - lane + 8 * (rg + k) + sub;
          const T* src = static_cast<const T*>(q.q) + row_at(r8) * q.row_stride + (size_t)head_at(r8) * q.head_stride;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            const int ch = (quarter + 4 * i) * 8;
            if (vector) {
#pragma unroll
              for (int e = 0; e < 8; e += Element<T>::kVec)
                Element<T>::unpack(r8 < u.rows && ch + e < q.head_dim ? __ldg(reinterpret_cast<const uint4*>(src + ch + e))
                                                                     : make_uint4(0u, 0u, 0u, 0u), x[k][i] + e);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) x[k][i][e] = r8 < u.rows && ch + e < q.head_dim ? Element<T>::to(src[ch + e]) : 0.f;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
          const int r8 = r - lane + 8 * (rg + k) + sub;
          float most = 0.f;
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[k][i][e]));
          most = fmaxf(most, __shfl_xor_sync(kFull, most, 8));
          most = fmaxf(most, __shfl_xor_sync(kFull, most, 16));
          const float up = tc::f16_scale(most);
          if (quarter == 0) scales[r8] = up;
          // scores are q.k times a factor that is not negative
          const float sign = q.scale_log2 < 0.f ? -up : up;
#pragma unroll
          for (int i = 0; i < D / 32; ++i) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) tc::split_f16x2(x[k][i][2 * e] * sign, x[k][i][2 * e + 1] * sign, hi[e], lo[e]);
            uint8_t* at = tile + tc::blk16(r8 & (kHalfRows - 1), (quarter + 4 * i) * 8, D) * 2;
            *reinterpret_cast<uint4*>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (TERMS == 2) *reinterpret_cast<uint4*>(at + S::kQTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          }
        }
      }
      __syncwarp();
      factor = fabsf(q.scale_log2) / scales[r];
    }
    const uint32_t tmem = ready();
    const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t at_q = lanes + h * S::kQ, at_o = lanes + S::kO + h * D;
    if (count > 0) {
      if constexpr (!S::kQInSmem) {
#pragma unroll
        for (int term = 0; term < TERMS; ++term)
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t w[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4 v = *reinterpret_cast<const uint4*>(
                  tile + term * S::kQTile + tc::blk16(r & (kHalfRows - 1), c0 + 8 * i, D) * 2);
              w[4 * i] = v.x;
              w[4 * i + 1] = v.y;
              w[4 * i + 2] = v.z;
              w[4 * i + 3] = v.w;
            }
            tc::tmem_st16u(at_q + term * (D / 2) + c0 / 2, w);
          }
      }
      tc::tmem_st_wait();
      tc::fence_async_smem();
      tc::fence_before_sync();
      tc::bar_arrive(&q_full[h]);
    }
    // 16-byte chunk k of a row of outputs, or of its sums, where Q was (it has
    // gone to tensor memory, or its products are done)
    auto staged = [&](int r8, int k) {
      return reinterpret_cast<uint4*>(tile + k / (D / 8) * S::kQTile +
                                      tc::blk16(r8 & (kHalfRows - 1), k % (D / 8) * 8, D) * 2);
    };
    // the same of the sums
    const size_t sum_slot =
        part.packed ? ((packed_block(u.first_row, q.group, kTileRows, u.b) + z % blocks_per_seq) * c.heads + head) *
                              part.chunks + chunk
                    : slot;
    auto sum_at = [&](int k) {
      return FAR ? part.sums + ((sum_slot * 2 + h) * (D / 4) + k) * kHalfRows + (r & (kHalfRows - 1))
                 : reinterpret_cast<float4*>(staged(r, k));
    };
    auto sum_read = [&](int k) { return FAR ? __ldcg(sum_at(k)) : *sum_at(k); };
    // The products of tile j.  A waiter may be a tile behind them or ahead, so
    // each parity of tiles has a barrier: a wait is exact within one phase only.
    auto o_done = [&](int j) { return tc::bar_wait(&o_full[2 * h + (j & 1)], (j >> 1) & 1); };
    for (int j = 0; j < count; ++j) {
      const int stage = j % kStages;
      // both: the tile's scales (converters) and its scores (products)
      alive = __all_sync(kFull, tc::bar_wait(&kv_full[stage], (j / kStages) & 1) &&
                                    tc::bar_wait(&s_full[2 * h + (j & 1)], (j >> 1) & 1));
      if (!alive) break;
      const uint32_t at_s = lanes + S::kS + (2 * h + (j & 1)) * kKeys;
      tc::fence_after_sync();
      const float4 ks = *reinterpret_cast<const float4*>(meta + stage * 8);
      const float4 vs = *reinterpret_cast<const float4*>(meta + stage * 8 + 4);
      // not 0, so that a masked score stays -inf
      auto positive = [](float f) { return fmaxf(f, 2e-38f); };
      const float fk[4] = {positive(ks.x * factor), positive(ks.y * factor), positive(ks.z * factor),
                           positive(ks.w * factor)};
      float sv[4] = {vs.x, vs.y, vs.z, vs.w};
      const int pos = (begin + j) * kKeys;
      if (pos < u.lo || pos + kKeys - 1 > sure) {
        // masked scores become -inf in place; few tiles need it, so the code below does not carry it
#pragma unroll 1
        for (int c0 = 0; c0 < kKeys; c0 += 16) {
          float x[16];
          tc::tmem_ld16(at_s + c0, x);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (pos + c0 + i < u.lo || pos + c0 + i > limit) x[i] = -INFINITY;
          tc::tmem_st16(at_s + c0, x);
        }
        tc::tmem_st_wait();
        // scales of 16 tokens that the row sees nothing of do not move its O's
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (pos + 16 * g + 16 <= u.lo || pos + 16 * g > limit) sv[g] = 0.f;
      }
      // The scores are read twice, for their maximum and for their
      // exponentials: 64 at once spill.
      // Sixteen columns at a time, the next ones on their way under the
      // current ones' arithmetic: a load's latency is as long as that.
      uint32_t column[2][16];
      float mx = m;
      tmem_ld16_async(at_s, column[0]);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        tmem_wait(column[g & 1]);
        if (g < 3) tmem_ld16_async(at_s + 16 * (g + 1), column[(g + 1) & 1]);
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(column[g & 1][i]);
        const float a0 = max3(max3(y[0], y[1], y[2]), y[3], y[4]), a1 = max3(max3(y[5], y[6], y[7]), y[8], y[9]);
        const float a2 = max3(max3(y[10], y[11], y[12]), y[13], max3(a0, a1, y[14]));
        mx = fmaxf(mx, fmaxf(a2, y[15]) * fk[g]);
      }
      int top = ev;
#pragma unroll
      for (int g = 0; g < 4; ++g) top = max(top, exponent_of(sv[g]));
      const bool close = SUMS && j > 0 && j % kSumTiles == 0;  // O joins the sums
      if (__any_sync(kFull, close || mx > m + kLazy || top != ev)) {
        const float shrink = ex2_ftz(m - (mx == -INFINITY ? 0.f : mx));
        l *= shrink;
        const float change = shrink * (top != ev ? power_of_two(max(ev - top, -126)) : 1.f);
        m = mx;
        ev = top;
        if (j > 0) {
          // the products before this tile's are in O
          alive = __all_sync(kFull, o_done(j - 1));
          if (!alive) break;
          tc::fence_after_sync();
          const bool summed = SUMS && j > kSumTiles;  // there are sums already
#pragma unroll 1
          for (int c0 = 0; c0 < D; c0 += 16) {
            float o[16];
            tc::tmem_ld16(at_o + c0, o);
            if (SUMS && (close || summed)) {
              const bool add = FAR && close && summed && !__any_sync(kFull, change != 1.f);
#pragma unroll
              for (int i = 0; i < 16; i += 4) {
                if (add) {
                  add_f32x4(sum_at((c0 + i) / 4), o[i], o[i + 1], o[i + 2], o[i + 3]);
                  continue;
                }
                float4 v = summed ? sum_read((c0 + i) / 4) : make_float4(0.f, 0.f, 0.f, 0.f);
                if (close) v = make_float4(v.x + o[i], v.y + o[i + 1], v.z + o[i + 2], v.w + o[i + 3]);
                *sum_at((c0 + i) / 4) = make_float4(v.x * change, v.y * change, v.z * change, v.w * change);
              }
            }
            if (!close) {  // else this tile's products begin O again
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] *= change;
              tc::tmem_st16(at_o + c0, o);
            }
          }
        }
      }
      const float base = m == -INFINITY ? 0.f : m;
      const float2 nbase = splat2(-base);
      const float unit = power_of_two(-ev);
      float2 sum = make_float2(0.f, 0.f);
      const float* page_scales = meta + stage * 8;
      tmem_ld16_async(at_s, column[0]);
      tmem_wait(column[0]);
      tmem_ld16_async(at_s + 16, column[1]);
#pragma unroll
      for (int g = 0; g < 4; ++g) {  // 16 tokens, at most one page
        const float2 f = splat2(positive(page_scales[g] * factor));
        // finite also where the row does not see the tokens: their weights stay 0
        const float2 v = splat2(fminf(page_scales[4 + g] * unit * kProbScale, 1e38f));
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 x = make_float2(__uint_as_float(column[g & 1][2 * i]), __uint_as_float(column[g & 1][2 * i + 1]));
          const float2 y = fma2(x, f, nbase);
          const float2 p = make_float2(ex2_ftz(y.x), ex2_ftz(y.y));
          sum = add2(sum, p);
          const float2 w = mul2(p, v);
          if constexpr (TERMS == 2) {
            pair_f16x2(w, hi[i], lo[i]);
          } else {
            const __half2 h2 = __floats2half2_rn(w.x, w.y);
            hi[i] = *reinterpret_cast<const uint32_t*>(&h2);
          }
        }
        // the next columns before the store, so that their arithmetic does not
        // wait for the end of these
        if (g < 3) tmem_wait(column[(g + 1) & 1]);
        if (g < 2) tmem_ld16_async(at_s + 16 * (g + 2), column[g & 1]);
        // P over its own scores' columns: hi in the first 8, lo behind
        tmem_st8(at_s + 16 * g, hi);
        if constexpr (TERMS == 2) tmem_st8(at_s + 16 * g + 8, lo);
      }
      l += sum.x + sum.y;
      tc::tmem_st_wait();
      tc::fence_before_sync();
      tc::bar_arrive(&p_full[2 * h + (j & 1)]);
    }
    if (count > 0 && alive) alive = __all_sync(kFull, o_done(count - 1));
    if (!alive) *failed = 1;
    tc::fence_after_sync();
    // (what a converter may still write here is behind this half's last position)
    int bad_k = INT_MAX, bad_v = INT_MAX;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      bad_k = min(bad_k, spoilt[2 * g]);
      bad_v = min(bad_v, spoilt[2 * g + 1]);
    }
    if (bad_k <= limit) l = NAN;
    const float inverse = bad_v <= limit ? NAN : l == 0.f ? 0.f : power_of_two(ev) * (1.f / kProbScale) / l;
    float lse = l == 0.f ? -INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
    if (!alive) lse = NAN;
    const size_t row = u.first_row + tok;
    const int a = head_at(r);
    T* out = static_cast<T*>(q.out) + (row * q.heads + a) * q.head_dim;
    float* po = part.o + (slot * kTileRows + r) * D;
    const bool wide = q.head_dim % Element<T>::kVec == 0 && (reinterpret_cast<uintptr_t>(q.out) & 15) == 0;
    if (there) {
      if (part.chunks > 1) part.lse[slot * kTileRows + r] = lse;
      else if (q.lse) q.lse[(size_t)a * t.rows + row] = lse;
    }
    constexpr int VEC = Element<T>::kVec;
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += 16) {
      float o[16];
      if (count > 0) tc::tmem_ld16(at_o + c0, o);
      if (SUMS && count > kSumTiles) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          const float4 v = sum_read((c0 + i) / 4);
          o[i] += v.x;
          o[i + 1] += v.y;
          o[i + 2] += v.z;
          o[i + 3] += v.w;
        }
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = !alive ? NAN : l == 0.f ? 0.f : o[i] * inverse;
      if (sizeof(T) == 2 && part.chunks > 1) {
        if (there) {
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(po + c0 + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      } else if (wide || part.chunks > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += VEC) *staged(r, (c0 + i) / VEC) = Element<T>::pack(o + i);
      } else if (there) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c0 + i < q.head_dim) out[c0 + i] = Element<T>::from(o[i]);
      }
      __syncwarp();  // tensor memory is read by whole warps
    }
    const bool partial = sizeof(T) == 4 && part.chunks > 1;  // FP32 rows are staged as they are
    if (partial || (part.chunks == 1 && wide)) {
      const int width = partial ? D : q.head_dim;
#pragma unroll
      for (int rg = 0; rg < 4; ++rg) {
        const int r8 = r - lane + 8 * rg + sub;
        T* to = partial ? reinterpret_cast<T*>(part.o + (slot * kTileRows + r8) * D)
                        : static_cast<T*>(q.out) + (row_at(r8) * q.heads + head_at(r8)) * q.head_dim;
#pragma unroll
        for (int i = 0; i < D / VEC / 4; ++i) {
          const int k = quarter + 4 * i;
          if (r8 < u.rows && k * VEC < width) *reinterpret_cast<uint4*>(to + k * VEC) = *staged(r8, k);
        }
      }
    }
  } else if (warp < 12) {
    // 16 codes a piece; 8 lanes take one piece column of 8 rows, whose FP16
    // chunks are 128 contiguous bytes each
    constexpr int PIECES = D / 32;  // of K and of V, a thread and tile
    const int ct = threadIdx.x - 8 * 32;
    uint4 kq[PIECES], vq[PIECES];
    int pages[PIECES], scale_page = -1;
    float sk = 1.f, sv = 0.f;
    auto row_of = [&](int i) { return (ct + kConverters * i) / (8 * (D / 16)) * 8 + (ct & 7); };
    auto channel_of = [&](int i) { return ((ct + kConverters * i) >> 3) % (D / 16) * 16; };
    // The page of a token: -1 out of the pool, -2 where no row sees the page;
    // that is not looked up, its tokens are masked, as zeros.
    auto look_up = [&](int pos) {
      const int first_of_page = pos & ~(c.tokens - 1);
      return first_of_page < u.hi && first_of_page + c.tokens > u.lo ? page_of(t, c, u.b, pos >> c.shift) : -2;
    };
    // Page numbers are read two tiles ahead and codes one, so that neither is waited for.
    auto find = [&](int j) {
      const int pos = (begin + j) * kKeys;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) pages[i] = i > 0 && c.tokens >= kKeys ? pages[0] : look_up(pos + row_of(i));
      if (ct < 4) scale_page = look_up(pos + 16 * ct);
    };
    const size_t page_bytes = (size_t)c.heads * c.tokens * c.width;
    const int8_t* k_head = c.k + (size_t)head * c.tokens * c.width;
    const int8_t* v_head = c.v + (size_t)head * c.tokens * c.width;
    auto load = [&](int j) {
      const int pos = (begin + j) * kKeys;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        kq[i] = vq[i] = make_uint4(0u, 0u, 0u, 0u);
        if (pages[i] >= 0) {
          const size_t from = pages[i] * page_bytes + ((pos + row_of(i)) & (c.tokens - 1)) * c.width + channel_of(i);
          kq[i] = __ldg(reinterpret_cast<const uint4*>(k_head + from));
          vq[i] = __ldg(reinterpret_cast<const uint4*>(v_head + from));
        }
      }
      if (ct < 4) {
        sk = 1.f;
        sv = 0.f;
        if (scale_page >= 0) {
          sk = __ldg(c.k_scale + c.scale_at(scale_page, head));
          sv = __ldg(c.v_scale + c.scale_at(scale_page, head));
        } else if (scale_page == -1) {
          sk = sv = NAN;
          if (q.status) atomicOr(q.status, kBadPage);
        }
      }
    };
    auto store = [&](uint8_t* tile, const uint4 (&codes)[PIECES]) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        const uint32_t w[4] = {codes[i].x ^ 0x80808080u, codes[i].y ^ 0x80808080u, codes[i].z ^ 0x80808080u,
                               codes[i].w ^ 0x80808080u};
        __half* to = reinterpret_cast<__half*>(tile) + tc::blk16(row_of(i), channel_of(i), D);
        *reinterpret_cast<uint4*>(to) = make_uint4(codes_to_f16(w[0], 0x4140), codes_to_f16(w[0], 0x4342),
                                                   codes_to_f16(w[1], 0x4140), codes_to_f16(w[1], 0x4342));
        *reinterpret_cast<uint4*>(to + 64) = make_uint4(codes_to_f16(w[2], 0x4140), codes_to_f16(w[2], 0x4342),
                                                        codes_to_f16(w[3], 0x4140), codes_to_f16(w[3], 0x4342));
      }
    };
    if (count1 > 0) {
      find(0);
      load(0);
      if (count1 > 1) find(1);
    }
    ready();
    for (int j = 0; j < count1; ++j) {
      const int stage = j % kStages;
      if (j >= kStages && !tc::bar_wait(&kv_free[stage], (j / kStages - 1) & 1)) {
        *failed = 1;
        break;
      }
      uint8_t* tile = smem + stage * 2 * S::kOperand;
      store(tile, kq);
      store(tile + S::kOperand, vq);
      if (ct < 4) {
        meta[stage * 8 + ct] = sk == sk ? sk : 1.f;
        meta[stage * 8 + 4 + ct] = sv == sv ? sv : 0.f;
        const int group = (begin + j) * kKeys + 16 * ct, at = max(group, u.lo);
        if (group + 16 > u.lo) {
          if (sk != sk) spoilt[2 * ct] = min(spoilt[2 * ct], at);
          if (sv != sv) spoilt[2 * ct + 1] = min(spoilt[2 * ct + 1], at);
        }
      }
      tc::fence_async_smem();
      tc::bar_arrive(&kv_full[stage]);
      if (j + 1 < count1) load(j + 1);
      if (j + 2 < count1) find(j + 2);
    }
  } else {
    // The issuer of a half.  The whole warp waits, one lane issues: everything
    // it works with is uniform, which keeps the instructions between two
    // products few (from a single diverged lane a product took about 100
    // cycles to issue).
    const int h = warp - 12;
    const uint32_t tmem = ready();
    const bool elected = elect_one();
    const int count = h ? (both ? count1 : 0) : (both ? count0 : count1);
    constexpr uint32_t kIdS = tc::idesc_f16(128, kKeys), kIdO = tc::idesc_f16(128, D, true);
    const uint64_t k0 = tc::desc_kmajor16(smem, D, 0), v0 = tc::desc_mn16(smem + S::kOperand, D, 0);
    const uint64_t q0 = tc::desc_kmajor16(smem + S::kQueries + h * TERMS * S::kQTile, D, 0);
    constexpr uint64_t kStep = 256 >> 4, vStep = D / 8 * 256 >> 4, kStage = 2 * S::kOperand >> 4;
    const uint32_t at_q = tmem + h * S::kQ, at_s = tmem + S::kS + 2 * h * kKeys, at_o = tmem + S::kO + h * D;
    auto scores = [&](int j) {
      const uint64_t k = k0 + (j % kStages) * kStage;
      const uint32_t to = at_s + (j & 1) * kKeys;
#pragma unroll
      for (int term = 0; term < TERMS; ++term) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          const bool add = term > 0 || s > 0;
          if constexpr (S::kQInSmem) mma_ss(to, q0 + term * (S::kQTile >> 4) + s * kStep, k + s * kStep, kIdS, add);
          else mma_ts(to, at_q + term * (D / 2) + 8 * s, k + s * kStep, kIdS, add);
        }
      }
    };
    auto values = [&](int j) {
      const uint64_t v = v0 + (j % kStages) * kStage;
#pragma unroll
      for (int s = 0; s < kKeys / 16; ++s) {
        const uint32_t p = at_s + (j & 1) * kKeys + 16 * s;  // 16 tokens
        mma_ts(at_o, p, v + s * vStep, kIdO, (SUMS ? j % kSumTiles : j) > 0 || s > 0);
        if constexpr (TERMS == 2) mma_ts(at_o, p + 8, v + s * vStep, kIdO, true);
      }
    };
    auto full = [&](int j) { return tc::bar_wait(&kv_full[j % kStages], (j / kStages) & 1); };
    bool ok = true;
    if (count > 0) ok = __all_sync(kFull, tc::bar_wait(&q_full[h], 0));
    // the first two tiles' scores
    for (int j = 0; j < 2 && j < count && ok; ++j) {
      ok = __all_sync(kFull, full(j));
      tc::fence_after_sync();
      if (ok && elected) {
        scores(j);
        tc::commit(&s_full[2 * h + j]);
      }
      __syncwarp();
    }
    for (int j = 0; j < count && ok; ++j) {
      ok = __all_sync(kFull, tc::bar_wait(&p_full[2 * h + (j & 1)], (j >> 1) & 1));
      tc::fence_after_sync();
      if (ok && elected) {
        values(j);
        tc::commit(&o_full[2 * h + (j & 1)]);
        tc::commit(&kv_free[j % kStages]);
      }
      __syncwarp();
      if (j + 2 >= count || !ok) continue;
      // Scores of tile j + 2 go over the probabilities of tile j: not before
      // the products that read them are done (only products of one
      // accumulator and shape are ordered among themselves).
      ok = __all_sync(kFull, full(j + 2) && tc::bar_wait(&o_full[2 * h + (j & 1)], (j >> 1) & 1));
      tc::fence_after_sync();
      if (ok && elected) {
        scores(j + 2);
        tc::commit(&s_full[2 * h + (j & 1)]);
      }
      __syncwarp();
    }
    // the tiles that only the other half sees: released once they are full, so
    // that no phase counts this half twice
    for (int j = count; both && j < count1 && ok; ++j) {
      ok = __all_sync(kFull, full(j));
      if (ok && elected) tc::bar_arrive(&kv_free[j % kStages]);
    }
    if (!ok) *failed = 1;
    // nothing is in flight when tensor memory is given back
    if (elected) tc::commit(&drained[h]);
    if (!tc::bar_wait(&drained[h], 0)) *failed = 1;
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 12) {
    tc::fence_after_sync();
    tc::tmem_dealloc(*tmem_at, 512);
  }
  if (threadIdx.x == 0 && *failed && q.status) atomicOr(q.status, kGaveUp);
}

// Joins the chunks of a unit's rows.  WARPS warps share a row's chunks: 8 for
// the few rows of the split kernel, whose chunks may be hundreds, 1 for tiles.
// A launch and one pass over a few KB, bound by latency: 4 x 2000 FP32 tokens of
// 4 heads of 64 take 8.4 us with it, 1 x 256 without it 6.1.
template <class T, int D, int ROWS, int WARPS>
__global__ void __launch_bounds__(256)
    join_chunks(View c, Batch t, Queries q, Partials part, int blocks_per_seq) {
  constexpr int C = D / 32;
  __shared__ float sums[8], values[8][D];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int head = blockIdx.y, z = blockIdx.x;
  const int r = WARPS == 1 ? blockIdx.z * 8 + warp : blockIdx.z;
  const Unit u = unit_of<ROWS>(c, t, q, z, blocks_per_seq);
  if (u.bad || r >= u.rows) return;
  const size_t slot = ((size_t)z * c.heads + head) * part.chunks;
  const float* lse = part.lse + slot * ROWS + r;
  float top = -INFINITY;
  for (int i = lane; i < part.chunks; i += 32) top = fmaxf(top, lse[(size_t)i * ROWS]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, value[C];
#pragma unroll
  for (int k = 0; k < C; ++k) value[k] = 0.f;
  constexpr int AHEAD = 4;
  for (int i = WARPS == 1 ? 0 : warp; i < part.chunks; i += WARPS * AHEAD) {
    float f[AHEAD], x[AHEAD][C];
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const int at = i + e * WARPS;
      const float s = at < part.chunks ? lse[(size_t)at * ROWS] : -INFINITY;
      f[e] = s == -INFINITY ? 0.f : ex2_ftz(s - base);  // saw nothing: its outputs were not written
      const float* po = part.o + ((slot + at) * ROWS + r) * D;
#pragma unroll
      for (int k = 0; k < C; ++k) x[e][k] = s == -INFINITY ? 0.f : po[lane + 32 * k];
    }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      sum += f[e];
#pragma unroll
      for (int k = 0; k < C; ++k) value[k] = fmaf(f[e], x[e][k], value[k]);
    }
  }
  if (WARPS > 1) {
    if (lane == 0) sums[warp] = sum;
#pragma unroll
    for (int k = 0; k < C; ++k) values[warp][lane + 32 * k] = value[k];
    __syncthreads();
    if (warp > 0) return;
    for (int w = 1; w < WARPS; ++w) {
      sum += sums[w];
#pragma unroll
      for (int k = 0; k < C; ++k) value[k] += values[w][lane + 32 * k];
    }
  }
  const int row = u.row0 + r;
  const size_t at = u.first_row + row / q.group;
  const int a = head * q.group + row % q.group;
  T* out = static_cast<T*>(q.out) + (at * q.heads + a) * q.head_dim;
#pragma unroll
  for (int k = 0; k < C; ++k)
    if (lane + 32 * k < q.head_dim) out[lane + 32 * k] = Element<T>::from(sum == 0.f ? 0.f : value[k] / sum);
  if (lane == 0 && q.lse) q.lse[(size_t)a * t.rows + at] = sum == 0.f ? -INFINITY : base + log2f(sum);
}

// ---------------------------------------------------------------- host side
struct Plan {
  int unit_rows;       // kTileRows: the tile kernel, else the split kernel with 8 or 16
  int blocks_per_seq;  // row blocks of a sequence
  size_t units;        // sequences times row blocks
  int chunks, chunk_tiles;
  size_t packed;       // row blocks that all rows can fill
  size_t sums;         // bytes of the sums of O, first in the workspace
  size_t workspace;    // bytes
};

// More rows a sequence and key head on average go to the tile kernel: 8 x 8192
// tokens, 8 bfloat16 heads of 128, split against tiles 44 : 99 us with 8 rows,
// 83 : 104 with 32, 140 : 105 with 64; 64 x 1024 tokens, 8 FP32 heads of 64,
// 25 : 93, 72 : 95 with 8 and 32.
constexpr size_t kSplitMost = 32;

inline Plan make_plan(size_t batch, size_t rows, uint32_t kv_heads, uint32_t group, uint32_t width, uint32_t max_new,
                      uint32_t max_tokens, uint32_t dtype) {
  Plan p;
  const size_t most_rows = (size_t)max_new * group;
  require(most_rows <= (1u << 30), "too many new rows for one call");
  const bool use_tiles = rows * group > kSplitMost * batch;
  p.unit_rows = use_tiles ? kTileRows : dtype != MB_F32 && most_rows > 8 ? 16 : 8;
  const size_t unit_rows = p.unit_rows, keys = use_tiles ? kKeys : kTile;
  p.blocks_per_seq = (int)((most_rows + unit_rows - 1) / unit_rows);
  p.units = batch * p.blocks_per_seq;
  // Chunks for the CTAs that the GPU holds at a time, none shorter than eight
  // tiles (two a warp of the split kernel).  Long sequences are cut further, as
  // long as a chunk keeps 128 tiles: unequal lengths and ends even out.
  const int resident = use_tiles ? 1 : width > 64 ? 3 : width > 32 ? 4 : 5;
  const size_t slots = (size_t)sm_count() * resident, have = std::max<size_t>(1, p.units * kv_heads);
  const size_t tiles = std::max<size_t>(1, ((size_t)max_tokens + keys - 1) / keys);
  size_t chunks = std::max<size_t>(1, std::min((tiles + 7) / 8, slots / have));
  for (int waves = 2; waves <= 4; ++waves)
    if (tiles * have >= slots * waves * 128) chunks = std::max(chunks, slots * waves / have);
  p.chunk_tiles = (int)((tiles + chunks - 1) / chunks + kSplitWarps - 1) / kSplitWarps * kSplitWarps;
  p.chunks = (int)((tiles + p.chunk_tiles - 1) / p.chunk_tiles);
  const size_t rows_in = p.units * kv_heads * p.chunks * unit_rows;
  p.packed = packed_block(rows, (int)group, kTileRows, batch);
  p.sums = 0;
  if (use_tiles && dtype == MB_F32 && width > (uint32_t)kSumWidth)
    p.sums = std::min(p.units, p.packed) * kv_heads * p.chunks * kTileRows * width * sizeof(float);
  p.workspace = p.sums + (p.chunks > 1 ? rows_in * (width + 1) * sizeof(float) : 0);
  return p;
}

template <class T, int D, int ROWS>
void launch_rows(const View& c, const Batch& t, const Queries& q, const Plan& p, void* workspace, cudaStream_t st) {
  constexpr bool TILES = ROWS == kTileRows;
  const size_t slots = p.units * c.heads * p.chunks;
  // vectors first: they need the workspace's alignment
  float* o = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.sums);
  const Partials part{o + slots * ROWS * D, o, p.chunks, p.chunk_tiles, static_cast<float4*>(workspace),
                      p.packed < p.units};
  constexpr int bytes = TILES ? TileShape<D, sizeof(T) == 4 ? 2 : 1>::kBytes : SplitSmem<D, TILES ? 8 : ROWS>::kBytes;
  void (*kernel)(View, Batch, Queries, Partials, int);
  if constexpr (TILES) kernel = attend_tiles<T, D>;
  else kernel = attend_split<T, D, ROWS>;
  static DeviceOnce once;  // one a kernel
  once([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
  kernel<<<dim3((unsigned)(p.units * p.chunks), (unsigned)c.heads), TILES ? kTileThreads : kSplitThreads, bytes, st>>>(
      c, t, q, part, p.blocks_per_seq);
  launched("cache attention");
  if (p.chunks == 1) return;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)p.units, (unsigned)c.heads, TILES ? ROWS / 8 : ROWS);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  launched("cache attention join",
           cudaLaunchKernelEx(&cfg, join_chunks<T, D, ROWS, TILES ? 1 : 8>, c, t, q, part, p.blocks_per_seq));
}

template <class T, int D>
void launch(const View& c, const Batch& t, const Queries& q, const Plan& p, void* workspace, cudaStream_t st) {
  if (p.unit_rows == kTileRows) return launch_rows<T, D, kTileRows>(c, t, q, p, workspace, st);
  if constexpr (sizeof(T) == 2)
    if (p.unit_rows == 16) return launch_rows<T, D, 16>(c, t, q, p, workspace, st);
  launch_rows<T, D, 8>(c, t, q, p, workspace, st);
}

}  // namespace cache
}  // namespace mb

extern "C" {

int mb_op_cache_attention_workspace(uint32_t batch, size_t rows, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim,
                                    uint32_t dtype, uint32_t max_new, uint32_t max_tokens, size_t* bytes) {
  using namespace mb::cache;
  return mb::guarded([&] {
    mb::need(bytes, "bytes");
    mb::require(kv_heads >= 1 && q_heads >= 1 && q_heads % kv_heads == 0, "kv_heads must divide q_heads");
    const uint32_t width = (head_dim + 31) / 32 * 32;
    *bytes = batch == 0 ? 0 : make_plan(batch, rows, kv_heads, q_heads / kv_heads, width, max_new, max_tokens, dtype).workspace;
  });
}

int mb_op_cache_attention(const mb_cache_attention_args* a, void* stream) {
  using namespace mb::cache;
  return mb::guarded([&] {
    mb::need(a, "args");
    const View c = view_of(a->cache, a->head_dim);
    const uint32_t q_heads = a->q_heads, max_new = a->max_new, max_tokens = a->max_tokens;
    const Batch t = batch_of(a->where, max_new);
    mb::require(q_heads >= 1 && q_heads % c.heads == 0 && q_heads / c.heads <= 1024,
                "the cache's heads must divide q_heads");
    mb::require(std::isfinite(a->scale), "scale must be finite");
    mb::require(max_tokens <= (uint32_t)INT_MAX, "max_tokens must be below 2^31");
    if (t.rows == 0) return;
    mb::require(t.count > 0, "rows without a sequence");
    mb::require(max_new >= 1, "max_new must be positive where there are rows");
    const void* q = a->q;
    void *out = a->out, *workspace = a->workspace;
    const size_t workspace_bytes = a->workspace_bytes;
    mb::need(q, "q");
    mb::need(out, "out");
    const Queries qs{q, a->q_row_stride, a->q_head_stride, out, a->lse, (int)q_heads, (int)(q_heads / c.heads),
                     (int)a->head_dim, a->scale * mb::kLog2e, a->first, a->d_status};
    const Plan p = make_plan(t.count, t.rows, c.heads, qs.group, c.width, max_new, max_tokens, a->dtype);
    mb::require(p.units * p.chunks <= (size_t)INT_MAX, "too many row blocks for one call");
    mb::require(p.workspace == 0 || (workspace != nullptr && workspace_bytes >= p.workspace &&
                                     reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "workspace missing, too small or not 16-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    mb::with_dtype(a->dtype, [&](auto tag) {
      using T = typename decltype(tag)::type;
      for (const void* x : {q, (const void*)out})
        mb::aligned_to(x, sizeof(T), "q and out must be aligned to their elements");
      switch (c.width) {
        case 32: return launch<T, 32>(c, t, qs, p, workspace, st);
        case 64: return launch<T, 64>(c, t, qs, p, workspace, st);
        case 96: return launch<T, 96>(c, t, qs, p, workspace, st);
        default: return launch<T, 128>(c, t, qs, p, workspace, st);
      }
    });
  });
}

}  // extern "C"
