// lookup.cu -- rows of a table by index, times a scale, and the table's gradient.
//
//   out[t, :] = scale * table[index[t], :]
//   grad_table[v, :] = scale * sum of grad_out[t, :] over the t with index[t] = v
//
// The gradient's sums run in fp32 in an order that the inputs alone decide (no
// floating atomics): the tokens are sorted by row (stable, so equal rows keep
// their order), cut into windows of equal length whatever the rows' counts, and
// each thread adds up one column vector of one window.  Rows that lie in one
// window are written at once; rows that cross windows leave partial sums, which a
// second kernel joins.  Rows that no token names are zeros.  Few rows or few tokens
// need no sort: each row looks for its own.
//
// Memory traffic bounds it: every token's gradient row is read once, the table's
// gradient is written once (and the rows that are used once more).  Up to 90112
// tokens are sorted by one cluster through distributed shared memory while the
// rest of the GPU writes the zeros.  131072 x 4096 bf16, 16384 tokens: lookup 31 us,
// zeros 142 us (7.5 TB/s, the sort's 19 behind them), sums 45 us, joins 11 us.
#include <cooperative_groups.h>

#include "common.cuh"
#include "primitives.h"  // bits_for
#include "training.h"
#include "vec.cuh"

namespace sinkslot {

namespace cg = cooperative_groups;

constexpr int kLookThreads = 256;

__device__ __forceinline__ int64_t index_at(const void* index, int bytes, int64_t t) {
  return bytes == 8 ? static_cast<const int64_t*>(index)[t]
                    : (int64_t) static_cast<const int32_t*>(index)[t];
}

// 16 bytes from any element's address, out of the two aligned vectors around it.
// [begin, end): what may be read; elements outside come as zeros (callers ask for
// vectors that reach over a row's ends, and drop what is not the row's).
template <typename T>
__device__ __forceinline__ uint4 load16(const T* p, const T* begin, const T* end) {
  constexpr int N = Vec16<T>::N;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint32_t phase = (uint32_t)(a & 15);
  const T* v = reinterpret_cast<const T*>(a - phase);
  if (v >= begin && v + 2 * N <= end) {
    const uint4 lo = __ldg(reinterpret_cast<const uint4*>(v));
    if (phase == 0) return lo;
    const uint4 hi = __ldg(reinterpret_cast<const uint4*>(v) + 1);
    // shifted by two words, by one, then by the bytes within a word (selects: the
    // phase is another for every row)
    const bool two = phase & 8, one = phase & 4;
    const uint32_t x0 = two ? lo.z : lo.x, x1 = two ? lo.w : lo.y, x2 = two ? hi.x : lo.z,
                   x3 = two ? hi.y : lo.w, x4 = two ? hi.z : hi.x, x5 = two ? hi.w : hi.y;
    const uint32_t y0 = one ? x1 : x0, y1 = one ? x2 : x1, y2 = one ? x3 : x2,
                   y3 = one ? x4 : x3, y4 = one ? x5 : x4;
    if (sizeof(T) == 4) return make_uint4(y0, y1, y2, y3);
    const uint32_t r = (phase & 3) * 8;
    return make_uint4(__funnelshift_r(y0, y1, r), __funnelshift_r(y1, y2, r),
                      __funnelshift_r(y2, y3, r), __funnelshift_r(y3, y4, r));
  }
  T t[N];
#pragma unroll
  for (int j = 0; j < N; ++j) t[j] = p + j >= begin && p + j < end ? p[j] : from_f32<T>(0.0f);
  uint4 u;
  memcpy(&u, t, 16);
  return u;
}

// --------------------------------------------------------------------------
// Lookup: the output is one array of 16-byte vectors whatever the width of its
// rows, so a vector may hold the end of one row and the beginning of the next.
// Four vectors for each thread: the index, then the rows' data, are waited for
// once for all four.
// --------------------------------------------------------------------------
constexpr int kLookVecs = 4;

// kAligned: all rows begin on 16-byte boundaries.  I: 32 bits where the output's
// elements fit (a division of 64 bits costs more than the copy).  A thread's vectors
// lie `skip` rows and `over` columns apart.
template <typename T, typename I, bool kAligned>
__global__ void __launch_bounds__(kLookThreads) lookup_kernel(const T* __restrict__ table,
                                                              int64_t stride, int64_t rows, I dim,
                                                              I skip, I over,
                                                              const void* __restrict__ index,
                                                              int index_bytes, I total,
                                                              float scale, T* __restrict__ out) {
  constexpr int N = Vec16<T>::N;
  const I vecs = total / N;
  const T* end = table + (rows - 1) * stride + (int64_t)dim;
  const I v0 = (I)blockIdx.x * (kLookThreads * kLookVecs) + threadIdx.x;
  int64_t r[kLookVecs], next[kLookVecs];
  I c[kLookVecs];
  uint4 u[kLookVecs], w[kLookVecs];
  I t = v0 * N / dim, col = v0 * N - t * dim;
#pragma unroll
  for (int k = 0; k < kLookVecs; ++k) {
    const I v = v0 + k * kLookThreads;
    r[k] = next[k] = -1;
    if (k > 0) {
      t += skip;
      col += over;
      if (col >= dim) {
        col -= dim;
        ++t;
      }
    }
    c[k] = col;
    if (v < vecs) {
      r[k] = index_at(index, index_bytes, (int64_t)t);
      if (!kAligned && c[k] + N > dim) next[k] = index_at(index, index_bytes, (int64_t)t + 1);
    }
  }
#pragma unroll
  for (int k = 0; k < kLookVecs; ++k) {
    if (r[k] >= 0 && r[k] < rows) {
      const T* p = table + r[k] * stride + (int64_t)c[k];
      u[k] = kAligned ? __ldg(reinterpret_cast<const uint4*>(p)) : load16(p, table, end);
    }
    if (!kAligned && next[k] >= 0 && next[k] < rows)
      w[k] = load16(table + next[k] * stride + (int64_t)c[k] - (int64_t)dim, table, end);
  }
#pragma unroll
  for (int k = 0; k < kLookVecs; ++k) {
    const I v = v0 + k * kLookThreads;
    if (v >= vecs) continue;
    float f[N];
    if (r[k] >= 0 && r[k] < rows) {
      unpack(u[k], f, (const T*)nullptr);
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] *= scale;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) f[j] = __int_as_float(0x7fc00000);
    }
    if (!kAligned && c[k] + N > dim) {
      float h[N];
      const bool on = next[k] >= 0 && next[k] < rows;
      if (on) unpack(w[k], h, (const T*)nullptr);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (c[k] + j >= dim) f[j] = on ? h[j] * scale : __int_as_float(0x7fc00000);
    }
    reinterpret_cast<uint4*>(out)[v] = pack(f, (const T*)nullptr);
  }
  if (!kAligned && blockIdx.x == 0 && threadIdx.x < total - vecs * N) {
    const I e = vecs * N + threadIdx.x, te = e / dim;
    const int64_t row = index_at(index, index_bytes, (int64_t)te);
    out[e] = from_f32<T>(row >= 0 && row < rows
                             ? to_f32(table[row * stride + (int64_t)(e - te * dim)]) * scale
                             : __int_as_float(0x7fc00000));
  }
}

// Rows narrower than a vector: an element for each thread.
template <typename T>
__global__ void __launch_bounds__(kLookThreads) lookup_narrow_kernel(
    const T* __restrict__ table, int64_t stride, int64_t rows, uint32_t dim,
    const void* __restrict__ index, int index_bytes, int64_t total, float scale,
    T* __restrict__ out) {
  const int64_t e = (int64_t)blockIdx.x * kLookThreads + threadIdx.x;
  if (e >= total) return;
  const int64_t t = total < (int64_t(1) << 32) ? (int64_t)((uint32_t)e / dim) : e / dim;
  const int64_t row = index_at(index, index_bytes, t);
  out[e] = from_f32<T>(row >= 0 && row < rows ? to_f32(table[row * stride + (e - t * dim)]) * scale
                                              : __int_as_float(0x7fc00000));
}

template <typename T>
static int launch_lookup(const void* table, int64_t stride, int64_t rows, int64_t dim,
                         const void* index, int index_bytes, int64_t count, float scale, void* out,
                         cudaStream_t st) {
  constexpr int N = Vec16<T>::N;
  const int64_t total = count * dim;
  if (dim < N) {
    const int64_t grid = ceil_div64(total, kLookThreads);
    SINKSLOT_REQUIRE(grid <= 0x7fffffff, "lookup: sizes too large");
    lookup_narrow_kernel<T><<<(unsigned)grid, kLookThreads, 0, st>>>(
        (const T*)table, stride, rows, (uint32_t)dim, index, index_bytes, total, scale, (T*)out);
    SINKSLOT_CHECK_LAUNCH();
    return kOk;
  }
  const int64_t grid = ceil_div64(total / N + 1, kLookThreads * kLookVecs);
  SINKSLOT_REQUIRE(grid <= 0x7fffffff, "lookup: sizes too large");
  const bool rows16 = (reinterpret_cast<uintptr_t>(table) & 15) == 0 && dim % N == 0 &&
                      stride % N == 0;
  const bool narrow = total + kLookThreads * kLookVecs * N < (int64_t(1) << 32);
#define GO(I, A)                                                                          \
  lookup_kernel<T, I, A><<<(unsigned)grid, kLookThreads, 0, st>>>(                        \
      (const T*)table, stride, rows, (I)dim, (I)(kLookThreads * N / dim),                 \
      (I)(kLookThreads * N % dim), index, index_bytes, (I)total, scale, (T*)out)
  if (rows16) {
    if (narrow) GO(uint32_t, true); else GO(int64_t, true);
  } else {
    if (narrow) GO(uint32_t, false); else GO(int64_t, false);
  }
#undef GO
  SINKSLOT_CHECK_LAUNCH();
  return kOk;
}

int lookup(const void* table, int dtype, int64_t stride, int64_t rows, int64_t dim,
           const void* index, int index_bytes, int64_t count, double scale, void* out,
           cudaStream_t st) {
  SINKSLOT_REQUIRE(dtype_ok(dtype), "lookup: dtype must be 0, 1 or 2");
  SINKSLOT_REQUIRE(rows >= 1 && dim >= 1 && count >= 0 && stride >= 0, "lookup: bad sizes");
  SINKSLOT_REQUIRE(index_bytes == 4 || index_bytes == 8, "lookup: index must be int32 or int64");
  if (count == 0) return kOk;
  SINKSLOT_REQUIRE(table && index && out, "lookup: null argument");
  SINKSLOT_REQUIRE((reinterpret_cast<uintptr_t>(out) & 15) == 0,
                   "lookup: out must begin on a 16-byte boundary");
  const float s = (float)scale;
  if (dtype == kF32)
    return launch_lookup<float>(table, stride, rows, dim, index, index_bytes, count, s, out, st);
  if (dtype == kF16)
    return launch_lookup<__half>(table, stride, rows, dim, index, index_bytes, count, s, out, st);
  return launch_lookup<__nv_bfloat16>(table, stride, rows, dim, index, index_bytes, count, s, out,
                                      st);
}

// --------------------------------------------------------------------------
// Gradient, first part: the tokens sorted by row.
// --------------------------------------------------------------------------

// Sort key: the row, or `rows` for a token that gets no gradient (padding, or an
// index out of range), which sorts behind all rows.
__device__ __forceinline__ uint32_t key_of(const void* index, int bytes, int64_t t, int64_t rows,
                                           int64_t padding) {
  const int64_t r = index_at(index, bytes, t);
  return (uint32_t)(r < 0 || r >= rows || r == padding ? rows : r);
}

// One cluster (the grid's first) sorts; the other CTAs write the table's zeros.
// Least significant digit first, 9 bits a pass: the 18 bits of a table of 2^17
// rows take two.  Each warp ranks a run of its CTA's tokens by digit (match, in
// order), counts are joined over warps, then over the cluster's CTAs, and every
// token goes straight to its place in the shared memory of the CTA that holds it
// in the next pass.
constexpr int kSortCta = 1024;
constexpr int kSortCtaWarps = kSortCta / 32;
constexpr int kDigitBits = 9;
constexpr int kDigits = 1 << kDigitBits;
constexpr int kSortRounds = 11;  // tokens per thread (their keys and values, twice, fill 227 KB)
constexpr int kSortMost = 8 * kSortRounds * kSortCta;  // tokens of the largest cluster: 90112

struct SortShared {
  uint16_t warp_count[kSortCtaWarps][kDigits];
  uint32_t total[8][kDigits];  // digit counts of the cluster's CTAs
  uint32_t base[kDigits];      // where this CTA's tokens of a digit begin
  uint32_t scan[kDigits / 32];
};

constexpr int64_t kFillWithSort = 32 << 20;  // bytes of zeros that the sort hides

static size_t sort_smem(int per) { return sizeof(SortShared) + (size_t)per * 16; }

__global__ void __launch_bounds__(kSortCta, 1) lookup_sort_kernel(
    const void* __restrict__ index, int index_bytes, int count, int64_t rows, int64_t padding,
    int per, int bits, uint2* __restrict__ items, uint32_t* __restrict__ chains,
    uint4* __restrict__ zeros, int64_t zero_vecs, int64_t zero_tail) {
  cg::cluster_group cl = cg::this_cluster();
  const int split = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  chain_release();  // what fills the rest of the table waits for nothing here
  if ((int)blockIdx.x >= split) {
    const int64_t at = ((int64_t)blockIdx.x - split) * kSortCta + threadIdx.x;
    const int64_t step = ((int64_t)gridDim.x - split) * kSortCta;
    for (int64_t i = at; i < zero_vecs; i += step) zeros[i] = make_uint4(0, 0, 0, 0);
    if (at < zero_tail) reinterpret_cast<uint16_t*>(zeros + zero_vecs)[at] = 0;
    return;
  }
  cluster_started();
  extern __shared__ __align__(16) unsigned char raw[];
  SortShared& sh = *reinterpret_cast<SortShared*>(raw);
  uint2* buf = reinterpret_cast<uint2*>(raw + sizeof(SortShared));  // (row, token) twice
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mine = max(0, min(per, count - rank * per));
  const int run = per / kSortCtaWarps;  // a warp's tokens (per is a multiple of kSortCta)
  if (rank == 0 && threadIdx.x == 0) chains[0] = 0;
  int cur = 0;
  for (int shift = 0; shift < bits; shift += kDigitBits, cur ^= 1) {
    const bool last = shift + kDigitBits >= bits;
    for (int i = threadIdx.x; i < kSortCtaWarps * kDigits / 2; i += kSortCta)
      reinterpret_cast<uint32_t*>(sh.warp_count)[i] = 0;
    __syncthreads();
    uint2 item[kSortRounds];
    uint16_t loc[kSortRounds];
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r * 32 >= run) break;
      const int i = warp * run + r * 32 + lane;
      const bool on = i < mine;
      item[r] = make_uint2(0, 0);
      if (on)
        item[r] = shift == 0 ? make_uint2(key_of(index, index_bytes, rank * per + i, rows, padding),
                                          (uint32_t)(rank * per + i))
                             : buf[cur * per + i];
      const uint32_t dg = on ? (item[r].x >> shift) & (kDigits - 1) : kDigits;
      const uint32_t peers = __match_any_sync(0xffffffffu, dg);
      const uint32_t before = __popc(peers & ((1u << lane) - 1u));
      uint32_t base = 0;
      if (on) base = sh.warp_count[warp][dg];
      __syncwarp();
      if (on && before == 0) sh.warp_count[warp][dg] = (uint16_t)(base + __popc(peers));
      __syncwarp();
      loc[r] = (uint16_t)(base + before);
    }
    __syncthreads();
    if (shift == 0) cluster_wait_started();
    if (threadIdx.x < kDigits) {
      uint32_t sum = 0;
#pragma unroll 8
      for (int w = 0; w < kSortCtaWarps; ++w) {
        const uint32_t c = sh.warp_count[w][threadIdx.x];
        sh.warp_count[w][threadIdx.x] = (uint16_t)sum;
        sum += c;
      }
      for (int k = 0; k < split; ++k)
        cl.map_shared_rank(&sh.total[0][0], k)[rank * kDigits + threadIdx.x] = sum;
    }
    cl.sync();
    uint32_t all = 0, ahead = 0, incl = 0;
    if (threadIdx.x < kDigits) {
      for (int k = 0; k < split; ++k) {
        const uint32_t c = sh.total[k][threadIdx.x];
        if (k < rank) ahead += c;
        all += c;
      }
      incl = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
      }
      if (lane == 31) sh.scan[warp] = incl;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      uint32_t before = 0;
      for (int k = 0; k < warp; ++k) before += sh.scan[k];
      sh.base[threadIdx.x] = before + incl - all + ahead;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kSortRounds; ++r) {
      if (r * 32 >= run) break;
      if (warp * run + r * 32 + lane < mine) {
        const uint32_t dg = (item[r].x >> shift) & (kDigits - 1);
        const uint32_t pos = sh.base[dg] + sh.warp_count[warp][dg] + loc[r];
        if (last) {
          items[pos] = item[r];
        } else {
          const uint32_t to = pos / (uint32_t)per, at = pos - to * (uint32_t)per;
          cl.map_shared_rank(buf, to)[(cur ^ 1) * per + at] = item[r];
        }
      }
    }
    // (the last pass as well: no CTA leaves while others read or write its memory)
    cl.sync();
  }
}

// More tokens than a cluster holds: the same passes over tiles of kTile tokens, three
// kernels each.  Digit counts of every tile; their sums over the tiles before (a warp
// for each digit); tokens ranked within their tile, put in digit order in shared
// memory and written out run by run.
constexpr int kTileThreads = 512;
constexpr int kTileWarps = kTileThreads / 32;
constexpr int kTileRounds = 8;
constexpr int kTile = kTileThreads * kTileRounds;

struct TileSource {
  const void* index;  // the first pass reads the indices, later ones the items
  int index_bytes;
  int64_t count, rows, padding;
  const uint2* items;
  int shift;
};

__device__ __forceinline__ uint2 tile_item(const TileSource& a, int64_t t) {
  return a.items ? a.items[t]
                 : make_uint2(key_of(a.index, a.index_bytes, t, a.rows, a.padding), (uint32_t)t);
}

__global__ void __launch_bounds__(kTileThreads) tile_count_kernel(TileSource a, int tiles,
                                                                  uint32_t* __restrict__ counts) {
  __shared__ uint32_t n[kDigits];
  for (int i = threadIdx.x; i < kDigits; i += kTileThreads) n[i] = 0;
  __syncthreads();
  chain_enter();
  chain_release();
  const int64_t t0 = (int64_t)blockIdx.x * kTile + threadIdx.x;
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int64_t t = t0 + r * kTileThreads;
    if (t < a.count) atomicAdd(&n[(tile_item(a, t).x >> a.shift) & (kDigits - 1)], 1u);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kDigits; i += kTileThreads)
    counts[(int64_t)i * tiles + blockIdx.x] = n[i];
}

__global__ void __launch_bounds__(256) tile_scan_kernel(uint32_t* __restrict__ counts, int tiles,
                                                        uint32_t* __restrict__ totals) {
  chain_enter();
  chain_release();
  const int digit = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  uint32_t* c = counts + (int64_t)digit * tiles;
  uint32_t before = 0;
  for (int k = 0; k < tiles; k += 32) {
    const uint32_t v = k + lane < tiles ? c[k + lane] : 0;
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (k + lane < tiles) c[k + lane] = before + incl - v;
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  if (lane == 0) totals[digit] = before;
}

// Sum of v over the threads before this one; kDigits threads, all of the CTA.
__device__ __forceinline__ uint32_t digits_before(uint32_t v, uint32_t* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  uint32_t before = 0;
  for (int k = 0; k < warp; ++k) before += warp_sum[k];
  return before + incl - v;
}

__global__ void __launch_bounds__(kTileThreads) tile_scatter_kernel(
    TileSource a, int tiles, const uint32_t* __restrict__ counts,
    const uint32_t* __restrict__ totals, uint2* __restrict__ out) {
  static_assert(kTileThreads == kDigits, "a thread for each digit");
  __shared__ uint2 sorted[kTile];  // before it, the warps' digit counts
  uint16_t(*warp_count)[kDigits] = reinterpret_cast<uint16_t(*)[kDigits]>(sorted);
  static_assert(sizeof(uint16_t) * kTileWarps * kDigits <= sizeof(uint2) * kTile, "fits");
  __shared__ uint32_t begin[kDigits], global[kDigits], warp_sum[kTileWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < kTileWarps * kDigits / 2; i += kTileThreads)
    reinterpret_cast<uint32_t*>(warp_count)[i] = 0;
  __syncthreads();
  chain_enter();
  chain_release();
  const int64_t t0 = (int64_t)blockIdx.x * kTile;
  const int mine = (int)min((int64_t)kTile, a.count - t0);
  uint2 item[kTileRounds];
  uint16_t loc[kTileRounds];
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int i = warp * (kTile / kTileWarps) + r * 32 + lane;
    item[r] = i < mine ? tile_item(a, t0 + i) : make_uint2(0, 0);
  }
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const bool on = warp * (kTile / kTileWarps) + r * 32 + lane < mine;
    const uint32_t dg = on ? (item[r].x >> a.shift) & (kDigits - 1) : kDigits;
    const uint32_t peers = __match_any_sync(0xffffffffu, dg);
    const uint32_t before = __popc(peers & ((1u << lane) - 1u));
    uint32_t base = 0;
    if (on) base = warp_count[warp][dg];
    __syncwarp();
    if (on && before == 0) warp_count[warp][dg] = (uint16_t)(base + __popc(peers));
    __syncwarp();
    loc[r] = (uint16_t)(base + before);
  }
  __syncthreads();
  {
    const int d = threadIdx.x;
    uint32_t sum = 0;
#pragma unroll
    for (int w = 0; w < kTileWarps; ++w) {
      const uint32_t c = warp_count[w][d];
      warp_count[w][d] = (uint16_t)sum;
      sum += c;
    }
    begin[d] = digits_before(sum, warp_sum);
    global[d] = digits_before(totals[d], warp_sum) + counts[(int64_t)d * tiles + blockIdx.x];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r)
    if (warp * (kTile / kTileWarps) + r * 32 + lane < mine) {
      const uint32_t dg = (item[r].x >> a.shift) & (kDigits - 1);
      loc[r] = (uint16_t)(begin[dg] + warp_count[warp][dg] + loc[r]);
    }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r)
    if (warp * (kTile / kTileWarps) + r * 32 + lane < mine) sorted[loc[r]] = item[r];
  __syncthreads();
  for (int i = threadIdx.x; i < mine; i += kTileThreads) {
    const uint2 v = sorted[i];
    const uint32_t dg = (v.x >> a.shift) & (kDigits - 1);
    out[global[dg] + (i - begin[dg])] = v;
  }
}

// Zeros, 8 KB for each CTA, while the sort runs (launched behind it without
// waiting for it; the last CTA waits at its end, so that this kernel's completion
// stands for both).  1 GiB: 7.4 TB/s, where CTAs that stride over the table reach
// 6.0 and the sort kernel's own spare CTAs 4.4.
constexpr int kFillVecs = 2;
__global__ void __launch_bounds__(kLookThreads) lookup_zero_kernel(uint4* __restrict__ zeros,
                                                                   int64_t vecs, int64_t tail) {
  const int64_t at = (int64_t)blockIdx.x * (kLookThreads * kFillVecs) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < kFillVecs; ++k)
    if (at + k * kLookThreads < vecs) zeros[at + k * kLookThreads] = make_uint4(0, 0, 0, 0);
  if (blockIdx.x == gridDim.x - 1) {
    if (threadIdx.x < tail) reinterpret_cast<uint16_t*>(zeros + vecs)[threadIdx.x] = 0;
    chain_enter();
  }
}

// --------------------------------------------------------------------------
// Gradient, second part: the sums.  VN columns for each thread: a 16-byte vector
// of the gradient's row, cut by that row's own boundaries (chunk j holds the
// columns [j VN - shift, (j + 1) VN - shift), shift the row's phase), or, for
// narrow tables, one column.
// --------------------------------------------------------------------------
constexpr int kAhead = 8;  // loads in flight per thread; windows are multiples of it

struct SumArgs {
  const uint2* items;  // (row, token), sorted
  int64_t count, rows, stride, dim, ncv;
  int window;
  float scale;
  float* part;
  uint32_t* chains;  // [0]: how many; then the windows where a crossing row begins
};

template <typename T, int VN>
__device__ __forceinline__ int64_t first_column(const T* row, int64_t j) {
  if (VN == 1) return j;
  return j * VN - (int64_t)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

template <typename T, int VN>
__device__ __forceinline__ void store_row(T* row, int64_t j, int64_t dim, const float (&acc)[VN],
                                          float scale) {
  const int64_t c = first_column<T, VN>(row, j);
  if constexpr (VN == 1) {
    row[c] = from_f32<T>(acc[0] * scale);
  } else {
    float f[VN];
#pragma unroll
    for (int k = 0; k < VN; ++k) f[k] = acc[k] * scale;
    if (c >= 0 && c + VN <= dim) {
      *reinterpret_cast<uint4*>(row + c) = pack(f, (const T*)nullptr);
    } else {
#pragma unroll
      for (int k = 0; k < VN; ++k)
        if (c + k >= 0 && c + k < dim) row[c + k] = from_f32<T>(f[k]);
    }
  }
}

template <int VN>
__device__ __forceinline__ float* part_at(const SumArgs& a, int64_t slot, int64_t j) {
  return a.part + (slot * a.ncv + j) * VN;
}

template <int VN>
__device__ __forceinline__ void store_part(float* p, const float (&acc)[VN]) {
#pragma unroll
  for (int k = 0; k < VN; ++k) p[k] = acc[k];
}

// Where a finished sum goes.  part slot 2 w: the sum of window w's first row where
// that row began in an earlier window; 2 w + 1: of its last row where it began here
// and goes on.  (Not inlined: the summing loops call it at each of their steps.)
template <typename T, int VN>
__device__ __noinline__ void put_row(T* out, int64_t dim, uint32_t row, int64_t j, float scale,
                                     float a0, float a1, float a2, float a3, float a4, float a5,
                                     float a6, float a7) {
  const float all[8] = {a0, a1, a2, a3, a4, a5, a6, a7};
  float acc[VN];
#pragma unroll
  for (int k = 0; k < VN; ++k) acc[k] = all[k];
  store_row<T, VN>(out + (int64_t)row * dim, j, dim, acc, scale);
}

template <typename T, int VN>
__device__ __forceinline__ void put_sum(const SumArgs& a, T* out, bool head, int64_t w, int64_t j,
                                        uint32_t row, const float (&acc)[VN]) {
  if (head) {
    store_part<VN>(part_at<VN>(a, 2 * w, j), acc);
  } else if constexpr (VN == 8) {
    put_row<T, VN>(out, a.dim, row, j, a.scale, acc[0], acc[1], acc[2], acc[3], acc[4], acc[5],
                   acc[6], acc[7]);
  } else if constexpr (VN == 4) {
    put_row<T, VN>(out, a.dim, row, j, a.scale, acc[0], acc[1], acc[2], acc[3], 0, 0, 0, 0);
  } else {
    store_row<T, VN>(out + (int64_t)row * a.dim, j, a.dim, acc, a.scale);
  }
}

// kAligned: all rows of both arrays begin on 16-byte boundaries.  The windows'
// keys and positions are staged in shared memory where a CTA meets few windows
// (ncv of kStageFrom or more).  Registers are held to 64 for four CTAs on an SM
// (5003 x 771 fp16, 40009 tokens, sort and all: 87 us at three, 73 at four, 89 at five).
// The vector variants spill at four already (staged, 16-bit types: 112 bytes stored and
// 132 loaded for each thread on any alignment, 44 and 104 aligned; float32: 28 and 24,
// 36 and 96).
constexpr int kStageFrom = 64;
constexpr int kStaged = (kLookThreads / kStageFrom + 1) * 64;

template <typename T, int VN, bool kAligned, bool kStage>
__global__ void __launch_bounds__(kLookThreads, 4) lookup_sum_kernel(SumArgs a,
                                                                  const T* __restrict__ g,
                                                                  T* __restrict__ out) {
  __shared__ uint2 staged[kStage ? kStaged : 1];
  const int64_t q = (int64_t)blockIdx.x * kLookThreads + threadIdx.x;
  const int64_t w = q / a.ncv, j = q - w * a.ncv;
  const int64_t i0 = w * a.window;
  int64_t s0 = 0;
  if constexpr (kStage) {
    s0 = (int64_t)blockIdx.x * kLookThreads / a.ncv * a.window;
    const int64_t s1 =
        min(a.count, (((int64_t)blockIdx.x + 1) * kLookThreads - 1) / a.ncv * a.window + a.window);
    for (int64_t i = s0 + threadIdx.x; i < s1; i += kLookThreads)
      staged[i - s0] = a.items[i];
    __syncthreads();
  }
  auto entry = [&](int64_t i) {
    if constexpr (kStage)
      return staged[i - s0];
    else
      return a.items[i];
  };
  chain_release();
  if (i0 >= a.count) return;
  const int n = (int)min((int64_t)a.window, a.count - i0);
  uint32_t cur = entry(i0).x;
  if (cur >= a.rows) return;
  const T* gend = g + (a.count - 1) * a.stride + a.dim;
  bool head = i0 > 0 && a.items[i0 - 1].x == cur;
  float acc[VN];
#pragma unroll
  for (int k = 0; k < VN; ++k) acc[k] = 0.0f;
  for (int b = 0; b < n; b += kAhead) {
    uint32_t key[kAhead];
    uint4 u[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const uint2 en = b + k < n ? entry(i0 + b + k) : make_uint2(0xffffffffu, 0);
      key[k] = en.x;
      u[k] = make_uint4(0, 0, 0, 0);
      if (key[k] < a.rows) {
        const T* p = g + (int64_t)en.y * a.stride;
        if constexpr (VN == 1) {
          u[k].x = __float_as_uint(to_f32(p[j]));
        } else if constexpr (kAligned) {
          u[k] = __ldg(reinterpret_cast<const uint4*>(p) + j);
        } else {
          u[k] = load16(p + first_column<T, VN>(out + (int64_t)key[k] * a.dim, j), g, gend);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (b + k >= n) break;
      if (key[k] != cur) {
        put_sum<T, VN>(a, out, head, w, j, cur, acc);
        head = false;
        cur = key[k];
        if (cur >= a.rows) return;  // the tokens without a gradient
#pragma unroll
        for (int m = 0; m < VN; ++m) acc[m] = 0.0f;
      }
      if constexpr (VN == 1) {
        acc[0] += __uint_as_float(u[k].x);
      } else {
        float f[VN];
        unpack(u[k], f, (const T*)nullptr);
#pragma unroll
        for (int m = 0; m < VN; ++m) acc[m] += f[m];
      }
    }
  }
  if (!head && i0 + n < a.count && a.items[i0 + n].x == cur) {
    store_part<VN>(part_at<VN>(a, 2 * w + 1, j), acc);
    // (the order of the list decides nothing but who joins which row)
    if (j == 0) a.chains[1 + atomicAdd(a.chains, 1u)] = (uint32_t)w;
  } else {
    put_sum<T, VN>(a, out, head, w, j, cur, acc);
  }
}

// Rows that cross windows.  A warp takes a row and up to 32 chunks of its columns
// (blockIdx.y): where there are fewer, its lanes share the row's windows as well.  Rows
// over many windows are left to the CTA's warps together.  All sums are joined in an
// order that the row's place alone decides.
constexpr int kLongChain = 4;  // windows for each lane group of a warp

template <typename T, int VN>
__global__ void __launch_bounds__(kLookThreads) lookup_join_kernel(SumArgs a, int lanes,
                                                                   T* __restrict__ out) {
  constexpr int kWarps = kLookThreads / 32;
  __shared__ float sums[kWarps][32][VN + 1];
  __shared__ uint32_t long_w[kWarps], long_n[kWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int parts = 32 / lanes, mine = lane / lanes;  // lane groups, and this lane's
  const int64_t j = (int64_t)blockIdx.y * 32 + lane % lanes;
  const bool on = j < a.ncv;
  // windows [k0, k1) of the row that begins in window w: w's tail, then heads
  auto add = [&](float (&acc)[VN], int64_t w, int64_t k0, int64_t k1) {
#pragma unroll 4
    for (int64_t k = k0; k < k1; ++k) {
      const float* p = part_at<VN>(a, 2 * (w + k) + (k == 0), j);
      if constexpr (VN == 1) {
        acc[0] += *p;
      } else {
#pragma unroll
        for (int m = 0; m < VN; m += 4) {
          const float4 v = *reinterpret_cast<const float4*>(p + m);
          acc[m] += v.x; acc[m + 1] += v.y; acc[m + 2] += v.z; acc[m + 3] += v.w;
        }
      }
    }
  };
  auto over_groups = [&](float (&acc)[VN]) {
    for (int d = lanes; d < 32; d <<= 1) {
#pragma unroll
      for (int m = 0; m < VN; ++m) acc[m] += __shfl_xor_sync(0xffffffffu, acc[m], d);
    }
  };
  chain_enter();
  const uint32_t chains = a.chains[0];
  const int64_t windows = (a.count + a.window - 1) / a.window;
  // (CTA by CTA first, warp by warp then: a few rows go to as many CTAs)
  for (uint32_t item0 = blockIdx.x; item0 < chains; item0 += gridDim.x * kWarps) {
    const uint32_t item = item0 + gridDim.x * warp;
    int64_t w = 0, n = 0;
    uint32_t cur = 0;
    if (item < chains) {
      w = a.chains[1 + item];
      cur = a.items[(w + 1) * a.window - 1].x;
      // the first window behind w that does not begin with this row: the next 32, then
      // 32 probes a step; lo begins with it, the answer is in (lo, hi]
      int64_t lo = w + 1, hi = windows, step = 1;
      while (hi - lo > 1) {
        const int64_t at = lo + step * (lane + 1);
        const bool same = at < hi && a.items[at * a.window].x == cur;
        const int found = __popc(__ballot_sync(0xffffffffu, same));  // a prefix of the lanes
        const int64_t next = lo + step * (found + 1);
        lo += step * found;
        if (found < 32 && next < hi) hi = next;
        step = (hi - lo + 31) / 32;
      }
      n = hi - w;  // partial sums
    }
    const bool lengthy = n > (int64_t)kLongChain * parts;
    if (n > 0 && !lengthy) {
      float acc[VN];
#pragma unroll
      for (int m = 0; m < VN; ++m) acc[m] = 0.0f;
      if (on) add(acc, w, n * mine / parts, n * (mine + 1) / parts);
      over_groups(acc);
      if (on && mine == 0) store_row<T, VN>(out + (int64_t)cur * a.dim, j, a.dim, acc, a.scale);
    }
    __syncthreads();
    if (lane == 0) {
      long_w[warp] = (uint32_t)w;
      long_n[warp] = lengthy ? (uint32_t)n : 0;
    }
    __syncthreads();
    for (int c = 0; c < kWarps; ++c) {
      if (long_n[c] == 0) continue;
      const int64_t lw = long_w[c], ln = long_n[c];
      const int all = kWarps * parts, me = warp * parts + mine;
      float acc[VN];
#pragma unroll
      for (int m = 0; m < VN; ++m) acc[m] = 0.0f;
      if (on) add(acc, lw, ln * me / all, ln * (me + 1) / all);
      over_groups(acc);
      __syncthreads();
#pragma unroll
      for (int m = 0; m < VN; ++m) sums[warp][lane][m] = acc[m];
      __syncthreads();
      if (warp == 0 && mine == 0 && on) {
        for (int k = 1; k < kWarps; ++k) {
#pragma unroll
          for (int m = 0; m < VN; ++m) acc[m] += sums[k][lane][m];
        }
        const uint32_t row = a.items[(lw + 1) * a.window - 1].x;
        store_row<T, VN>(out + (int64_t)row * a.dim, j, a.dim, acc, a.scale);
      }
    }
  }
}

// Tokens per window: as few as keep the GPU's threads busy about once over (small
// calls want threads, large ones few partial sums), at most 64.
static int window_of(int64_t count, int64_t dim) {
  int w = kAhead;
  while (w < 64 && count / w * (dim / 8 + 1) > (int64_t)kNumSMs * 1024) w *= 2;
  return w;
}

struct LookWs {
  uint2 *items, *other;
  uint32_t *chains, *counts, *totals;
  float* part;
};

static void carve_look(Carver& cv, LookWs& w, int64_t count, int64_t dim) {
  const int64_t e = count > 0 ? count : 1;
  const int64_t windows = ceil_div64(e, window_of(e, dim));
  w.chains = cv.take<uint32_t>(windows + 1);
  w.items = cv.take<uint2>(e);
  w.other = nullptr;
  w.counts = w.totals = nullptr;
  if (e > kSortMost) {
    w.other = cv.take<uint2>(e);
    w.counts = cv.take<uint32_t>(kDigits * ceil_div64(e, kTile));
    w.totals = cv.take<uint32_t>(kDigits);
  }
  w.part = cv.take<float>((size_t)(2 * windows * (dim + 16)));  // a row cut by its boundaries
}

size_t lookup_grad_workspace_bytes(int64_t count, int64_t rows, int64_t dim) {
  (void)rows;
  Carver cv(nullptr, 0);
  LookWs w;
  carve_look(cv, w, count, dim);
  return cv.used;
}

template <typename T, int VN, bool kAligned>
static int launch_sums(SumArgs a, const void* g, void* out, cudaStream_t st) {
  a.ncv = kAligned ? a.dim / VN : (a.dim + 2 * VN - 2) / VN;
  const int64_t windows = ceil_div64(a.count, a.window);
  const int64_t grid = ceil_div64(windows * a.ncv, kLookThreads);
  const int64_t groups = ceil_div64(a.ncv, 32);
  SINKSLOT_REQUIRE(grid <= 0x7fffffff && groups <= 65535, "lookup_grad: sizes too large");
  if (a.ncv >= kStageFrom)
    lookup_sum_kernel<T, VN, kAligned, true><<<(unsigned)grid, kLookThreads, 0, st>>>(
        a, (const T*)g, (T*)out);
  else
    lookup_sum_kernel<T, VN, kAligned, false><<<(unsigned)grid, kLookThreads, 0, st>>>(
        a, (const T*)g, (T*)out);
  SINKSLOT_CHECK_LAUNCH();
  if (windows == 1) return kOk;  // nothing crosses
  int lanes = 1;
  while (lanes < 32 && lanes < a.ncv) lanes *= 2;
  int64_t x = ceil_div64(6 * num_sms(), groups);
  if (x > windows) x = windows;
  SINKSLOT_CUDA_TRY(launch_chained(lookup_join_kernel<T, VN>, dim3((unsigned)x, (unsigned)groups),
                                   dim3(kLookThreads), 0, st, a, lanes, (T*)out));
  return kOk;
}

template <typename T>
static int launch_sums_of(SumArgs a, const void* g, void* out, cudaStream_t st) {
  constexpr int N = Vec16<T>::N;
  // under two vectors, a thread for each column: vectors would be mostly edges
  if (a.dim < 2 * N) return launch_sums<T, 1, true>(a, g, out, st);
  const bool rows16 = (reinterpret_cast<uintptr_t>(g) & 15) == 0 && a.dim % N == 0 &&
                      a.stride % N == 0;
  return rows16 ? launch_sums<T, N, true>(a, g, out, st) : launch_sums<T, N, false>(a, g, out, st);
}

// Sorts the tokens and writes the table's zeros.
static int sort_tokens(const void* index, int index_bytes, int64_t count, int64_t rows,
                       int64_t padding, void* out, int64_t out_bytes, LookWs& w,
                       cudaStream_t st) {
  const int bits = bits_for((uint64_t)rows + 1);
  if (count > kSortMost) {
    SINKSLOT_CUDA_TRY(cudaMemsetAsync(out, 0, (size_t)out_bytes, st));
    SINKSLOT_CUDA_TRY(cudaMemsetAsync(w.chains, 0, sizeof(uint32_t), st));
    const int tiles = (int)ceil_div64(count, kTile);
    const int passes = (bits + kDigitBits - 1) / kDigitBits;
    TileSource a = {index, index_bytes, count, rows, padding, nullptr, 0};
    for (int k = 0; k < passes; ++k, a.shift += kDigitBits) {
      uint2* to = (passes - k) & 1 ? w.items : w.other;  // the last pass fills w.items
      SINKSLOT_CUDA_TRY(launch_chained(tile_count_kernel, dim3((unsigned)tiles),
                                       dim3(kTileThreads), 0, st, a, tiles, w.counts));
      SINKSLOT_CUDA_TRY(launch_chained(tile_scan_kernel, dim3(kDigits / 8), dim3(256), 0, st,
                                       w.counts, tiles, w.totals));
      SINKSLOT_CUDA_TRY(launch_chained(tile_scatter_kernel, dim3((unsigned)tiles),
                                       dim3(kTileThreads), 0, st, a, tiles,
                                       (const uint32_t*)w.counts, (const uint32_t*)w.totals, to));
      a.items = to;
    }
    return kOk;
  }
  int split = 1;
  while (split < 8 && count > (int64_t)split * 4 * kSortCta) split *= 2;
  const int per = (int)(ceil_div64(ceil_div64(count, split), kSortCta) * kSortCta);
  {
    // the shared-memory limit is a per-device function attribute
    static bool configured[64] = {};
    int dev = 0;
    SINKSLOT_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
      SINKSLOT_CUDA_TRY(cudaFuncSetAttribute(lookup_sort_kernel,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)sort_smem(kSortRounds * kSortCta)));
      if (dev >= 0 && dev < 64) configured[dev] = true;
    }
  }
  // zeros: by spare CTAs of the sort's own launch while that hides them
  const int64_t vecs = out_bytes / 16, tail = (out_bytes - vecs * 16) / 2;
  const bool apart = out_bytes > kFillWithSort;
  int64_t fill = apart ? 0 : ceil_div64(vecs > 0 ? vecs : 1, (int64_t)kSortCta * 4);
  const int64_t room = num_sms() - split;
  if (fill > room) fill = room;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(split + ceil_div64(fill, split) * split));
  cfg.blockDim = dim3(kSortCta);
  cfg.dynamicSmemBytes = sort_smem(per);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)split;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SINKSLOT_CUDA_TRY(cudaLaunchKernelEx(
      &cfg, lookup_sort_kernel, index, index_bytes, (int)count, rows, padding, per, bits,
      w.items, w.chains, (uint4*)out, vecs, tail));
  if (apart) {
    const int64_t grid = ceil_div64(vecs, kLookThreads * kFillVecs);
    SINKSLOT_REQUIRE(grid <= 0x7fffffff, "lookup_grad: sizes too large");
    SINKSLOT_CUDA_TRY(launch_chained(lookup_zero_kernel, dim3((unsigned)grid), dim3(kLookThreads),
                                     0, st, (uint4*)out, vecs, tail));
  }
  return kOk;
}

// --------------------------------------------------------------------------
// Few rows or few tokens: one launch.  A CTA for each row of the table (and 256 of its
// columns) looks through all indices, lists the tokens that name the row, and adds
// their gradients up: `lanes` threads for the columns, the others take every
// (256 / lanes)th token of the list; their sums are joined as a tree.  The order
// follows from the indices alone.
// --------------------------------------------------------------------------
constexpr int kRowScan = 8;  // indices under way for each thread
constexpr int kRowTile = kRowScan * kLookThreads;

template <typename T, typename I>
__global__ void __launch_bounds__(kLookThreads) lookup_row_sum_kernel(
    const I* __restrict__ index, int count, int64_t padding, const T* __restrict__ g,
    int64_t stride, int64_t dim, int lanes, float scale, T* __restrict__ out) {
  constexpr int kWarps = kLookThreads / 32;
  __shared__ int list[2][kRowTile];
  __shared__ int found[2][kWarps];
  __shared__ float part[kLookThreads];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slice = threadIdx.x / (unsigned)lanes, slices = kLookThreads / lanes;
  const int64_t col = (int64_t)blockIdx.y * kLookThreads + (threadIdx.x & (lanes - 1));
  const bool on = col < dim;
  const T* at = g + (on ? col : 0);
  float sum = 0.0f;
  const int end = row == padding ? 0 : count;
  for (int first = 0, turn = 0; first < end; first += kRowTile, turn ^= 1) {
    I idx[kRowScan];
#pragma unroll
    for (int k = 0; k < kRowScan; ++k) {
      const int i = first + k * kLookThreads + (int)threadIdx.x;
      idx[k] = i < end ? __ldg(index + i) : (I)-1;
    }
    uint32_t hits[kRowScan];
    int mine = 0;
#pragma unroll
    for (int k = 0; k < kRowScan; ++k) {
      hits[k] = __ballot_sync(0xffffffffu, (int64_t)idx[k] == row);
      mine += __popc(hits[k]);
    }
    if (lane == 0) found[turn][warp] = mine;
    __syncthreads();
    int to = 0, n = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) to = n;
      n += found[turn][w];
    }
    if (n == 0) continue;
#pragma unroll
    for (int k = 0; k < kRowScan; ++k) {
      if (hits[k] >> lane & 1)
        list[turn][to + __popc(hits[k] & ((1u << lane) - 1u))] =
            first + k * kLookThreads + (int)threadIdx.x;
      to += __popc(hits[k]);
    }
    __syncthreads();  // (the next tile writes the other list)
    int j = slice;
    for (; j + 7 * slices < n; j += 8 * slices) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = to_f32(at[list[turn][j + k * slices] * stride]);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum += v[k];
    }
    for (; j < n; j += slices) sum += to_f32(at[list[turn][j] * stride]);
  }
  if (slices > 1) {
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int k = slices / 2; k >= 1; k /= 2) {
      if (slice < k) part[threadIdx.x] += part[threadIdx.x + k * lanes];
      __syncthreads();
    }
    sum = part[threadIdx.x];
  }
  if (on && slice == 0) out[row * dim + col] = from_f32<T>(sum * scale);
}

static int lanes_of(int64_t dim) {
  int lanes = 1;
  while (lanes < kLookThreads && lanes < dim) lanes *= 2;
  return lanes;
}

// Against the sort, us for the gradient (tokens spread evenly, and all on one row):
//   256 x 3, 10000 tokens      6.1 (16.6), 11.1 (14.6)     512 x 512, 512   4.5 (14.8), 19.6 (14.6)
//   50 x 771, 256              3.3 (14.4), 10.9 (13.8)     64 x 8, 16384    9.0 (19.2), 24.1 (15.2)
//   4096 x 256, 256            8.9 (12.1), 12.5 (13.9)     8192 x 256, 256  15.7 (12.7)
//   2048 x 4, 8192            17.8 (22.0), 12.8 (17.5)     16384 x 64, 64   31.9 (11.3)
// The first limit bounds what one row's tokens may cost, the second the CTAs' launch
// and the third the indices that are read.
static bool few_rows(int64_t count, int64_t rows, int64_t dim) {
  const int64_t ctas = rows * ceil_div64(dim, kLookThreads);
  return count * lanes_of(dim) <= (int64_t(1) << 16) && ctas <= 4096 &&
         ctas * count <= (int64_t(1) << 23);
}

template <typename T>
static int launch_row_sums(const void* index, int index_bytes, int64_t count, int64_t rows,
                           int64_t dim, int64_t padding, const void* g, int64_t stride,
                           float scale, void* out, cudaStream_t st) {
  const dim3 grid((unsigned)rows, (unsigned)ceil_div64(dim, kLookThreads));
  if (index_bytes == 8)
    lookup_row_sum_kernel<T, int64_t><<<grid, kLookThreads, 0, st>>>(
        (const int64_t*)index, (int)count, padding, (const T*)g, stride, dim, lanes_of(dim), scale,
        (T*)out);
  else
    lookup_row_sum_kernel<T, int32_t><<<grid, kLookThreads, 0, st>>>(
        (const int32_t*)index, (int)count, padding, (const T*)g, stride, dim, lanes_of(dim), scale,
        (T*)out);
  SINKSLOT_CHECK_LAUNCH();
  return kOk;
}

int lookup_grad(const void* grad_out, int dtype, int64_t stride, const void* index,
                int index_bytes, int64_t count, int64_t rows, int64_t dim, double scale,
                int64_t padding, void* grad_table, void* ws, size_t ws_bytes, cudaStream_t st) {
  SINKSLOT_REQUIRE(dtype_ok(dtype), "lookup_grad: dtype must be 0, 1 or 2");
  SINKSLOT_REQUIRE(rows >= 1 && rows < (int64_t(1) << 31) && dim >= 1 && count >= 0 && stride >= 0,
                   "lookup_grad: bad sizes");
  SINKSLOT_REQUIRE(count < (int64_t(1) << 31), "lookup_grad: 2^31 tokens or more");
  SINKSLOT_REQUIRE(index_bytes == 4 || index_bytes == 8,
                   "lookup_grad: index must be int32 or int64");
  SINKSLOT_REQUIRE(grad_table, "lookup_grad: null argument");
  SINKSLOT_REQUIRE((reinterpret_cast<uintptr_t>(grad_table) & 15) == 0,
                   "lookup_grad: grad_table must begin on a 16-byte boundary");
  const int64_t out_bytes = rows * dim * dtype_bytes(dtype);
  if (count == 0) {
    SINKSLOT_CUDA_TRY(cudaMemsetAsync(grad_table, 0, (size_t)out_bytes, st));
    return kOk;
  }
  SINKSLOT_REQUIRE(grad_out && index && ws, "lookup_grad: null argument");
  Carver cv(ws, ws_bytes);
  LookWs w;
  carve_look(cv, w, count, dim);
  if (!cv.ok) {
    set_error("lookup_grad: workspace too small");
    return kWorkspaceTooSmall;
  }
  if (few_rows(count, rows, dim)) {
#define GO(T)                                                                                \
  return launch_row_sums<T>(index, index_bytes, count, rows, dim, padding, grad_out, stride, \
                            (float)scale, grad_table, st)
    if (dtype == kF32) GO(float);
    if (dtype == kF16) GO(__half);
    GO(__nv_bfloat16);
#undef GO
  }
  SumArgs a = {};
  SINKSLOT_TRY(sort_tokens(index, index_bytes, count, rows, padding, grad_table, out_bytes, w,
                           st));
  a.items = w.items;
  a.count = count;
  a.rows = rows;
  a.stride = stride;
  a.dim = dim;
  a.window = window_of(count, dim);
  a.scale = (float)scale;
  a.part = w.part;
  a.chains = w.chains;
  if (dtype == kF32) return launch_sums_of<float>(a, grad_out, grad_table, st);
  if (dtype == kF16) return launch_sums_of<__half>(a, grad_out, grad_table, st);
  return launch_sums_of<__nv_bfloat16>(a, grad_out, grad_table, st);
}

}  // namespace sinkslot
