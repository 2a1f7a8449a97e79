// lookup.cu -- rows of a table by index, times a scale, and the table's gradient.
//
//   out[t, :] = scale * table[index[t], :]
//   grad_table[v, :] = scale * sum of grad_out[t, :] over the t with index[t] = v
//
// The gradient's sums run in fp32 in an order that the inputs alone decide (no
// floating atomics): the tokens are sorted by row (stable, so equal rows keep
// their order), cut into windows of equal length whatever the rows' counts, and
// each thread adds up one column vector of one window.  Rows that lie in one window are
// written at once; rows that cross windows leave partial sums, joined by a
// second kernel.  Rows that no token names are zeros.
#include "common.cuh"
#include "primitives.h"
#include "training.h"
#include "vec.cuh"

namespace sinkslot {

constexpr int kLookThreads = 256;

__device__ __forceinline__ int64_t index_at(const void* index, int bytes, int64_t t) {
  return bytes == 8 ? static_cast<const int64_t*>(index)[t]
                    : (int64_t) static_cast<const int32_t*>(index)[t];
}

// VN elements for each thread: a 16-byte vector, or one element where rows do
// not begin on such a boundary.
template <typename T, int VN>
__global__ void __launch_bounds__(kLookThreads) lookup_kernel(const T* __restrict__ table,
                                                              int64_t stride, int64_t rows,
                                                              int64_t dim, int64_t ncv,
                                                              const void* __restrict__ index,
                                                              int index_bytes, int64_t count,
                                                              float scale, T* __restrict__ out) {
  const int64_t total = count * ncv;
  for (int64_t q = (int64_t)blockIdx.x * kLookThreads + threadIdx.x; q < total;
       q += (int64_t)gridDim.x * kLookThreads) {
    const int64_t t = q / ncv, c = (q - t * ncv) * VN;
    const int64_t r = index_at(index, index_bytes, t);
    const bool ok = r >= 0 && r < rows;
    float f[VN];
    if constexpr (VN > 1) {
      if (ok) {
        unpack(__ldg(reinterpret_cast<const uint4*>(table + r * stride + c)), f, (const T*)nullptr);
      }
    } else {
      if (ok) f[0] = to_f32(table[r * stride + c]);
    }
#pragma unroll
    for (int j = 0; j < VN; ++j) f[j] = ok ? f[j] * scale : __int_as_float(0x7fc00000);
    if constexpr (VN > 1)
      *reinterpret_cast<uint4*>(out + t * dim + c) = pack(f, (const T*)nullptr);
    else
      out[t * dim + c] = from_f32<T>(f[0]);
  }
}

static bool aligned16(const void* p, int64_t stride, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride * dtype_bytes(dtype) % 16 == 0;
}

template <typename T>
static int launch_lookup(const void* table, int dtype, int64_t stride, int64_t rows, int64_t dim,
                         const void* index, int index_bytes, int64_t count, float scale, void* out,
                         cudaStream_t st) {
  const bool vec = aligned16(table, stride, dtype) && aligned16(out, dim, dtype);
  const int64_t ncv = vec ? dim / Vec16<T>::N : dim;
  int64_t grid = ceil_div64(count * ncv, kLookThreads);
  if (grid > 0x7fffffff) grid = 0x7fffffff;
  if (vec)
    lookup_kernel<T, Vec16<T>::N><<<(unsigned)grid, kLookThreads, 0, st>>>(
        (const T*)table, stride, rows, dim, ncv, index, index_bytes, count, scale, (T*)out);
  else
    lookup_kernel<T, 1><<<(unsigned)grid, kLookThreads, 0, st>>>(
        (const T*)table, stride, rows, dim, ncv, index, index_bytes, count, scale, (T*)out);
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
  const float s = (float)scale;
  if (dtype == kF32)
    return launch_lookup<float>(table, dtype, stride, rows, dim, index, index_bytes, count, s, out,
                                st);
  if (dtype == kF16)
    return launch_lookup<__half>(table, dtype, stride, rows, dim, index, index_bytes, count, s,
                                 out, st);
  return launch_lookup<__nv_bfloat16>(table, dtype, stride, rows, dim, index, index_bytes, count,
                                      s, out, st);
}

// --------------------------------------------------------------------------
// Gradient
// --------------------------------------------------------------------------
constexpr int kWindow = 32;  // sorted tokens per thread
constexpr int kAhead = 8;    // loads in flight per thread

// Sort keys: the row, or `rows` for a token that gets no gradient (padding, or
// an index out of range), which sorts behind all rows.
__global__ void __launch_bounds__(256) lookup_key_kernel(const void* __restrict__ index,
                                                         int index_bytes, int64_t count,
                                                         int64_t rows, int64_t padding,
                                                         uint32_t* __restrict__ keys) {
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= count) return;
  const int64_t r = index_at(index, index_bytes, t);
  keys[t] = (uint32_t)(r < 0 || r >= rows || r == padding ? rows : r);
}

template <typename T, int VN>
__device__ __forceinline__ void store_row(T* p, const float (&acc)[VN], float scale) {
  float f[VN];
#pragma unroll
  for (int j = 0; j < VN; ++j) f[j] = acc[j] * scale;
  if constexpr (VN > 1)
    *reinterpret_cast<uint4*>(p) = pack(f, (const T*)nullptr);
  else
    *p = from_f32<T>(f[0]);
}

template <int VN>
__device__ __forceinline__ void store_part(float* p, const float (&acc)[VN]) {
#pragma unroll
  for (int j = 0; j < VN; ++j) p[j] = acc[j];
}

// part[(2 w + 0) dim ...]: the sum of window w's first row where that row began
// in an earlier window; part[(2 w + 1) dim ...]: of its last row where it began
// here and goes on in the next window.
template <typename T, int VN>
__global__ void __launch_bounds__(kLookThreads) lookup_grad_kernel(
    const uint32_t* __restrict__ keys, const uint32_t* __restrict__ perm, int64_t count,
    int64_t rows, const T* __restrict__ g, int64_t stride, int64_t dim, int64_t ncv, float scale,
    T* __restrict__ out, float* __restrict__ part) {
  const int64_t q = (int64_t)blockIdx.x * kLookThreads + threadIdx.x;
  const int64_t w = q / ncv, c = (q - w * ncv) * VN;
  const int64_t i0 = w * kWindow;
  if (i0 >= count) return;
  const int n = (int)min((int64_t)kWindow, count - i0);
  uint32_t cur = keys[i0];
  if (cur >= rows) return;
  bool head = i0 > 0 && keys[i0 - 1] == cur;
  float acc[VN];
#pragma unroll
  for (int j = 0; j < VN; ++j) acc[j] = 0.0f;
  for (int b = 0; b < n; b += kAhead) {
    uint32_t key[kAhead];
    float f[kAhead][VN];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      key[k] = b + k < n ? keys[i0 + b + k] : 0xffffffffu;
      if (key[k] < rows) {
        const T* p = g + (int64_t)perm[i0 + b + k] * stride + c;
        if constexpr (VN > 1)
          unpack(__ldg(reinterpret_cast<const uint4*>(p)), f[k], (const T*)nullptr);
        else
          f[k][0] = to_f32(*p);
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      if (b + k >= n) break;
      if (key[k] != cur) {
        if (head)
          store_part<VN>(part + 2 * w * dim + c, acc);
        else
          store_row<T, VN>(out + (int64_t)cur * dim + c, acc, scale);
        head = false;
        cur = key[k];
        if (cur >= rows) return;  // the tokens without a gradient
#pragma unroll
        for (int j = 0; j < VN; ++j) acc[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < VN; ++j) acc[j] += f[k][j];
    }
  }
  const bool on = i0 + n < count && keys[i0 + n] == cur;
  if (head)
    store_part<VN>(part + 2 * w * dim + c, acc);
  else if (on)
    store_part<VN>(part + (2 * w + 1) * dim + c, acc);
  else
    store_row<T, VN>(out + (int64_t)cur * dim + c, acc, scale);
}

// Rows that begin in window w and go on behind it.
template <typename T, int VN>
__global__ void __launch_bounds__(kLookThreads) lookup_join_kernel(
    const uint32_t* __restrict__ keys, int64_t count, int64_t rows, int64_t dim, int64_t ncv,
    float scale, const float* __restrict__ part, T* __restrict__ out) {
  const int64_t q = (int64_t)blockIdx.x * kLookThreads + threadIdx.x;
  const int64_t w = q / ncv, c = (q - w * ncv) * VN;
  const int64_t i0 = w * kWindow, i1 = i0 + kWindow;
  if (i1 >= count) return;
  const uint32_t cur = keys[i1 - 1];
  if (cur >= rows || keys[i1] != cur) return;
  if (i0 > 0 && keys[i0] == cur && keys[i0 - 1] == cur) return;  // began earlier
  float acc[VN];
  const float* p = part + (2 * w + 1) * dim + c;
#pragma unroll
  for (int j = 0; j < VN; ++j) acc[j] = p[j];
  for (int64_t k = w + 1; k * kWindow < count && keys[k * kWindow] == cur; ++k) {
    p = part + 2 * k * dim + c;
#pragma unroll
    for (int j = 0; j < VN; ++j) acc[j] += p[j];
  }
  store_row<T, VN>(out + (int64_t)cur * dim + c, acc, scale);
}

struct LookWs {
  uint32_t *k1, *v1, *k2, *v2;
  int64_t *hist, *stmp;
  float* part;
};

static void carve_look(Carver& cv, LookWs& w, int64_t count, int64_t dim) {
  const int64_t e = count > 0 ? count : 1;
  w.k1 = cv.take<uint32_t>(e); w.v1 = cv.take<uint32_t>(e);
  w.k2 = cv.take<uint32_t>(e); w.v2 = cv.take<uint32_t>(e);
  const int64_t nh = radix_hist_elems(1, e);
  w.hist = cv.take<int64_t>(nh);
  w.stmp = cv.take<int64_t>(scan_tmp_elems(nh));
  w.part = cv.take<float>((size_t)(2 * ceil_div64(e, kWindow) * dim));
}

size_t lookup_grad_workspace_bytes(int64_t count, int64_t rows, int64_t dim) {
  (void)rows;
  Carver cv(nullptr, 0);
  LookWs w;
  carve_look(cv, w, count, dim);
  return cv.used;
}

template <typename T, int VN>
static int launch_sums(const uint32_t* keys, const uint32_t* perm, int64_t count, int64_t rows,
                       const void* g, int64_t stride, int64_t dim, float scale, void* out,
                       float* part, cudaStream_t st) {
  const int64_t ncv = dim / VN;
  const int64_t grid = ceil_div64(ceil_div64(count, kWindow) * ncv, kLookThreads);
  SINKSLOT_REQUIRE(grid <= 0x7fffffff, "lookup_grad: sizes too large");
  lookup_grad_kernel<T, VN><<<(unsigned)grid, kLookThreads, 0, st>>>(
      keys, perm, count, rows, (const T*)g, stride, dim, ncv, scale, (T*)out, part);
  SINKSLOT_CHECK_LAUNCH();
  lookup_join_kernel<T, VN><<<(unsigned)grid, kLookThreads, 0, st>>>(
      keys, count, rows, dim, ncv, scale, part, (T*)out);
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
  SINKSLOT_CUDA_TRY(cudaMemsetAsync(grad_table, 0, (size_t)(rows * dim) * dtype_bytes(dtype), st));
  if (count == 0) return kOk;
  SINKSLOT_REQUIRE(grad_out && index && ws, "lookup_grad: null argument");
  Carver cv(ws, ws_bytes);
  LookWs w;
  carve_look(cv, w, count, dim);
  if (!cv.ok) {
    set_error("lookup_grad: workspace too small");
    return kWorkspaceTooSmall;
  }
  lookup_key_kernel<<<(unsigned)ceil_div64(count, 256), 256, 0, st>>>(index, index_bytes, count,
                                                                     rows, padding, w.k1);
  SINKSLOT_CHECK_LAUNCH();
  bool alt = false;
  SINKSLOT_TRY(radix_sort_pairs<uint32_t>(w.k1, w.v1, w.k2, w.v2, true, 1, count,
                                          bits_for((uint64_t)rows + 1), w.hist, w.stmp, &alt, st));
  const uint32_t* keys = alt ? w.k2 : w.k1;
  const uint32_t* perm = alt ? w.v2 : w.v1;
  const float s = (float)scale;
  const bool vec = aligned16(grad_out, stride, dtype) && aligned16(grad_table, dim, dtype);
#define GO(T)                                                                                    \
  return vec ? launch_sums<T, Vec16<T>::N>(keys, perm, count, rows, grad_out, stride, dim, s,    \
                                           grad_table, w.part, st)                               \
             : launch_sums<T, 1>(keys, perm, count, rows, grad_out, stride, dim, s, grad_table,  \
                                 w.part, st)
  if (dtype == kF32) GO(float);
  if (dtype == kF16) GO(__half);
  GO(__nv_bfloat16);
#undef GO
}

}  // namespace sinkslot
