// The norm over all elements of many buffers - the gradients of a model - and their clipping by it: what a
// training step does between the Allreduce of its gradients and the optimizer.
//
//   norm   = sqrt(sum over tensors and elements of g^2)
//   factor = 1 if norm + eps <= max_norm, else max_norm / (norm + eps)
//   out    = g * factor, rounded once
//
// The list is cut once, when it is made, into chunks of at most kChunkBytes of one tensor, in a table on the
// device; a workgroup takes every gridDim-th chunk, so the cut and the order of all additions depend on the
// list alone.  Squares are exact in 64 bits and are summed there: no fp32 gradient is too large or too small
// to be squared, and the length of the sum does not matter.
#include <algorithm>
#include <memory>
#include <new>
#include <utility>
#include <vector>

#include "alamd_rows.h"

namespace alamd {

// A piece of one tensor.
struct Chunk {
  const char *in;
  char *out;
  unsigned count;  // elements
  int dtype;
};

// Memory from `at` to `end`.
struct Span { uintptr_t at, end; };

}  // namespace alamd

struct alamd_tensor_list {
  int device;
  size_t chunks;
  size_t bytes;
  alamd::Chunk *table;  // in device memory
  void *workspace;      // behind the table
  std::vector<alamd::Span> written, all;  // what the list's tensors occupy, in order and joined where they touch
};

namespace alamd {
namespace {

constexpr int kThreads = 256;
constexpr int kU = 4;  // vectors a lane has under way (2 or 8: up to 3 % slower)
constexpr size_t kChunkBytes = (size_t)64 << 10;
constexpr size_t kParts = ALAMD_GLOBAL_NORM_WORKSPACE_BYTES / sizeof(double);

// ---- norm -------------------------------------------------------------------

template <typename T> __device__ __forceinline__ double square_of(const char *at, unsigned e) {
  const double x = (double)Row<T>::get(at, e);
  return x * x;
}

// The squares of a chunk, this lane's part.
template <typename T, int AUX> __device__ __forceinline__ double chunk_squares(const Chunk &c) {
  constexpr unsigned VE = Row<T>::VE;
  const unsigned head = (unsigned)head_count(sizeof(T), c.in, c.in, c.count), vecs = (c.count - head) / VE;
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(c.in + head * sizeof(T)), 0, (int)(vecs * 16u), kRsrcFlags);
  double a = 0.0;
  for (unsigned i = threadIdx.x; i < vecs + threadIdx.x; i += kThreads * kU) {
    u32x4 raw[kU];  // behind the last vector: zeros
#pragma unroll
    for (int u = 0; u < kU; ++u) raw[u] = __builtin_amdgcn_raw_buffer_load_b128(r, (i + (unsigned)u * kThreads) * 16u, 0, AUX);
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      float x[VE];
      Row<T>::unpack(x, raw[u]);
#pragma unroll
      for (unsigned j = 0; j < VE; ++j) a = fma((double)x[j], (double)x[j], a);
    }
  }
  // the elements in front of the first 64-byte boundary and behind the last vector
  if (threadIdx.x < head) a += square_of<T>(c.in, threadIdx.x);
  const unsigned e = head + vecs * VE + threadIdx.x;
  if (e < c.count) a += square_of<T>(c.in, e);
  return a;
}

// The sum over the workgroup, in every lane.
__device__ __forceinline__ double block_sum(double a) {
  __shared__ double lds[kThreads / 64];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) a += __shfl_xor(a, d);
  if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  a = lds[0];
#pragma unroll
  for (int k = 1; k < kThreads / 64; ++k) a += lds[k];
  return a;
}

template <int AUX> __device__ __forceinline__ double chunk_squares(const Chunk &c) {
  return c.dtype == ALAMD_F32    ? chunk_squares<float, AUX>(c)
         : c.dtype == ALAMD_BF16 ? chunk_squares<bf16_t, AUX>(c)
                                 : chunk_squares<f16_t, AUX>(c);
}

template <int AUX>
__global__ void __launch_bounds__(kThreads) squares_kernel(const Chunk *table, unsigned long long chunks, double *parts) {
  double a = 0.0;
  Chunk next = table[blockIdx.x];
  for (unsigned long long k = blockIdx.x; k < chunks; k += gridDim.x) {
    const Chunk c = next;
    next = table[k + gridDim.x < chunks ? k + gridDim.x : k];
    a += chunk_squares<AUX>(c);
  }
  a = block_sum(a);
  if (threadIdx.x == 0) parts[blockIdx.x] = a;
}

// The norm from the workgroups' parts, in every lane of a workgroup.
__device__ __forceinline__ float norm_of_parts(const double *parts, unsigned n) {
  double a = 0.0;
  for (unsigned k = threadIdx.x; k < n; k += kThreads * 8) {
    double x[8];
#pragma unroll
    for (unsigned u = 0; u < 8; ++u) x[u] = k + u * kThreads < n ? parts[k + u * kThreads] : 0.0;
#pragma unroll
    for (unsigned u = 0; u < 8; ++u) a += x[u];
  }
  return (float)sqrt(block_sum(a));
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double *parts, unsigned n, float *norm) {
  const float x = norm_of_parts(parts, n);
  if (threadIdx.x == 0) *norm = x;
}

// ---- clipping ---------------------------------------------------------------

// A chunk's part that `LANES` lanes with U vectors each take, from vector `from` on; with it the chunk's elements
// outside of its vectors where `ends` is set.
template <typename T, int LANES, int U, int AUX>
__device__ __forceinline__ void scale_part(const Chunk &c, float by, unsigned from, unsigned step, bool ends) {
  constexpr unsigned VE = Row<T>::VE;
  const unsigned head = (unsigned)head_count(sizeof(T), c.out, c.in, c.count), vecs = (c.count - head) / VE;
  const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(c.in + head * sizeof(T)), 0, (int)(vecs * 16u), kRsrcFlags);
  const auto w = __builtin_amdgcn_make_buffer_rsrc(c.out + head * sizeof(T), 0, (int)(vecs * 16u), kRsrcFlags);
  for (unsigned i = from; i < vecs; i += step) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __builtin_amdgcn_raw_buffer_load_b128(r, (i + threadIdx.x + (unsigned)u * LANES) * 16u, 0, AUX);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VE];
      Row<T>::unpack(x, raw[u]);
#pragma unroll
      for (unsigned j = 0; j < VE; ++j) x[j] *= by;
      __builtin_amdgcn_raw_buffer_store_b128(Row<T>::pack(x), w, (i + threadIdx.x + (unsigned)u * LANES) * 16u, 0, kAuxStoreRow);
    }
  }
  if (!ends) return;
  if (threadIdx.x < head) Row<T>::put(c.out, threadIdx.x, Row<T>::get(c.in, threadIdx.x) * by);
  const unsigned e = head + vecs * VE + threadIdx.x;
  if (e < c.count) Row<T>::put(c.out, e, Row<T>::get(c.in, e) * by);
}
template <int LANES, int U, int AUX>
__device__ __forceinline__ void scale_part(const Chunk &c, float by, unsigned from, unsigned step, bool ends) {
  if (c.dtype == ALAMD_F32) scale_part<float, LANES, U, AUX>(c, by, from, step, ends);
  else if (c.dtype == ALAMD_BF16) scale_part<bf16_t, LANES, U, AUX>(c, by, from, step, ends);
  else scale_part<f16_t, LANES, U, AUX>(c, by, from, step, ends);
}

__device__ __forceinline__ float clip_factor(float norm, float max_norm, float eps) {
  norm += eps;
  return norm <= max_norm ? 1.0f : max_norm / norm;
}

// A workgroup a chunk.  Clips to the norm in *norm, or, with PARTS, to the norm that those make, which the first
// workgroup writes to *norm: a launch less.  From the last chunk to the first: what the pass before has read last
// is the likeliest to be in a cache.
template <bool PARTS>
__global__ void __launch_bounds__(kThreads) clip_kernel(const Chunk *table, unsigned long long chunks, const double *parts, unsigned n,
                                                        float *norm, float max_norm, float eps) {
  Chunk next = table[chunks - 1 - blockIdx.x];
  float total;
  if constexpr (PARTS) {
    total = norm_of_parts(parts, n);
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  } else {
    total = *norm;
  }
  const float by = clip_factor(total, max_norm, eps);
  for (unsigned long long k = blockIdx.x; k < chunks; k += gridDim.x) {
    const Chunk c = next;
    next = table[k + gridDim.x < chunks ? chunks - 1 - k - gridDim.x : 0];
    if (by == 1.0f && c.in == c.out) continue;  // nothing to clip
    scale_part<kThreads, kU, kAuxLoadCached>(c, by, 0, kThreads * kU, true);
  }
}

// A wave for every KiB: the addresses that are under way at once stay close together, which a long list's pass is
// faster for (norm and clipping of 1.38 GB: 613 us, with a chunk of 64 KiB a workgroup 672 us; with LDS asked for so
// that fewer waves fit on a CU 647 to 715 us).
constexpr unsigned kTile = 64, kTilesPerChunk = kChunkBytes / 16 / kTile;
template <int AUX>
__global__ void __launch_bounds__(kTile) clip_tile_kernel(const Chunk *table, const float *norm, float max_norm, float eps) {
  // the last chunk first, as above (table: that chunk)
  const Chunk c = table[-(ptrdiff_t)(blockIdx.x / kTilesPerChunk)];
  const unsigned tile = blockIdx.x % kTilesPerChunk;
  const float by = clip_factor(*norm, max_norm, eps);
  if (by == 1.0f && c.in == c.out) return;
  scale_part<kTile, 1, AUX>(c, by, tile * kTile, kTilesPerChunk * kTile, tile == 0);  // one turn
}

// ---- host side ----------------------------------------------------------------

struct Range { uintptr_t at, end; size_t tensor; };

int check_list(const alamd_tensor_list *list) {
  if (!list) return set_error(ALAMD_ERR_INVALID_ARG, "null tensor list");
  int dev = 0;
  ALAMD_HIP(hipGetDevice(&dev));
  if (dev != list->device)
    return set_error(ALAMD_ERR_INVALID_ARG, "the tensor list belongs to device %d, the current device is %d", list->device, dev);
  return ALAMD_OK;
}

// Sorted, with spans that touch or overlap joined.
void join(std::vector<Span> &s) {
  std::sort(s.begin(), s.end(), [](const Span &a, const Span &b) { return a.at < b.at; });
  size_t n = 0;
  for (const Span &x : s) {
    if (n > 0 && x.at <= s[n - 1].end) s[n - 1].end = std::max(s[n - 1].end, x.end);
    else s[n++] = x;
  }
  s.resize(n);
}
int check_apart(const std::vector<Span> &s, const void *p, size_t bytes, const char *name) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  const auto first = std::upper_bound(s.begin(), s.end(), at, [](uintptr_t v, const Span &x) { return v < x.end; });
  if (first != s.end() && first->at < at + bytes) return set_error(ALAMD_ERR_OVERLAP, "%s lies in a tensor of the list", name);
  return ALAMD_OK;
}

int check_clip(const float *norm, float max_norm, float eps) {
  if (!norm || !aligned_to(norm, 4)) return set_error(ALAMD_ERR_INVALID_ARG, "norm is null or not aligned to fp32");
  if (!(max_norm >= 0.0f) || !(eps >= 0.0f)) return set_error(ALAMD_ERR_INVALID_ARG, "max_norm or eps is negative or not a number");
  return ALAMD_OK;
}

// Workgroups of a pass; one that has done its chunk takes the next one that far on.  The norm runs at the rate of a large
// copy with four or two workgroups a CU (847 MB of bf16: 130 us, 6.5 TB/s; eight a CU 136 us); the clipping by chunks
// likes one of them a workgroup.
constexpr size_t kNormGrid = 1024, kClipGrid = (size_t)1 << 16;
static_assert(kNormGrid <= kParts, "the workspace holds a part of every workgroup");

unsigned launch_squares(const alamd_tensor_list *list, bool cached, double *parts, hipStream_t stream) {
  const unsigned grid = (unsigned)(list->chunks < kNormGrid ? list->chunks : kNormGrid);
  if (grid)
    hipLaunchKernelGGL(cached ? squares_kernel<kAuxLoadCached> : squares_kernel<kAuxLoadStream>, dim3(grid), dim3(kThreads), 0, stream,
                       list->table, list->chunks, parts);
  return grid;
}

int launch_norm(const alamd_tensor_list *list, bool cached, float *norm, double *parts, hipStream_t stream) {
  const unsigned n = launch_squares(list, cached, parts, stream);
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, stream, parts, n, norm);
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

// Norm and clipping in one call read a list of up to kCachedBytes through the caches, whose memory-side 256 MiB then
// hold most of it for the second pass; a longer one past them (us, through / past: lists of 30 MiB 17.9 / 21.7,
// 207 MiB 108 / 117, 272 MiB 140 / 150, 1.3 GiB 747 / 687; keeping the last 64 to 224 MiB of that: 682 to 708).
constexpr size_t kCachedBytes = (size_t)288 << 20;
// From kTiledBytes on a list whose chunks are not small is clipped KiB by KiB, with the norm made in a launch of its own
// (us, tiles / chunks: 25 MiB 17.7 / 16.6, 30 MiB 19.2 / 17.8, 35 to 47 MiB the same, 73 MiB 38.1 / 38.4, 136 MiB 70.5 /
// 74.2, 272 MiB 129 / 134, 1.3 GiB 613 / 672).
constexpr size_t kTiledBytes = (size_t)64 << 20;
bool in_tiles(const alamd_tensor_list *list) { return list->bytes >= kTiledBytes && list->bytes / list->chunks >= kChunkBytes / 2; }

// Clips to *norm, or by chunks with `parts` to what those make.
int launch_clip(const alamd_tensor_list *list, bool cached, const double *parts, unsigned n, float *norm, float max_norm, float eps,
                hipStream_t stream) {
  if (!parts && in_tiles(list)) {
    constexpr size_t most = (size_t)1 << 18;  // chunks of a launch: 2^24 workgroups
    auto kern = cached ? clip_tile_kernel<kAuxLoadCached> : clip_tile_kernel<kAuxLoadStream>;
    for (size_t left = list->chunks; left > 0;) {
      const size_t now = left < most ? left : most;
      hipLaunchKernelGGL(kern, dim3((unsigned)now * kTilesPerChunk), dim3(kTile), 0, stream, list->table + left - 1, norm, max_norm, eps);
      left -= now;
    }
  } else if (list->chunks > 0) {
    const unsigned grid = (unsigned)(list->chunks < kClipGrid ? list->chunks : kClipGrid);
    hipLaunchKernelGGL(parts ? clip_kernel<true> : clip_kernel<false>, dim3(grid), dim3(kThreads), 0, stream, list->table,
                       list->chunks, parts, n, norm, max_norm, eps);
  }
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

int check_workspace(const alamd_tensor_list *list, const void *workspace, const float *norm) {
  if (!workspace || !aligned_to(workspace, 8))
    return set_error(ALAMD_ERR_INVALID_ARG, "the workspace is null or not aligned to 8 bytes");
  const uintptr_t w = reinterpret_cast<uintptr_t>(workspace), n = reinterpret_cast<uintptr_t>(norm);
  if (n + sizeof(float) > w && n < w + ALAMD_GLOBAL_NORM_WORKSPACE_BYTES)
    return set_error(ALAMD_ERR_OVERLAP, "the norm lies in the workspace");
  if (int rc = check_apart(list->all, norm, sizeof(float), "the norm")) return rc;
  return check_apart(list->all, workspace, ALAMD_GLOBAL_NORM_WORKSPACE_BYTES, "the workspace");
}

int make_chunks(std::vector<Chunk> &table, std::vector<Span> &taken, std::vector<Span> &all, void *const *outs,
                const void *const *ins, const size_t *counts, const int *dtypes, size_t n) {
  std::vector<Range> written;
  for (size_t t = 0; t < n; ++t) {
    if (dtypes[t] != ALAMD_F16 && dtypes[t] != ALAMD_BF16 && dtypes[t] != ALAMD_F32)
      return set_error(ALAMD_ERR_UNSUPPORTED_TYPE, "tensor %zu: a list takes fp16, bf16 and fp32, not dtype %d", t, dtypes[t]);
    if (counts[t] == 0) continue;
    const size_t es = alamd_dtype_size(dtypes[t]);
    const char *in = static_cast<const char *>(ins[t]);
    char *out = outs ? static_cast<char *>(outs[t]) : const_cast<char *>(in);
    if (!in || !out) return set_error(ALAMD_ERR_INVALID_ARG, "tensor %zu is null", t);
    if (!aligned_to(in, es) || !aligned_to(out, es))
      return set_error(ALAMD_ERR_INVALID_ARG, "tensor %zu is not aligned to its element type", t);
    // more than any device holds: a wrong count is refused before a table of its chunks is built
    if (counts[t] > ((size_t)1 << 39) / es) return set_error(ALAMD_ERR_INVALID_ARG, "tensor %zu is too large", t);
    const uintptr_t at = reinterpret_cast<uintptr_t>(out);
    written.push_back({at, at + counts[t] * es, t});
    // the first chunk ends on a 64-byte boundary of the output (of the input, where they lie apart by no whole
    // number of dwords), so that all others start on one
    const size_t per = kChunkBytes / es, head = head_count(es, out, in, counts[t]);
    for (size_t e = 0; e < counts[t];) {
      const size_t left = counts[t] - e, most = e == 0 && head ? per - 64 / es + head : per;
      const size_t count = left < most ? left : most;
      table.push_back({in + e * es, out + e * es, (unsigned)count, dtypes[t]});
      e += count;
    }
  }
  // what is written is written once, and read by its own tensor alone
  std::sort(written.begin(), written.end(), [](const Range &a, const Range &b) { return a.at < b.at; });
  for (size_t k = 1; k < written.size(); ++k)
    if (written[k].at < written[k - 1].end)
      return set_error(ALAMD_ERR_OVERLAP, "tensors %zu and %zu overlap", written[k - 1].tensor, written[k].tensor);
  for (const Range &r : written) taken.push_back({r.at, r.end});
  join(taken);
  all = taken;
  if (!outs) return ALAMD_OK;
  for (size_t t = 0; t < n; ++t) {
    if (counts[t] == 0) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(ins[t]), end = at + counts[t] * alamd_dtype_size(dtypes[t]);
    auto w = std::upper_bound(written.begin(), written.end(), at, [](uintptr_t v, const Range &r) { return v < r.end; });
    for (; w != written.end() && w->at < end; ++w)
      if (w->tensor != t || w->at != at)
        return set_error(ALAMD_ERR_OVERLAP, "the output of tensor %zu overlaps the input of tensor %zu", w->tensor, t);
    all.push_back({at, end});
  }
  join(all);
  return ALAMD_OK;
}

}  // namespace
}  // namespace alamd

using namespace alamd;

extern "C" {

int alamd_tensor_list_create(alamd_tensor_list **list, void *const *outs, const void *const *ins, const size_t *counts,
                             const int *dtypes, size_t n) {
  if (!list || (n && (!ins || !counts || !dtypes))) return set_error(ALAMD_ERR_INVALID_ARG, "null pointer");
  *list = nullptr;
  try {
    std::vector<Chunk> table;
    std::vector<Span> written, all;
    if (int rc = make_chunks(table, written, all, outs, ins, counts, dtypes, n)) return rc;
    std::unique_ptr<alamd_tensor_list> made(
        new alamd_tensor_list{0, table.size(), 0, nullptr, nullptr, std::move(written), std::move(all)});
    for (const Chunk &c : table) made->bytes += c.count * alamd_dtype_size(c.dtype);
    ALAMD_HIP(hipGetDevice(&made->device));
    // (memory of the list's own, not of an allocator that hands it on in the order of another stream)
    const size_t table_bytes = (table.size() * sizeof(Chunk) + 255) & ~(size_t)255;
    ALAMD_HIP(hipMalloc(reinterpret_cast<void **>(&made->table), table_bytes + ALAMD_GLOBAL_NORM_WORKSPACE_BYTES));
    made->workspace = reinterpret_cast<char *>(made->table) + table_bytes;
    if (!table.empty()) {
      const hipError_t e = hipMemcpy(made->table, table.data(), table.size() * sizeof(Chunk), hipMemcpyHostToDevice);
      if (e != hipSuccess) {
        (void)hipFree(made->table);
        return set_error(ALAMD_ERR_HIP, "hipMemcpy failed: %s", hipGetErrorString(e));
      }
    }
    *list = made.release();
    return ALAMD_OK;
  } catch (...) {  // no C++ exception leaves a C entry
    return set_error(ALAMD_ERR_INVALID_ARG, "no host memory for a list of %zu tensors", n);
  }
}

int alamd_tensor_list_destroy(alamd_tensor_list *list) {
  if (!list) return ALAMD_OK;
  alamd::Chunk *table = list->table;
  delete list;
  if (table) ALAMD_HIP(hipFree(table));
  return ALAMD_OK;
}

void *alamd_tensor_list_workspace(const alamd_tensor_list *list) { return list ? list->workspace : nullptr; }

int alamd_global_norm(const alamd_tensor_list *list, float *norm, void *workspace, void *stream) {
  if (int rc = check_list(list)) return rc;
  if (int rc = check_clip(norm, 0.0f, 0.0f)) return rc;
  if (int rc = check_workspace(list, workspace, norm)) return rc;
  return launch_norm(list, false, norm, static_cast<double *>(workspace), as_stream(stream));
}

int alamd_clip_to_norm(const alamd_tensor_list *list, const float *norm, float max_norm, float eps, void *stream) {
  if (int rc = check_list(list)) return rc;
  if (int rc = check_clip(norm, max_norm, eps)) return rc;
  if (int rc = check_apart(list->written, norm, sizeof(float), "the norm")) return rc;
  return launch_clip(list, false, nullptr, 0, const_cast<float *>(norm), max_norm, eps, as_stream(stream));
}

int alamd_clip_global_norm(const alamd_tensor_list *list, float *norm, float max_norm, float eps, void *workspace,
                           void *stream) {
  if (int rc = check_list(list)) return rc;
  if (int rc = check_clip(norm, max_norm, eps)) return rc;
  if (int rc = check_workspace(list, workspace, norm)) return rc;
  double *parts = static_cast<double *>(workspace);
  const bool cached = list->bytes <= kCachedBytes;
  if (list->chunks == 0 || in_tiles(list)) {
    if (int rc = launch_norm(list, cached, norm, parts, as_stream(stream))) return rc;
    return launch_clip(list, cached, nullptr, 0, norm, max_norm, eps, as_stream(stream));
  }
  const unsigned n = launch_squares(list, cached, parts, as_stream(stream));
  return launch_clip(list, cached, parts, n, norm, max_norm, eps, as_stream(stream));
}

}  // extern "C"
