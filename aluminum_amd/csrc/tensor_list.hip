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

}  // namespace alamd

struct alamd_tensor_list {
  int device;
  size_t chunks;
  alamd::Chunk *table;  // in device memory
};

namespace alamd {
namespace {

constexpr int kThreads = 256;
constexpr size_t kChunkBytes = (size_t)64 << 10;
constexpr size_t kParts = ALAMD_GLOBAL_NORM_WORKSPACE_BYTES / sizeof(double);

// ---- norm -------------------------------------------------------------------

template <typename T> __device__ __forceinline__ double chunk_squares(const Chunk &c) {
  constexpr unsigned VE = Row<T>::VE;
  const unsigned vecs = c.count / VE;
  double a = 0.0;
  for (unsigned i = threadIdx.x; i < vecs; i += kThreads) {
    float x[VE];
    Row<T>::unpack(x, *reinterpret_cast<const u32x4 *>(c.in + (size_t)i * 16));
#pragma unroll
    for (unsigned j = 0; j < VE; ++j) a = fma((double)x[j], (double)x[j], a);
  }
  const unsigned e = vecs * VE + threadIdx.x;
  if (e < c.count) {
    const double x = (double)Row<T>::get(c.in, e);
    a = fma(x, x, a);
  }
  return a;
}

// The sum over the workgroup, in every lane.
template <int THREADS> __device__ __forceinline__ double block_sum(double a) {
  __shared__ double lds[THREADS / 64];
#pragma unroll
  for (int d = 1; d < 64; d *= 2) a += __shfl_xor(a, d);
  if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = a;
  __syncthreads();
  a = lds[0];
#pragma unroll
  for (int k = 1; k < THREADS / 64; ++k) a += lds[k];
  return a;
}

__global__ void __launch_bounds__(kThreads) squares_kernel(const Chunk *table, unsigned long long chunks, double *parts) {
  double a = 0.0;
  for (unsigned long long k = blockIdx.x; k < chunks; k += gridDim.x) {
    const Chunk c = table[k];
    a += c.dtype == ALAMD_F32 ? chunk_squares<float>(c) : c.dtype == ALAMD_BF16 ? chunk_squares<bf16_t>(c) : chunk_squares<f16_t>(c);
  }
  a = block_sum<kThreads>(a);
  if (threadIdx.x == 0) parts[blockIdx.x] = a;
}

__global__ void __launch_bounds__(kThreads) norm_kernel(const double *parts, unsigned n, float *norm) {
  double a = 0.0;
  for (unsigned k = threadIdx.x; k < n; k += kThreads) a += parts[k];
  a = block_sum<kThreads>(a);
  if (threadIdx.x == 0) *norm = (float)sqrt(a);
}

// ---- clipping ---------------------------------------------------------------

template <typename T> __device__ __forceinline__ void chunk_scale(const Chunk &c, float by) {
  constexpr unsigned VE = Row<T>::VE;
  const unsigned vecs = c.count / VE;
  for (unsigned i = threadIdx.x; i < vecs; i += kThreads) {
    float x[VE];
    Row<T>::unpack(x, *reinterpret_cast<const u32x4 *>(c.in + (size_t)i * 16));
#pragma unroll
    for (unsigned j = 0; j < VE; ++j) x[j] *= by;
    *reinterpret_cast<u32x4 *>(c.out + (size_t)i * 16) = Row<T>::pack(x);
  }
  const unsigned e = vecs * VE + threadIdx.x;
  if (e < c.count) Row<T>::put(c.out, e, Row<T>::get(c.in, e) * by);
}

__global__ void __launch_bounds__(kThreads) clip_kernel(const Chunk *table, unsigned long long chunks, const float *norm,
                                                        float max_norm, float eps) {
  const float n = *norm + eps;
  const float by = n <= max_norm ? 1.0f : max_norm / n;
  for (unsigned long long k = blockIdx.x; k < chunks; k += gridDim.x) {
    const Chunk c = table[k];
    if (by == 1.0f && c.in == c.out) continue;  // nothing to clip
    if (c.dtype == ALAMD_F32) chunk_scale<float>(c, by);
    else if (c.dtype == ALAMD_BF16) chunk_scale<bf16_t>(c, by);
    else chunk_scale<f16_t>(c, by);
  }
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

int check_clip(const float *norm, float max_norm, float eps) {
  if (!norm || !aligned_to(norm, 4)) return set_error(ALAMD_ERR_INVALID_ARG, "norm is null or not aligned to fp32");
  if (!(max_norm >= 0.0f) || !(eps >= 0.0f)) return set_error(ALAMD_ERR_INVALID_ARG, "max_norm or eps is negative or not a number");
  return ALAMD_OK;
}

int launch_norm(const alamd_tensor_list *list, float *norm, void *workspace, hipStream_t stream) {
  const unsigned parts = (unsigned)(list->chunks < kParts ? list->chunks : kParts);
  double *sums = static_cast<double *>(workspace);
  if (parts) hipLaunchKernelGGL(squares_kernel, dim3(parts), dim3(kThreads), 0, stream, list->table, list->chunks, sums);
  hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(kThreads), 0, stream, sums, parts, norm);
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

// Workgroups of a clipping launch: a workgroup that has done its chunk takes the next one that far on.
constexpr size_t kMaxClipGrid = (size_t)1 << 20;

int launch_clip(const alamd_tensor_list *list, const float *norm, float max_norm, float eps, hipStream_t stream) {
  if (list->chunks == 0) return ALAMD_OK;
  const unsigned grid = (unsigned)(list->chunks < kMaxClipGrid ? list->chunks : kMaxClipGrid);
  hipLaunchKernelGGL(clip_kernel, dim3(grid), dim3(kThreads), 0, stream, list->table, list->chunks, norm, max_norm, eps);
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

int check_workspace(const void *workspace) {
  if (!workspace || !aligned_to(workspace, 8))
    return set_error(ALAMD_ERR_INVALID_ARG, "the workspace is null or not aligned to 8 bytes");
  return ALAMD_OK;
}

int make_chunks(std::vector<Chunk> &table, void *const *outs, const void *const *ins, const size_t *counts, const int *dtypes,
                size_t n) {
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
    if (counts[t] > ((size_t)1 << 46) / es) return set_error(ALAMD_ERR_INVALID_ARG, "tensor %zu is too large", t);
    const uintptr_t at = reinterpret_cast<uintptr_t>(out);
    written.push_back({at, at + counts[t] * es, t});
    const size_t per = kChunkBytes / es;
    for (size_t e = 0; e < counts[t]; e += per) {
      const size_t left = counts[t] - e;
      table.push_back({in + e * es, out + e * es, (unsigned)(left < per ? left : per), dtypes[t]});
    }
  }
  // what is written is written once, and read by its own tensor alone
  std::sort(written.begin(), written.end(), [](const Range &a, const Range &b) { return a.at < b.at; });
  for (size_t k = 1; k < written.size(); ++k)
    if (written[k].at < written[k - 1].end)
      return set_error(ALAMD_ERR_OVERLAP, "tensors %zu and %zu overlap", written[k - 1].tensor, written[k].tensor);
  if (!outs) return ALAMD_OK;
  for (size_t t = 0; t < n; ++t) {
    if (counts[t] == 0) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(ins[t]), end = at + counts[t] * alamd_dtype_size(dtypes[t]);
    auto w = std::upper_bound(written.begin(), written.end(), at, [](uintptr_t v, const Range &r) { return v < r.end; });
    for (; w != written.end() && w->at < end; ++w)
      if (w->tensor != t || w->at != at)
        return set_error(ALAMD_ERR_OVERLAP, "the output of tensor %zu overlaps the input of tensor %zu", w->tensor, t);
  }
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
    if (int rc = make_chunks(table, outs, ins, counts, dtypes, n)) return rc;
    std::unique_ptr<alamd_tensor_list> made(new alamd_tensor_list{0, table.size(), nullptr});
    ALAMD_HIP(hipGetDevice(&made->device));
    if (!table.empty()) {
      ALAMD_HIP(hipMalloc(reinterpret_cast<void **>(&made->table), table.size() * sizeof(Chunk)));
      const hipError_t e = hipMemcpy(made->table, table.data(), table.size() * sizeof(Chunk), hipMemcpyHostToDevice);
      if (e != hipSuccess) {
        (void)hipFree(made->table);
        return set_error(ALAMD_ERR_HIP, "hipMemcpy failed: %s", hipGetErrorString(e));
      }
    }
    *list = made.release();
    return ALAMD_OK;
  } catch (const std::bad_alloc &) {
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

int alamd_global_norm(const alamd_tensor_list *list, float *norm, void *workspace, void *stream) {
  if (int rc = check_list(list)) return rc;
  if (int rc = check_clip(norm, 0.0f, 0.0f)) return rc;
  if (int rc = check_workspace(workspace)) return rc;
  return launch_norm(list, norm, workspace, as_stream(stream));
}

int alamd_clip_to_norm(const alamd_tensor_list *list, const float *norm, float max_norm, float eps, void *stream) {
  if (int rc = check_list(list)) return rc;
  if (int rc = check_clip(norm, max_norm, eps)) return rc;
  return launch_clip(list, norm, max_norm, eps, as_stream(stream));
}

int alamd_clip_global_norm(const alamd_tensor_list *list, float *norm, float max_norm, float eps, void *workspace,
                           void *stream) {
  if (int rc = check_list(list)) return rc;
  if (int rc = check_clip(norm, max_norm, eps)) return rc;
  if (int rc = check_workspace(workspace)) return rc;
  if (int rc = launch_norm(list, norm, workspace, as_stream(stream))) return rc;
  return launch_clip(list, norm, max_norm, eps, as_stream(stream));
}

}  // extern "C"
