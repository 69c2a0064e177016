// Root-mean-square norm of the sum of P rank contributions and a residual, with its backward pass: what a
// layer split over ranks does with the result of its Allreduce, in the pass that folds it.
//
// Forward, per row of n = cols elements:
//   s    = x_0 + x_1 + .. + x_{P-1} (+ residual)     fp32, in that order
//   rstd = 1 / sqrt(sum(s^2) / n + eps)
//   y    = (s * w) * rstd
// y is rounded once, from the unrounded s; the `sum` that is written back for the next layer is s rounded.
// (s * w) * rstd instead of (s * rstd) * w: rounding is monotone, so max|y| = max|s * w| * rstd to the last
// bit, and the scale of a whole 8-bit row needs no second trip round the row.
//
// Backward, from the saved sum x and rstd, with dy = dy_0 + .. + dy_{P-1}, n_hat = x * rstd, g = dy * w:
//   dx = rstd * (g - n_hat * sum(g * n_hat) / n) (+ dsum),   dw = sum over rows of dy * n_hat
//
// A team of TEAM lanes holds a row in registers: NV 128-bit vectors per lane and stream, read once.  The
// elements behind the last whole vector belong to the next lane, whose vector is moved back so that it ends with
// the row: its first elements are another lane's as well, computed to the same bits, left out of every sum
// and stored twice.  Lanes without a vector read zeros and store nothing (the buffer descriptor's bound).
#include "alamd_rows.h"

namespace alamd {

namespace {

constexpr unsigned kMaxCols = ALAMD_RMS_NORM_MAX_COLS;

// ---- forward ----------------------------------------------------------------

struct NormParams {
  const char *in[ALAMD_MAX_RANKS];
  const char *res, *weight;
  char *sum, *out;
  float *rstd, *scales;
  unsigned long long in_pitch, res_pitch, out_pitch;  // bytes between rows
  unsigned long long rows;
  unsigned cols;
  int P;
  int w32;          // the weight is fp32 whatever the type of the rows
  unsigned group_log2, groups;  // columns of an 8-bit group, groups of a row
  float eps, inv_n;
};

enum { OUT_SAME = 0, OUT_E4M3_ROW = 1, OUT_E4M3_GROUP = 2 };

// The largest value e4m3 holds; the scale of a group whose largest |y| is a is max(a / 448, 2^-126), so that
// its reciprocal is finite whatever a is.
constexpr float kE4m3Max = 448.0f, kLeastScale = 1.17549435e-38f;
__device__ __forceinline__ float scale_of(unsigned amax_bits) {
  const float a = __uint_as_float(amax_bits) * (1.0f / kE4m3Max);
  return a < kLeastScale ? kLeastScale : a;  // a NaN passes
}

// Streams whose loads are issued together: eight vectors a lane.
template <int NV> constexpr int streams_at_once() { return NV >= 8 ? 1 : 8 / NV > 4 ? 4 : 8 / NV; }

// The sum of P streams of a row, in rank order.
template <int B, typename Team, typename T, int NV, int VE>
__device__ __forceinline__ void sum_streams(float (&s)[NV][VE], const Team &team, const char *const *in, int P,
                                            unsigned long long pitch, unsigned long long row, bool live) {
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < VE; ++j) s[v][j] = -0.0f;  // -0 + x is x, whatever x
  for (int k = 0; k < P; k += B) {
    u32x4 raw[B][NV];
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (k + b < P) team.load(raw[b], in[k + b], pitch, row, live);
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (k + b < P) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float x[VE];
          Row<T>::unpack(x, raw[b][v]);
#pragma unroll
          for (int j = 0; j < VE; ++j) s[v][j] += x[j];
        }
      }
  }
}

constexpr int kWaveTeams = 4;  // rows, one a wave, of a workgroup whose teams are waves

template <typename T, int TEAM, int NV, int OUT>
__global__ void __launch_bounds__(TEAM ? 64 * kWaveTeams : 1024) rms_norm_kernel(const NormParams p) {
  constexpr int VE = Row<T>::VE;
  constexpr int TEAMS = TEAM ? kWaveTeams : 1;
  __shared__ float lds[2][kWaves * 2];
  const RowTeam<T, TEAM, NV> team(p.cols);
  int turn = 0;
  for (unsigned long long r0 = (unsigned long long)blockIdx.x * TEAMS; r0 < p.rows;
       r0 += (unsigned long long)gridDim.x * TEAMS, turn ^= 1) {
    const unsigned long long row = r0 + team.index;
    const bool live = row < p.rows;
    u32x4 res[NV];
    if (p.res) team.load(res, p.res, p.res_pitch, row, live);
    float s[NV][VE];
    sum_streams<streams_at_once<NV>(), RowTeam<T, TEAM, NV>, T>(s, team, p.in, p.P, p.in_pitch, row, live);
    if (p.res) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x[VE];
        Row<T>::unpack(x, res[v]);
#pragma unroll
        for (int j = 0; j < VE; ++j) s[v][j] += x[j];
      }
    }
    float ss = 0.0f;
    if (team.ragged) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < VE; ++j) ss = fmaf(s[v][j], team.counts(v, j) ? s[v][j] : 0.0f, ss);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < VE; ++j) ss = fmaf(s[v][j], s[v][j], ss);
    }
    u32x4 sum[NV];
    if (p.sum) {
#pragma unroll
      for (int v = 0; v < NV; ++v) sum[v] = Row<T>::pack(s[v]);
    }
    if (p.weight) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float w[VE];
        team.load_weight(w, v, p.weight, p.w32);
#pragma unroll
        for (int j = 0; j < VE; ++j) s[v][j] *= w[j];
      }
    }
    // the largest |s * w| as bits: a NaN is above every number
    unsigned am = 0;
    if constexpr (OUT == OUT_E4M3_ROW) {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int j = 0; j < VE; ++j) am = umax(am, __float_as_uint(s[v][j]) & 0x7fffffffu);
      team_sum_max<TEAM>(ss, am, lds[turn]);
    } else {
      ss = team_sum<TEAM>(ss, lds[turn]);
    }
    // The team has met: every lane has read its part of the row.  Nothing is written before, because a vector
    // that was moved back reads what another lane writes where the sum takes the residual's place.
    if (p.sum) team.store(sum, p.sum, p.res_pitch, row, live);
    const float rstd = rsqrtf(fmaf(ss, p.inv_n, p.eps));
    if (p.rstd && live && team.lane == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; ++j) s[v][j] *= rstd;
    if constexpr (OUT == OUT_SAME) {
#pragma unroll
      for (int v = 0; v < NV; ++v) sum[v] = Row<T>::pack(s[v]);
      team.store(sum, p.out, p.out_pitch, row, live);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float scale;
        if constexpr (OUT == OUT_E4M3_ROW) {
          scale = scale_of(__float_as_uint(__uint_as_float(am) * rstd) & 0x7fffffffu);
          if (v == 0 && live && team.lane == 0) p.scales[row] = scale;
        } else {
          unsigned a = 0;
#pragma unroll
          for (int j = 0; j < VE; ++j) a = umax(a, team.counts(v, j) ? __float_as_uint(s[v][j]) & 0x7fffffffu : 0u);
          a = group_max(a, (1u << p.group_log2) / VE);
          scale = scale_of(a);
          const unsigned e = team.element(v);
          if (live && e < p.cols && (e & ((1u << p.group_log2) - 1)) == 0)
            p.scales[row * p.groups + (e >> p.group_log2)] = scale;
        }
        team.store_e4m3(s[v], v, __builtin_amdgcn_rcpf(scale), p.out, p.out_pitch, row, live);
      }
    }
  }
}

// Rows shorter than a vector: one lane walks a row.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) rms_norm_short_kernel(const NormParams p) {
  for (unsigned long long row = (unsigned long long)blockIdx.x * 256 + threadIdx.x; row < p.rows;
       row += (unsigned long long)gridDim.x * 256) {
    float s[8], ss = 0.0f;
    unsigned am = 0;
    for (unsigned c = 0; c < p.cols; ++c) {
      float x = 0.0f;
      for (int k = 0; k < p.P; ++k) {
        const float t = Row<T>::get(p.in[k] + row * p.in_pitch, c);
        x = k == 0 ? t : x + t;
      }
      if (p.res) x += Row<T>::get(p.res + row * p.res_pitch, c);
      s[c] = x;
      ss = fmaf(x, x, ss);
    }
    const float rstd = rsqrtf(fmaf(ss, p.inv_n, p.eps));
    if (p.rstd) p.rstd[row] = rstd;
    for (unsigned c = 0; c < p.cols; ++c) {
      if (p.sum) Row<T>::put(p.sum + row * p.res_pitch, c, s[c]);
      const float w = !p.weight ? 1.0f : p.w32 ? Row<float>::get(p.weight, c) : Row<T>::get(p.weight, c);
      s[c] = s[c] * w * rstd;
      const unsigned b = __float_as_uint(s[c]) & 0x7fffffffu;
      am = b > am ? b : am;
    }
    if constexpr (E4M3) {
      const float scale = scale_of(am), by = 1.0f / scale;
      p.scales[row] = scale;
      for (unsigned c = 0; c < p.cols; ++c)
        p.out[row * p.out_pitch + c] = (char)(__builtin_amdgcn_cvt_pk_fp8_f32(s[c] * by, 0.0f, 0, false) & 0xff);
    } else {
      for (unsigned c = 0; c < p.cols; ++c) Row<T>::put(p.out + row * p.out_pitch, c, s[c]);
    }
  }
}

// ---- backward ---------------------------------------------------------------

struct GradParams {
  const char *dy[ALAMD_MAX_RANKS];
  const char *x, *dsum, *weight;
  char *dx;
  const float *rstd;
  float *partial;  // [workgroups][cols]: the weight's gradient from each workgroup's rows
  unsigned long long dy_pitch, x_pitch, dsum_pitch, dx_pitch;
  unsigned long long rows;
  unsigned cols;
  int P;
  int w32;
  float inv_n;
};

template <typename T, int TEAM, int NV>
__global__ void __launch_bounds__(TEAM ? 64 * kWaveTeams : 1024) rms_norm_grad_kernel(const GradParams p) {
  constexpr int VE = Row<T>::VE;
  constexpr int TEAMS = TEAM ? kWaveTeams : 1;
  __shared__ float lds[2][kWaves];
  const RowTeam<T, TEAM, NV> team(p.cols);
  float dw[NV][VE];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < VE; ++j) dw[v][j] = 0.0f;
  int turn = 0;
  for (unsigned long long r0 = (unsigned long long)blockIdx.x * TEAMS; r0 < p.rows;
       r0 += (unsigned long long)gridDim.x * TEAMS, turn ^= 1) {
    const unsigned long long row = r0 + team.index;
    const bool live = row < p.rows;
    u32x4 xr[NV], ds[NV];
    team.load(xr, p.x, p.x_pitch, row, live);
    if (p.dsum) team.load(ds, p.dsum, p.dsum_pitch, row, live);
    const float rstd = live ? p.rstd[row] : 0.0f;
    float g[NV][VE];
    sum_streams<streams_at_once<NV>(), RowTeam<T, TEAM, NV>, T>(g, team, p.dy, p.P, p.dy_pitch, row, live);
    float dot = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float x[VE], w[VE];
      Row<T>::unpack(x, xr[v]);
      if (p.weight) team.load_weight(w, v, p.weight, p.w32);
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float n = x[j] * rstd;
        // a row that is not there has rstd = 0 and reads zeros
        dw[v][j] = fmaf(g[v][j], n, dw[v][j]);
        if (p.weight) g[v][j] *= w[j];
        dot = fmaf(g[v][j], team.counts(v, j) ? n : 0.0f, dot);
      }
    }
    if (p.dx) {
      const float c = team_sum<TEAM>(dot, lds[turn]) * p.inv_n;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float x[VE];
        Row<T>::unpack(x, xr[v]);
#pragma unroll
        for (int j = 0; j < VE; ++j) g[v][j] = rstd * fmaf(-(x[j] * rstd), c, g[v][j]);
      }
      // (dsum was read before the team met: dx may take its place)
      if (p.dsum) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float d[VE];
          Row<T>::unpack(d, ds[v]);
#pragma unroll
          for (int j = 0; j < VE; ++j) g[v][j] += d[j];
        }
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) ds[v] = Row<T>::pack(g[v]);
      team.store(ds, p.dx, p.dx_pitch, row, live);
    }
  }
  if (!p.partial) return;
  float *dst = p.partial + (size_t)blockIdx.x * p.cols;
  if constexpr (TEAMS == 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v) team.store_f32(dw[v], v, dst);
  } else {
    // the teams of the workgroup one after another, in their order
    __shared__ float part[TEAM * NV * VE];
    for (int t = 0; t < TEAMS; ++t) {
      if ((int)team.index == t) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            float &a = part[(v * VE + j) * TEAM + team.lane];
            dw[v][j] = t == 0 ? dw[v][j] : a + dw[v][j];
            a = dw[v][j];
          }
        if (t == TEAMS - 1)
#pragma unroll
          for (int v = 0; v < NV; ++v) team.store_f32(dw[v], v, dst);
      }
      __syncthreads();
    }
  }
}

template <typename T> __global__ void __launch_bounds__(256) rms_norm_grad_short_kernel(const GradParams p) {
  __shared__ float part[256][8];
  float dw[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (unsigned long long row = (unsigned long long)blockIdx.x * 256 + threadIdx.x; row < p.rows;
       row += (unsigned long long)gridDim.x * 256) {
    const float rstd = p.rstd[row];
    float g[8], n[8], dot = 0.0f;
    for (unsigned c = 0; c < p.cols; ++c) {
      float d = 0.0f;
      for (int k = 0; k < p.P; ++k) {
        const float t = Row<T>::get(p.dy[k] + row * p.dy_pitch, c);
        d = k == 0 ? t : d + t;
      }
      n[c] = Row<T>::get(p.x + row * p.x_pitch, c) * rstd;
      dw[c] = fmaf(d, n[c], dw[c]);
      const float w = !p.weight ? 1.0f : p.w32 ? Row<float>::get(p.weight, c) : Row<T>::get(p.weight, c);
      g[c] = d * w;
      dot = fmaf(g[c], n[c], dot);
    }
    if (!p.dx) continue;
    dot *= p.inv_n;
    for (unsigned c = 0; c < p.cols; ++c) {
      float d = rstd * fmaf(-n[c], dot, g[c]);
      if (p.dsum) d += Row<T>::get(p.dsum + row * p.dsum_pitch, c);
      Row<T>::put(p.dx + row * p.dx_pitch, c, d);
    }
  }
  if (!p.partial) return;
  for (int c = 0; c < 8; ++c) part[threadIdx.x][c] = dw[c];
  __syncthreads();
  if (threadIdx.x < p.cols) {
    float a = 0.0f;
    for (int t = 0; t < 256; ++t) a += part[t][threadIdx.x];
    p.partial[(size_t)blockIdx.x * p.cols + threadIdx.x] = a;
  }
}

// The workgroups' partial sums joined, column by column, in the order of the workgroups: 32 columns x 32
// slices of the workgroups per workgroup, then the slices.
template <typename W>
__global__ void __launch_bounds__(1024) rms_norm_dweight_kernel(char *dw, const float *partial, unsigned parts, unsigned cols) {
  __shared__ float lds[32][33];
  const unsigned c = threadIdx.x & 31u, slice = threadIdx.x >> 5, col = blockIdx.x * 32u + c;
  float a = 0.0f;
  if (col < cols) {
    const unsigned per = (parts + 31u) / 32u;
    const unsigned from = slice * per, to = from + per < parts ? from + per : parts;
    for (unsigned k = from; k < to; ++k) a += partial[(size_t)k * cols + col];
  }
  lds[slice][c] = a;
  __syncthreads();
  if (slice == 0 && col < cols) {
    for (int k = 1; k < 32; ++k) a += lds[k][c];
    Row<W>::put(dw, col, a);
  }
}

// ---- host side ----------------------------------------------------------------

// A matrix of the call: a name for messages, the first row, bytes between rows and of a row.
struct Matrix {
  const char *name;
  const void *p;
  size_t pitch, bytes;
  bool written;
};

// Whether two matrices of `rows` rows share memory: by their ranges, or, where rows of the same pitch
// interleave, by the columns they occupy.
bool share_memory(const Matrix &a, const Matrix &b, size_t rows) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.p), pb = reinterpret_cast<uintptr_t>(b.p);
  const size_t la = (rows - 1) * a.pitch + a.bytes, lb = (rows - 1) * b.pitch + b.bytes;
  if (pa + la <= pb || pb + lb <= pa) return false;
  if (a.pitch != b.pitch || rows == 1 || a.pitch == 0) return true;
  const bool a_first = pa <= pb;
  const size_t d = (a_first ? pb - pa : pa - pb) % a.pitch;
  return !(d >= (a_first ? a.bytes : b.bytes) && d + (a_first ? b.bytes : a.bytes) <= a.pitch);
}

int check_matrix(const void *p, const char *name, size_t stride, size_t rows, size_t cols, size_t es) {
  if (!p) return set_error(ALAMD_ERR_INVALID_ARG, "%s is null", name);
  if (!aligned_to(p, es)) return set_error(ALAMD_ERR_INVALID_ARG, "%s is not aligned to its element type", name);
  if (rows > 1 && stride < cols)
    return set_error(ALAMD_ERR_INVALID_ARG, "rows of %s are %zu elements long and %zu apart", name, cols, stride);
  if (stride > ((size_t)1 << 46) / es || (rows > 1 && rows - 1 > ((size_t)1 << 46) / (stride * es)))
    return set_error(ALAMD_ERR_INVALID_ARG, "%s is too large", name);
  return ALAMD_OK;
}

// Every written matrix against every other one; `same` allows a written matrix to be exactly a read one.
int check_overlaps(const Matrix *m, int n, size_t rows) {
  for (int a = 0; a < n; ++a) {
    if (!m[a].written || !m[a].p) continue;
    for (int b = 0; b < n; ++b) {
      if (b == a || !m[b].p || (m[b].written && b < a)) continue;
      if (!m[b].written && m[a].p == m[b].p && (m[a].pitch == m[b].pitch || rows == 1) && m[a].bytes == m[b].bytes) continue;
      if (share_memory(m[a], m[b], rows)) return set_error(ALAMD_ERR_OVERLAP, "%s overlaps %s", m[a].name, m[b].name);
    }
  }
  return ALAMD_OK;
}

int check_common(int P, size_t cols, int dtype, const void *weight, int weight_dtype, size_t *es, size_t *wes) {
  if (P < 1 || P > ALAMD_MAX_RANKS)
    return set_error(ALAMD_ERR_INVALID_ARG, "number of ranks %d outside [1, %d]", P, ALAMD_MAX_RANKS);
  if (dtype != ALAMD_F16 && dtype != ALAMD_BF16 && dtype != ALAMD_F32)
    return set_error(ALAMD_ERR_UNSUPPORTED_TYPE, "a norm takes fp16, bf16 or fp32 rows, not dtype %d", dtype);
  if (weight && weight_dtype != dtype && weight_dtype != ALAMD_F32)
    return set_error(ALAMD_ERR_UNSUPPORTED_TYPE, "the weight has the rows' type or fp32, not dtype %d", weight_dtype);
  if (cols > kMaxCols) return set_error(ALAMD_ERR_INVALID_ARG, "%zu columns, at most %u are taken", cols, kMaxCols);
  *es = alamd_dtype_size(dtype);
  *wes = alamd_dtype_size(weight ? weight_dtype : dtype);
  if (weight && !aligned_to(weight, *wes)) return set_error(ALAMD_ERR_INVALID_ARG, "weight is not aligned to its element type");
  return ALAMD_OK;
}

// Rows a launch has workgroups for; a workgroup that has done its row takes the next one that far on.
constexpr size_t kMaxGrid = (size_t)1 << 21;

template <typename T, int TEAM, int NV>
int launch_norm(const NormParams &p, int out, unsigned threads, hipStream_t stream) {
  constexpr size_t TEAMS = TEAM ? kWaveTeams : 1;
  size_t grid = (p.rows + TEAMS - 1) / TEAMS;
  if (grid > kMaxGrid) grid = kMaxGrid;
  auto kern = out == OUT_SAME ? rms_norm_kernel<T, TEAM, NV, OUT_SAME>
              : out == OUT_E4M3_ROW ? rms_norm_kernel<T, TEAM, NV, OUT_E4M3_ROW> : rms_norm_kernel<T, TEAM, NV, OUT_E4M3_GROUP>;
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(threads), 0, stream, p);
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

// Threads of a workgroup that holds a row of `need` vectors, nv of them a lane.
inline unsigned row_threads(unsigned need, unsigned nv) { return ((need + nv - 1) / nv + 63u) & ~63u; }

template <typename T> int norm_rows(const NormParams &p, int out, hipStream_t stream) {
  constexpr unsigned VE = Row<T>::VE;
  if (p.cols < VE) {
    size_t grid = (p.rows + 255) / 256;
    if (grid > kMaxGrid) grid = kMaxGrid;
    hipLaunchKernelGGL(out == OUT_SAME ? (rms_norm_short_kernel<T, false>) : (rms_norm_short_kernel<T, true>), dim3((unsigned)grid),
                       dim3(256), 0, stream, p);
    ALAMD_HIP(hipGetLastError());
    return ALAMD_OK;
  }
  const unsigned need = (p.cols + VE - 1) / VE;  // vectors of a row
  if (need <= 64) return launch_norm<T, 64, 1>(p, out, 64 * kWaveTeams, stream);
  if (need <= 128) return launch_norm<T, 64, 2>(p, out, 64 * kWaveTeams, stream);
  if (need <= 2048) return launch_norm<T, 0, 2>(p, out, row_threads(need, 2), stream);
  if (need <= 4096) return launch_norm<T, 0, 4>(p, out, row_threads(need, 4), stream);
  if constexpr (VE == 4) return launch_norm<T, 0, 8>(p, out, row_threads(need, 8), stream);
  return set_error(ALAMD_ERR_INVALID_ARG, "too many columns");
}

// Workgroups whose partial sums of the weight's gradient are kept.
constexpr size_t kGradParts = 512;

template <typename T, int TEAM, int NV>
int launch_grad(const GradParams &p, size_t *parts, unsigned threads, hipStream_t stream) {
  constexpr size_t TEAMS = TEAM ? kWaveTeams : 1;
  size_t grid = (p.rows + TEAMS - 1) / TEAMS;
  if (grid > kGradParts) grid = kGradParts;
  *parts = grid;
  hipLaunchKernelGGL((rms_norm_grad_kernel<T, TEAM, NV>), dim3((unsigned)grid), dim3(threads), 0, stream, p);
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

template <typename T> int grad_rows(const GradParams &p, size_t *parts, hipStream_t stream) {
  constexpr unsigned VE = Row<T>::VE;
  if (p.cols < VE) {
    size_t grid = (p.rows + 255) / 256;
    if (grid > kGradParts) grid = kGradParts;
    *parts = grid;
    hipLaunchKernelGGL(rms_norm_grad_short_kernel<T>, dim3((unsigned)grid), dim3(256), 0, stream, p);
    ALAMD_HIP(hipGetLastError());
    return ALAMD_OK;
  }
  const unsigned need = (p.cols + VE - 1) / VE;
  if (need <= 64) return launch_grad<T, 64, 1>(p, parts, 64 * kWaveTeams, stream);
  if (need <= 128) return launch_grad<T, 64, 2>(p, parts, 64 * kWaveTeams, stream);
  if (need <= 2048) return launch_grad<T, 0, 2>(p, parts, row_threads(need, 2), stream);
  if (need <= 4096) return launch_grad<T, 0, 4>(p, parts, row_threads(need, 4), stream);
  if constexpr (VE == 4) return launch_grad<T, 0, 8>(p, parts, row_threads(need, 8), stream);
  return set_error(ALAMD_ERR_INVALID_ARG, "too many columns");
}

}  // namespace
}  // namespace alamd

using namespace alamd;

extern "C" {

int alamd_rms_norm(void *out, size_t out_stride, void *sum, const void *residual, size_t residual_stride,
                   const void *const *ins, int P, size_t in_stride, const void *weight, int weight_dtype, float *rstd,
                   float *scales, size_t group, size_t rows, size_t cols, int dtype, float eps, void *stream) {
  size_t es, wes;
  if (int rc = check_common(P, cols, dtype, weight, weight_dtype, &es, &wes)) return rc;
  if (group != 0 && group != 32 && group != 64 && group != 128)
    return set_error(ALAMD_ERR_INVALID_ARG, "an 8-bit group has 32, 64 or 128 columns, or 0 for the whole row, not %zu", group);
  if (group != 0 && !scales) return set_error(ALAMD_ERR_INVALID_ARG, "a group size, but no scales");
  if (!(eps >= 0.0f)) return set_error(ALAMD_ERR_INVALID_ARG, "eps is negative or not a number");
  if (rows == 0 || cols == 0) return ALAMD_OK;
  if (!ins) return set_error(ALAMD_ERR_INVALID_ARG, "null pointer");
  const size_t oes = scales ? 1 : es;
  Matrix m[ALAMD_MAX_RANKS + 7];
  int n = 0, rc;
  for (int k = 0; k < P; ++k) {
    if ((rc = check_matrix(ins[k], "a rank's input", in_stride, rows, cols, es))) return rc;
    m[n++] = {"a rank's input", ins[k], in_stride * es, cols * es, false};
  }
  if (residual && (rc = check_matrix(residual, "the residual", residual_stride, rows, cols, es))) return rc;
  if (sum && (rc = check_matrix(sum, "the sum", residual_stride, rows, cols, es))) return rc;
  if ((rc = check_matrix(out, "the output", out_stride, rows, cols, oes))) return rc;
  if ((rstd && !aligned_to(rstd, 4)) || (scales && !aligned_to(scales, 4)))
    return set_error(ALAMD_ERR_INVALID_ARG, "rstd or scales not aligned to fp32");
  const size_t groups = scales && group ? (cols + group - 1) / group : 1;
  m[n++] = {"the residual", residual, residual_stride * es, cols * es, false};
  m[n++] = {"the weight", weight, 0, cols * wes, false};
  m[n++] = {"the sum", sum, residual_stride * es, cols * es, true};
  m[n++] = {"the output", out, out_stride * oes, cols * oes, true};
  m[n++] = {"rstd", rstd, 4, 4, true};
  m[n++] = {"the scales", scales, groups * 4, groups * 4, true};
  if ((rc = check_overlaps(m, n, rows))) return rc;
  NormParams p{};
  for (int k = 0; k < P; ++k) p.in[k] = static_cast<const char *>(ins[k]);
  p.res = static_cast<const char *>(residual);
  p.weight = static_cast<const char *>(weight);
  p.sum = static_cast<char *>(sum);
  p.out = static_cast<char *>(out);
  p.rstd = rstd;
  p.scales = scales;
  p.in_pitch = in_stride * es;
  p.res_pitch = residual_stride * es;
  p.out_pitch = out_stride * oes;
  p.rows = rows;
  p.cols = (unsigned)cols;
  p.P = P;
  p.w32 = weight && weight_dtype == ALAMD_F32;
  while (group >> p.group_log2 > 1) ++p.group_log2;
  p.groups = (unsigned)groups;
  p.eps = eps;
  p.inv_n = 1.0f / (float)cols;
  const int kind = !scales ? OUT_SAME : group == 0 || group >= cols ? OUT_E4M3_ROW : OUT_E4M3_GROUP;
  switch (dtype) {
  case ALAMD_F16: return norm_rows<f16_t>(p, kind, as_stream(stream));
  case ALAMD_BF16: return norm_rows<bf16_t>(p, kind, as_stream(stream));
  default: return norm_rows<float>(p, kind, as_stream(stream));
  }
}

size_t alamd_rms_norm_grad_workspace(size_t rows, size_t cols) {
  return (rows < kGradParts ? rows : kGradParts) * (cols < kMaxCols ? cols : kMaxCols) * sizeof(float);
}

int alamd_rms_norm_grad(void *dx, size_t dx_stride, const void *const *dys, int P, size_t dy_stride, const void *x,
                        size_t x_stride, const void *dsum, size_t dsum_stride, const float *rstd, const void *weight,
                        int weight_dtype, void *dweight, size_t rows, size_t cols, int dtype, void *workspace,
                        void *stream) {
  size_t es, wes;
  if (int rc = check_common(P, cols, dtype, weight ? weight : dweight, weight_dtype, &es, &wes)) return rc;
  if (!dx && !dweight) return set_error(ALAMD_ERR_INVALID_ARG, "neither dx nor dweight is wanted");
  if (dsum && !dx) return set_error(ALAMD_ERR_INVALID_ARG, "dsum without dx");
  if (cols == 0 || (rows == 0 && !dweight)) return ALAMD_OK;
  if (dweight && !aligned_to(dweight, wes)) return set_error(ALAMD_ERR_INVALID_ARG, "dweight is not aligned to its element type");
  size_t parts = 0;
  if (rows > 0) {
    if (!dys) return set_error(ALAMD_ERR_INVALID_ARG, "null pointer");
    Matrix m[ALAMD_MAX_RANKS + 8];
    int n = 0, rc;
    for (int k = 0; k < P; ++k) {
      if ((rc = check_matrix(dys[k], "a rank's gradient", dy_stride, rows, cols, es))) return rc;
      m[n++] = {"a rank's gradient", dys[k], dy_stride * es, cols * es, false};
    }
    if ((rc = check_matrix(x, "x", x_stride, rows, cols, es))) return rc;
    if (dsum && (rc = check_matrix(dsum, "dsum", dsum_stride, rows, cols, es))) return rc;
    if (dx && (rc = check_matrix(dx, "dx", dx_stride, rows, cols, es))) return rc;
    if (!rstd || !aligned_to(rstd, 4)) return set_error(ALAMD_ERR_INVALID_ARG, "rstd is null or not aligned to fp32");
    if (dweight && (!workspace || !aligned_to(workspace, 4)))
      return set_error(ALAMD_ERR_INVALID_ARG, "dweight needs a workspace aligned to fp32 (alamd_rms_norm_grad_workspace)");
    m[n++] = {"x", x, x_stride * es, cols * es, false};
    m[n++] = {"dsum", dsum, dsum_stride * es, cols * es, false};
    m[n++] = {"rstd", rstd, 4, 4, false};
    m[n++] = {"the weight", weight, 0, cols * wes, false};
    m[n++] = {"dx", dx, dx_stride * es, cols * es, true};
    m[n++] = {"dweight", dweight, 0, cols * wes, true};
    if (dweight) {
      // the workspace has rows of its own: as one stretch of bytes
      const size_t bytes = alamd_rms_norm_grad_workspace(rows, cols);
      m[n++] = {"the workspace", workspace, 0, bytes, true};
    }
    if ((rc = check_overlaps(m, n, rows))) return rc;
    GradParams p{};
    for (int k = 0; k < P; ++k) p.dy[k] = static_cast<const char *>(dys[k]);
    p.x = static_cast<const char *>(x);
    p.dsum = static_cast<const char *>(dsum);
    p.weight = static_cast<const char *>(weight);
    p.dx = static_cast<char *>(dx);
    p.rstd = rstd;
    p.partial = dweight ? static_cast<float *>(workspace) : nullptr;
    p.dy_pitch = dy_stride * es;
    p.x_pitch = x_stride * es;
    p.dsum_pitch = dsum_stride * es;
    p.dx_pitch = dx_stride * es;
    p.rows = rows;
    p.cols = (unsigned)cols;
    p.P = P;
    p.w32 = weight && weight_dtype == ALAMD_F32;
    p.inv_n = 1.0f / (float)cols;
    switch (dtype) {
    case ALAMD_F16: rc = grad_rows<f16_t>(p, &parts, as_stream(stream)); break;
    case ALAMD_BF16: rc = grad_rows<bf16_t>(p, &parts, as_stream(stream)); break;
    default: rc = grad_rows<float>(p, &parts, as_stream(stream)); break;
    }
    if (rc) return rc;
  }
  if (!dweight) return ALAMD_OK;
  const dim3 grid((unsigned)((cols + 31) / 32));
  const float *partial = static_cast<const float *>(workspace);
  switch (weight_dtype) {
  case ALAMD_F16: hipLaunchKernelGGL(rms_norm_dweight_kernel<f16_t>, grid, dim3(1024), 0, as_stream(stream), (char *)dweight, partial, (unsigned)parts, (unsigned)cols); break;
  case ALAMD_BF16: hipLaunchKernelGGL(rms_norm_dweight_kernel<bf16_t>, grid, dim3(1024), 0, as_stream(stream), (char *)dweight, partial, (unsigned)parts, (unsigned)cols); break;
  default: hipLaunchKernelGGL(rms_norm_dweight_kernel<float>, grid, dim3(1024), 0, as_stream(stream), (char *)dweight, partial, (unsigned)parts, (unsigned)cols); break;
  }
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

}  // extern "C"
