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
// with the factors of a row gathered: dx = rstd * (g - m * x) + dsum, m = rstd * sum(g * n_hat) / n.
//
// A team of waves holds a row in registers: NV 128-bit vectors per lane and stream, read once.  The elements
// behind the last whole vector belong to the next lane, whose vector is moved back so that it ends with the row:
// its first elements are another lane's as well, computed to the same bits, left out of every sum and stored
// twice.  Lanes without a vector read zeros and store nothing (the buffer descriptor's bound).
//
// Both passes are bound by memory from a few thousand rows on (8192 x 8192 bf16 with residual and sum: 537 MB in
// 88 us, 6.1 TB/s, where a large copy reaches 6.5; backward pass of 16384 x 8192 with dsum: 1.07 GB in 178 us,
// 6.0 TB/s), by the launches and one trip to memory below (one token of 8 x 4096: 3.6 us; backward pass of 64 x
// 1024 fp32 in two launches 5.2 us).  Where little moves for an element, what a wave does in turn counts: with 8-bit
// outputs (8191 x 4099 f16 in groups of 128: 26 us, of which 16 are the bytes') the vector units are busy for half of
// the time, and a wave's loads, arithmetic and stores follow one another, so a row is not cut finer than it has to be and
// nothing is in a loop that need not be.
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
  int apart;  // a vector that was moved back begins in another 8-bit group than it ends
  TeamShape shape;
  RowPolicy policy;
  float eps, inv_n;
};

enum { OUT_SAME = 0, OUT_E4M3_ROW = 1, OUT_E4M3_GROUP = 2 };

// The largest value e4m3 holds; the scale of a group whose largest |y| is a is max(a / 448, 2^-126), so that
// its reciprocal is finite whatever a is.
constexpr float kE4m3Max = 448.0f, kLeastScale = 1.17549435e-38f;
__device__ __forceinline__ float scale_of(float amax) {
  return __builtin_elementwise_maximum(amax * (1.0f / kE4m3Max), kLeastScale);  // a NaN passes
}

// y / scale = (s * w) * (448 / am), where am is the largest |s * w| of the group: rstd cancels, and with it its rounding
// and the scale's.  The factor for s * w, 448 / am rounded once (a product with the approximate reciprocal, and a step of
// Newton's iteration on what it leaves), so that a quotient is off by that rounding, its own, and that of s * w.  (Of 134
// million of 8191 x 4099 f16, 16 go to the wrong side of a middle between two e4m3 numbers, against 40 through rstd / scale,
// in the same time; the 1103 that lie in the middle go to either.)  A group of zeros has any factor.  Where am or rstd is
// out of range (2^-40 to 2^60, whose order is that of their bits; am * rstd / 448 is then above 2^-126), y is divided by
// the scale instead.
constexpr uint32_t kNear = 0x2b800000u, kFar = 0x5d800000u;
__device__ __forceinline__ bool factor_in_range(float am, float rstd) {
  const uint32_t bits = __float_as_uint(am);
  return ((bits == 0) | (bits - kNear <= kFar - kNear)) & (__float_as_uint(rstd) - kNear <= kFar - kNear);
}
__device__ __forceinline__ float factor_of(float am) {
  const uint32_t bits = __float_as_uint(am);
  const float a = __uint_as_float(bits < kNear ? kNear : bits), inv = __builtin_amdgcn_rcpf(a), by = kE4m3Max * inv;
  return fmaf(fmaf(-by, a, kE4m3Max), inv, by);
}
// The factor for what is left in s, which is y where the wave's part of the row has a group that is out of range.
template <int VE> __device__ __forceinline__ float quotient_factor(float (&s)[VE], float rstd, float am, float scale) {
  if (__builtin_amdgcn_ballot_w64(!factor_in_range(am, rstd)) == 0) return factor_of(am);
#pragma unroll
  for (int j = 0; j < VE; ++j) s[j] *= rstd;
  return __builtin_amdgcn_rcpf(scale);
}

template <typename T, int NV, int VE> __device__ __forceinline__ void set_row(float (&s)[NV][VE], const u32x4 (&raw)[NV]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) Row<T>::unpack(s[v], raw[v]);
}
template <typename T, int NV, int VE> __device__ __forceinline__ void add_row(float (&s)[NV][VE], const u32x4 (&raw)[NV]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    float x[VE];
    Row<T>::unpack(x, raw[v]);
#pragma unroll
    for (int j = 0; j < VE; ++j) s[v][j] += x[j];
  }
}

// Adds streams [from, P) of a row to s, in rank order, the loads of B streams issued together.
template <int B, typename T, int NV, int VE, bool HALVES>
__device__ __forceinline__ void add_streams(float (&s)[NV][VE], const RowTeam<T, NV, HALVES> &team, const char *const *in, int from, int P,
                                            unsigned long long pitch, unsigned long long row, bool live) {
  for (int k = from; k < P; k += B) {
    typename RowTeam<T, NV, HALVES>::Loaded got[B];
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (k + b < P) team.load(got[b], in[k + b], pitch, row, live);
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (k + b < P) {
        team.settle(got[b], in[k + b], pitch, row);
        add_row<T>(s, got[b].raw);
      }
  }
}

// MANY: more than one rank.
template <typename T, int NV, int OUT, bool MANY, bool HALVES>
__global__ void __launch_bounds__(1024) rms_norm_kernel(const NormParams p) {
  constexpr int VE = Row<T>::VE;
  constexpr int B = NV >= 8 ? 1 : NV >= 3 ? 2 : 4;
  __shared__ float lds[kMaxWaves * 2];
  using Team = RowTeam<T, NV, HALVES>;
  const Team team(p.cols, p.shape, p.policy);
  const unsigned long long row = (unsigned long long)blockIdx.x * p.shape.teams + team.index;
  const bool live = row < p.rows;
  typename Team::Loaded res;
  if (p.res) team.load(res, p.res, p.res_pitch, row, live);
  float s[NV][VE];
  if constexpr (MANY) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; ++j) s[v][j] = -0.0f;  // -0 + x is x, whatever x
    add_streams<B>(s, team, p.in, 0, p.P, p.in_pitch, row, live);
  } else {
    typename Team::Loaded only;
    team.load(only, p.in[0], p.in_pitch, row, live);
    team.settle(only, p.in[0], p.in_pitch, row);
    set_row<T>(s, only.raw);
  }
  if (p.res) {
    team.settle(res, p.res, p.res_pitch, row);
    add_row<T>(s, res.raw);
  }
  u32x4 raw[NV];
  float ss = 0.0f;
  if (team.ragged) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float x = team.counts(v, j) ? s[v][j] : 0.0f;  // both factors: an infinity times 0 is no number
        ss = fmaf(x, x, ss);
      }
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; ++j) ss = fmaf(s[v][j], s[v][j], ss);
  }
  if (p.sum) {
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = Row<T>::pack(s[v]);
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
  float am = 0.0f;  // the largest |s * w|
  if constexpr (OUT == OUT_E4M3_ROW) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; ++j) am = larger(am, s[v][j]);
    team.sum_max(ss, am, lds);
  } else {
    ss = team.sum(ss, lds);
  }
  // The team has met: every lane has read its part of the row.  Nothing is written before, because a vector
  // that was moved back reads what another lane writes where the sum takes the residual's place.
  if (p.sum) team.store(raw, p.sum, p.res_pitch, row, live);
  const float rstd = rsqrtf(fmaf(ss, p.inv_n, p.eps));
  if (p.rstd && live && team.lane == 0) p.rstd[row] = rstd;
  if constexpr (OUT == OUT_SAME) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < VE; ++j) s[v][j] *= rstd;
      raw[v] = Row<T>::pack(s[v]);
    }
    team.store(raw, p.out, p.out_pitch, row, live);
  } else if constexpr (OUT == OUT_E4M3_ROW) {
    const float scale = scale_of(__builtin_fabsf(am * rstd));
    if (live && team.lane == 0) p.scales[row] = scale;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const float by = quotient_factor(s[v], rstd, am, scale);
      team.store_e4m3(s[v], v, by, false, p.out, p.out_pitch, row, live);
    }
  } else {
    const unsigned lanes = (1u << p.group_log2) / VE;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float a = 0.0f;
      if (team.ragged) {
#pragma unroll
        for (int j = 0; j < VE; ++j) a = larger(a, team.counts(v, j) ? s[v][j] : 0.0f);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) a = larger(a, s[v][j]);
      }
      a = lanes_max(a, lanes);
      const float scale = scale_of(__builtin_fabsf(a * rstd));
      // one lane of a group writes its scale; a group behind the row has no place among them
      const auto r = team.rsrc(reinterpret_cast<const char *>(p.scales), p.groups * 4u, row, live, p.groups * 4u);
      const unsigned at = (team.lane & (lanes - 1)) == 0 ? (team.vector(v) * VE >> p.group_log2) * 4u : team.kNowhere;
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(scale), r, at, 0, 0);
      const float by = quotient_factor(s[v], rstd, a, scale);
      team.store_e4m3(s[v], v, by, p.apart, p.out, p.out_pitch, row, live);
    }
  }
}

// Rows shorter than a vector: one lane walks a row.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) rms_norm_short_kernel(const NormParams p) {
  const unsigned long long row = (unsigned long long)blockIdx.x * 256 + threadIdx.x;
  if (row < p.rows) {
    float s[8], ss = 0.0f, am = 0.0f;
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
      s[c] *= w;
      am = larger(am, s[c]);
    }
    if constexpr (E4M3) {
      const float scale = scale_of(__builtin_fabsf(am * rstd));
      const bool near = factor_in_range(am, rstd);  // (a wave has 64 rows here, and each keeps to itself)
      const float by = near ? factor_of(am) : __builtin_amdgcn_rcpf(scale);
      p.scales[row] = scale;
      for (unsigned c = 0; c < p.cols; ++c)
        p.out[row * p.out_pitch + c] = (char)(__builtin_amdgcn_cvt_pk_fp8_f32((near ? s[c] : s[c] * rstd) * by, 0.0f, 0, false) & 0xff);
    } else {
      for (unsigned c = 0; c < p.cols; ++c) Row<T>::put(p.out + row * p.out_pitch, c, s[c] * rstd);
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
  char *dweight;   // where a launch of one workgroup writes it to
  int dw32;        // in fp32
  int replaces_dsum;  // dx takes dsum's place, and rows do not end with a whole vector
  unsigned long long dy_pitch, x_pitch, dsum_pitch, dx_pitch;
  unsigned long long rows;
  unsigned cols;
  int P;
  int w32;
  float inv_n;
  TeamShape shape;
  RowPolicy policy;
};

// What is read of a row up front: x, dsum, rstd and B of the ranks' gradients.
template <typename T, int NV, int B> struct Fetched {
  using Team = RowTeam<T, NV, false>;
  typename Team::Loaded x, ds, dy[B];
  float rstd;
  __device__ __forceinline__ void fetch(const GradParams &p, const Team &team, unsigned long long row) {
    const bool live = row < p.rows;
#pragma unroll
    for (int b = 0; b < B; ++b)
      if (b < p.P) team.load(dy[b], p.dy[b], p.dy_pitch, row, live);
    team.load(x, p.x, p.x_pitch, row, live);
    if (p.dsum) team.load(ds, p.dsum, p.dsum_pitch, row, live);
    rstd = live ? p.rstd[row] : 0.0f;
  }
};

// WIDE: rows of so many vectors a lane that the weight's gradient is kept in LDS and nothing is read ahead.
template <typename T, int NV, int B, bool WIDE, int THREADS>
__global__ void __launch_bounds__(THREADS) rms_norm_grad_kernel(const GradParams p) {
  constexpr int VE = Row<T>::VE;
  constexpr bool AHEAD = !(WIDE || (NV == 2 && THREADS > 512));  // the next row is read ahead
  __shared__ float lds[2][kMaxWaves];
  extern __shared__ float4 kept[];  // WIDE: the weight's gradient; else room for half of the teams to hand it over
  using Team = RowTeam<T, NV, false>;
  const Team team(p.cols, p.shape, p.policy);
  auto slot = [&](int v, int j) -> float4 & { return kept[(unsigned)(v * (VE / 4) + j / 4) * team.size + team.lane]; };
  float dw[WIDE ? 1 : NV][VE], w[WIDE ? 1 : NV][VE];
  if constexpr (WIDE) {
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VE; j += 4) slot(v, j) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        dw[v][j] = 0.0f;
        w[v][j] = 1.0f;
      }
      if (p.weight) team.load_weight(w[v], v, p.weight, p.w32);
    }
  }
  int turn = 0;
  const unsigned long long step = (unsigned long long)gridDim.x * p.shape.teams;
  unsigned long long r0 = (unsigned long long)blockIdx.x * p.shape.teams;
  Fetched<T, NV, B> next;
  if constexpr (AHEAD) next.fetch(p, team, r0 + team.index);
  for (; r0 < p.rows; r0 += step, turn ^= 1) {
    const unsigned long long row = r0 + team.index;
    const bool live = row < p.rows;
    if constexpr (!AHEAD) next.fetch(p, team, row);
    Fetched<T, NV, B> now = next;
    // the next row's loads are on their way while this one's sum is made and its gradient written (two or three
    // rows ahead are no faster: 45.6 and 56.7 us against 43.8 for 4 ranks of 2777 x 5120 f16)
    if constexpr (AHEAD) next.fetch(p, team, row + step);
    float g[NV][VE];
    set_row<T>(g, now.dy[0].raw);
#pragma unroll
    for (int b = 1; b < B; ++b)
      if (b < p.P) add_row<T>(g, now.dy[b].raw);
    add_streams<(WIDE ? 1 : 4)>(g, team, p.dy, B, p.P, p.dy_pitch, row, live);
    float dot = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if constexpr (NV >= 4) __builtin_amdgcn_sched_barrier(0);  // one vector after another: registers are short
      float x[VE], wv[VE], d[VE];
      Row<T>::unpack(x, now.x.raw[v]);
      if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < VE; ++j) wv[j] = 1.0f;
        if (p.weight) team.load_weight(wv, v, p.weight, p.w32);
#pragma unroll
        for (int j = 0; j < VE; j += 4) {
          const float4 a = slot(v, j);
          d[j] = a.x, d[j + 1] = a.y, d[j + 2] = a.z, d[j + 3] = a.w;
        }
      }
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        x[j] *= now.rstd;
        // a row that is not there has rstd = 0 and reads zeros
        if constexpr (WIDE) d[j] = fmaf(g[v][j], x[j], d[j]);
        else dw[v][j] = fmaf(g[v][j], x[j], dw[v][j]);
        g[v][j] *= WIDE ? wv[j] : w[WIDE ? 0 : v][j];
      }
      if (team.ragged) {
#pragma unroll
        for (int j = 0; j < VE; ++j) dot = team.counts(v, j) ? fmaf(g[v][j], x[j], dot) : dot;  // (0 times an infinity is no number)
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j) dot = fmaf(g[v][j], x[j], dot);
      }
      if constexpr (WIDE) {
#pragma unroll
        for (int j = 0; j < VE; j += 4) slot(v, j) = make_float4(d[j], d[j + 1], d[j + 2], d[j + 3]);
      }
    }
    if (p.dx) {
      // Where dx takes dsum's place and a vector was moved back, the waves that hold it and the vector in front both read
      // the elements that the two share and, once the team has met, write them: no load of dsum may be under way then.
      // (What is read of the other streams has gone into `dot`.)
      if (p.replaces_dsum) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      const float m = team.sum(dot, lds[turn]) * p.inv_n * now.rstd;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if constexpr (NV >= 4) __builtin_amdgcn_sched_barrier(0);
        float x[VE];
        asm volatile("" : "+v"(now.x.raw[v]));  // x is widened again, not kept as floats
        Row<T>::unpack(x, now.x.raw[v]);
#pragma unroll
        for (int j = 0; j < VE; ++j) g[v][j] = fmaf(-m, x[j], g[v][j]);
        if (p.dsum) {
          float d[VE];
          Row<T>::unpack(d, now.ds.raw[v]);
#pragma unroll
          for (int j = 0; j < VE; ++j) g[v][j] = fmaf(now.rstd, g[v][j], d[j]);
        } else {
#pragma unroll
          for (int j = 0; j < VE; ++j) g[v][j] *= now.rstd;
        }
        now.x.raw[v] = Row<T>::pack(g[v]);
      }
      team.store(now.x.raw, p.dx, p.dx_pitch, row, live);
    }
  }
  if (!p.partial) return;
  float *dst = p.partial + (size_t)blockIdx.x * p.cols;
  auto put = [&](const float (&d)[VE], int v) {
    if (gridDim.x > 1) team.store_f32(d, v, dst);
    else if (p.dw32) team.store_f32(d, v, reinterpret_cast<float *>(p.dweight));
    else team.store_vector(d, v, p.dweight);
  };
  if constexpr (WIDE) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float d[VE];
#pragma unroll
      for (int j = 0; j < VE; j += 4) {
        const float4 a = slot(v, j);
        d[j] = a.x, d[j + 1] = a.y, d[j + 2] = a.z, d[j + 3] = a.w;
      }
      put(d, v);
    }
  } else {
    // the upper half of the teams hands its part to the lower half, until one team has all (rows of two vectors a lane
    // have one team)
    for (unsigned n = NV == 1 ? p.shape.teams : 1; n > 1;) {
      const unsigned half = (n + 1) / 2;
      const unsigned room = NV * (VE / 4) * team.size;
      if (team.index >= half && team.index < n) {
        float4 *to = kept + (team.index - half) * room;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int j = 0; j < VE; j += 4)
            to[(unsigned)(v * (VE / 4) + j / 4) * team.size + team.lane] = make_float4(dw[v][j], dw[v][j + 1], dw[v][j + 2], dw[v][j + 3]);
      }
      __syncthreads();
      if (team.index < n - half) {
        const float4 *from = kept + team.index * room;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int j = 0; j < VE; j += 4) {
            const float4 a = from[(unsigned)(v * (VE / 4) + j / 4) * team.size + team.lane];
            dw[v][j] += a.x, dw[v][j + 1] += a.y, dw[v][j + 2] += a.z, dw[v][j + 3] += a.w;
          }
      }
      __syncthreads();
      n = half;
    }
    if (team.index == 0) {
#pragma unroll
      for (int v = 0; v < NV; ++v) put(dw[v], v);
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
    for (unsigned k = slice; k < parts; k += 32u * 8u) {
      float x[8];
#pragma unroll
      for (unsigned u = 0; u < 8; ++u) x[u] = k + u * 32u < parts ? partial[(size_t)(k + u * 32u) * cols + col] : 0.0f;
#pragma unroll
      for (unsigned u = 0; u < 8; ++u) a += x[u];
    }
  }
  lds[slice][c] = a;
  __syncthreads();
  if (slice == 0 && col < cols) {
#pragma unroll
    for (int k = 1; k < 32; ++k) a += lds[k][c];
    Row<W>::put(dw, col, a);
  }
}

// ---- host side ----------------------------------------------------------------

// A matrix of the call: a name for messages, the first row, bytes between rows and of a row.  A written one may take
// the place of a read one if both are of the kind that allows it.
enum Use { READ, READ_REPLACEABLE, WRITTEN, WRITTEN_IN_PLACE };
struct Matrix {
  const char *name;
  const void *p;
  size_t pitch, bytes;
  Use use;
  bool written() const { return use == WRITTEN || use == WRITTEN_IN_PLACE; }
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

// Every written matrix against every other one.
int check_overlaps(const Matrix *m, int n, size_t rows) {
  for (int a = 0; a < n; ++a) {
    if (!m[a].written() || !m[a].p) continue;
    for (int b = 0; b < n; ++b) {
      if (b == a || !m[b].p || (m[b].written() && b < a)) continue;
      if (m[a].use == WRITTEN_IN_PLACE && m[b].use == READ_REPLACEABLE && m[a].p == m[b].p && m[a].bytes == m[b].bytes &&
          (m[a].pitch == m[b].pitch || rows == 1))
        continue;
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

// Workgroups of a launch; what is left is done by further ones.
constexpr size_t kMaxGrid = (size_t)1 << 21;

// Whether rows of 16-bit elements may start in the middle of a dword.
inline bool starts_in_a_dword(const void *at, size_t pitch) { return ((reinterpret_cast<uintptr_t>(at) | pitch) & 2u) != 0; }
// Whether rows cover whole 64-byte pieces of memory.
inline bool whole_lines(const void *at, size_t pitch, size_t bytes) {
  return ((reinterpret_cast<uintptr_t>(at) | pitch | bytes) & 63u) == 0;
}

// A call that moves less than this reads through the caches and stores past them (nt); from there on it reads past
// them, and writes through where rows cover whole 64-byte pieces.  Both ways in us, bf16 with residual and sum: 134 MB
// of 4096 x 4096 21.7 / 23.5, 268 MB of 4096 x 8192 48.4 / 47.2, 1.07 GB of 16384 x 8192 188 / 176; read past the
// caches and written through / nt: 8 ranks of 2048 x 8192 62.5 / 65.3, 16384 rows of 5125 columns, which share their
// 64-byte pieces, 154 / 126.  The backward pass, which mostly reads, gains from less on (residual's gradient with it,
// 4096 rows: 34 MB of 1024 columns 11.3 / 11.8, 134 MB of 4096 29.7 / 27.2).
constexpr size_t kStreamFromBytes = (size_t)256 << 20, kGradStreamFromBytes = (size_t)64 << 20;

// Waves that hold a row of `need` vectors, nv of them a lane.
constexpr unsigned waves_for(unsigned need, unsigned nv) { return (need + 64 * nv - 1) / (64 * nv); }

// The call on the rows from the first `done` on.
inline NormParams from_row(NormParams p, size_t done) {
  for (int k = 0; k < p.P; ++k) p.in[k] += done * p.in_pitch;
  if (p.res) p.res += done * p.res_pitch;
  if (p.sum) p.sum += done * p.res_pitch;
  p.out += done * p.out_pitch;
  if (p.rstd) p.rstd += done;
  if (p.scales) p.scales += done * p.groups;
  p.rows -= done;
  return p;
}

// Launches `kern`, whose workgroups have `threads` threads and do `per` rows each.
inline int launch_rows(void (*kern)(NormParams), const NormParams &p, size_t per, unsigned threads, hipStream_t stream) {
  for (size_t done = 0; done < p.rows; done += kMaxGrid * per) {
    const size_t left = (p.rows - done + per - 1) / per;
    hipLaunchKernelGGL(kern, dim3((unsigned)(left < kMaxGrid ? left : kMaxGrid)), dim3(threads), 0, stream,
                       done ? from_row(p, done) : p);
  }
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}

template <typename T, int NV, bool MANY> void (*norm_kernel(int out, bool halves))(NormParams) {
  if constexpr (sizeof(T) == 2)
    if (halves)
      return out == OUT_SAME       ? rms_norm_kernel<T, NV, OUT_SAME, MANY, true>
             : out == OUT_E4M3_ROW ? rms_norm_kernel<T, NV, OUT_E4M3_ROW, MANY, true>
                                   : rms_norm_kernel<T, NV, OUT_E4M3_GROUP, MANY, true>;
  return out == OUT_SAME       ? rms_norm_kernel<T, NV, OUT_SAME, MANY, false>
         : out == OUT_E4M3_ROW ? rms_norm_kernel<T, NV, OUT_E4M3_ROW, MANY, false>
                               : rms_norm_kernel<T, NV, OUT_E4M3_GROUP, MANY, false>;
}
template <typename T, int NV>
int launch_norm(NormParams &p, int out, bool halves, unsigned waves, unsigned teams, hipStream_t stream) {
  p.shape = {waves, teams};
  return launch_rows(p.P > 1 ? norm_kernel<T, NV, true>(out, halves) : norm_kernel<T, NV, false>(out, halves), p, teams,
                     64 * waves * teams, stream);
}

template <typename T> int norm_rows(NormParams &p, int out, hipStream_t stream) {
  constexpr unsigned VE = Row<T>::VE;
  if (p.cols < VE)
    return launch_rows(out == OUT_SAME ? rms_norm_short_kernel<T, false> : rms_norm_short_kernel<T, true>, p, 256, 256, stream);
  const unsigned need = (p.cols + VE - 1) / VE;  // vectors of a row
  bool halves = false;
  if (sizeof(T) == 2) {
    halves = p.res && starts_in_a_dword(p.res, p.res_pitch);
    for (int k = 0; k < p.P; ++k) halves = halves || starts_in_a_dword(p.in[k], p.in_pitch);
  }
  // One vector a lane where there are few rows and time is a matter of the longest chain (one / two in
  // us: bf16, 16 rows of 8192 3.1 / 3.2, 512 rows 6.8 / 7.1, 768 rows 10.0 / 9.2, of 5120 4.6 / 5.0 and 7.3 / 6.9; rows of
  // 2048 would gain up to 2048 of them, 7.0 / 7.2; 8191 rows of 5120 f16 33.5 / 29.6); otherwise two or three,
  // whichever leaves fewer places of the team's waves empty, because a wave takes its time however little it holds
  // (8191 rows of f16, two / three: 4096 columns 24.0 / 24.4 us, 4099 columns 27.0 / 24.8, to 8 bits in groups of
  // 128 30.7 / 25.9; one a lane 31.9 and 37.3, four 28.8 and 31.1).
  const unsigned one = waves_for(need, 1), two = waves_for(need, 2), three = waves_for(need, 3), four = waves_for(need, 4);
  if (one == 1) return launch_norm<T, 1>(p, out, halves, 1, 4, stream);
  if (p.rows <= 512 && one <= kMaxWaves) return launch_norm<T, 1>(p, out, halves, one, 1, stream);
  if (3 * three < 2 * two && three <= kMaxWaves) return launch_norm<T, 3>(p, out, halves, three, three == 1 ? 4 : 1, stream);
  if (two <= kMaxWaves) return launch_norm<T, 2>(p, out, halves, two, two == 1 ? 4 : 1, stream);
  if constexpr (sizeof(T) == 4)
    if (four > kMaxWaves) return launch_norm<T, 8>(p, out, halves, waves_for(need, 8), 1, stream);
  static_assert(waves_for(kMaxCols / VE, sizeof(T) == 4 ? 8 : 4) <= kMaxWaves, "the longest row fits a workgroup");
  return launch_norm<T, 4>(p, out, halves, four, 1, stream);
}

// Workgroups whose partial sums of the weight's gradient are kept: one for every CU.  (With two the parts, which grow
// with them, cost more than the second workgroup gains: 16384 x 8192 bf16 183 us against 179, 4 ranks of 2777 x 5120
// f16 47.8 against 43.9.)
constexpr size_t kGradParts = 256;

template <typename T, int NV, int B, bool WIDE, int THREADS>
int launch_grad_b(GradParams &p, size_t *parts, unsigned waves, unsigned teams, hipStream_t stream) {
  p.shape = {waves, teams};
  size_t grid = (p.rows + teams - 1) / teams;
  if (grid > kGradParts) grid = kGradParts;
  if (p.partial && p.rows <= 2 * (size_t)teams) grid = 1;
  *parts = grid == 1 ? 0 : grid;  // one workgroup has written the weight's gradient itself
  const size_t lds = (WIDE ? 1 : teams / 2) * (size_t)waves * 64 * NV * Row<T>::VE * sizeof(float);
  hipLaunchKernelGGL((rms_norm_grad_kernel<T, NV, B, WIDE, THREADS>), dim3((unsigned)grid), dim3(64 * waves * teams), lds, stream, p);
  ALAMD_HIP(hipGetLastError());
  return ALAMD_OK;
}
// Rows of one vector a lane.
template <typename T> int launch_grad(GradParams &p, size_t *parts, unsigned waves, hipStream_t stream) {
  // As many rows a workgroup as it has waves for, so that there are few parts to join; but every CU gets a row first,
  // except where one workgroup does the whole call in two turns, which saves the second launch.
  unsigned teams = kMaxWaves / waves;
  if (!p.partial || p.rows > 2 * (size_t)teams)
    while (teams > 1 && p.rows < (size_t)256 * teams) --teams;
  if (teams > p.rows) teams = (unsigned)p.rows;
  return p.P == 1 ? launch_grad_b<T, 1, 1, false, 1024>(p, parts, waves, teams, stream)
                  : launch_grad_b<T, 1, 4, false, 1024>(p, parts, waves, teams, stream);
}

template <typename T> int grad_rows(GradParams &p, size_t *parts, hipStream_t stream) {
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
  const unsigned one = waves_for(need, 1), two = waves_for(need, 2), four = waves_for(need, 4);
  // One vector a lane up to 12 waves, two from there on (us, one / two: 256 rows of 4096 bf16 8.1 / 8.6, 4 ranks of 2777 x
  // 5125 f16 53.7 / 55.7, 16384 x 8192 bf16 182 / 179; from 13 waves on fewer rows would gain from one, 256 of 8192 10.9 /
  // 11.4, 4096 of 7168 42.4 / 43.3); rows longer than a workgroup of eight waves can read ahead in its registers are read
  // as they come.
  if (one <= 12) return launch_grad<T>(p, parts, one, stream);
  if (two <= 8)
    return p.P == 1 ? launch_grad_b<T, 2, 1, false, 512>(p, parts, two, 1, stream)
                    : launch_grad_b<T, 2, 4, false, 512>(p, parts, two, 1, stream);
  if (two <= kMaxWaves) return launch_grad_b<T, 2, 1, false, 1024>(p, parts, two, 1, stream);
  if constexpr (sizeof(T) == 4)
    if (four > kMaxWaves) return launch_grad_b<T, 8, 1, true, 1024>(p, parts, waves_for(need, 8), 1, stream);
  return launch_grad_b<T, 4, 1, true, 1024>(p, parts, four, 1, stream);
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
    m[n++] = {"a rank's input", ins[k], in_stride * es, cols * es, READ_REPLACEABLE};
  }
  if (residual && (rc = check_matrix(residual, "the residual", residual_stride, rows, cols, es))) return rc;
  if (sum && (rc = check_matrix(sum, "the sum", residual_stride, rows, cols, es))) return rc;
  if ((rc = check_matrix(out, "the output", out_stride, rows, cols, oes))) return rc;
  if ((rstd && !aligned_to(rstd, 4)) || (scales && !aligned_to(scales, 4)))
    return set_error(ALAMD_ERR_INVALID_ARG, "rstd or scales not aligned to fp32");
  const size_t groups = scales && group ? (cols + group - 1) / group : 1;
  m[n++] = {"the residual", residual, residual_stride * es, cols * es, READ_REPLACEABLE};
  m[n++] = {"the weight", weight, 0, cols * wes, READ};
  m[n++] = {"the sum", sum, residual_stride * es, cols * es, WRITTEN_IN_PLACE};
  m[n++] = {"the output", out, out_stride * oes, cols * oes, WRITTEN_IN_PLACE};
  m[n++] = {"rstd", rstd, 4, 4, WRITTEN};
  m[n++] = {"the scales", scales, groups * 4, groups * 4, WRITTEN};
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
  p.apart = cols % (16 / es) != 0 && (cols - cols % (16 / es)) % (group ? group : cols) == 0;
  const size_t moved = rows * cols * (es * ((size_t)P + (residual ? 1 : 0) + (sum ? 1 : 0)) + oes);
  p.policy = {moved >= kStreamFromBytes, moved >= kStreamFromBytes && whole_lines(out, p.out_pitch, cols * oes) &&
                                             (!sum || whole_lines(sum, p.res_pitch, cols * es))};
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
      m[n++] = {"a rank's gradient", dys[k], dy_stride * es, cols * es, READ_REPLACEABLE};
    }
    if ((rc = check_matrix(x, "x", x_stride, rows, cols, es))) return rc;
    if (dsum && (rc = check_matrix(dsum, "dsum", dsum_stride, rows, cols, es))) return rc;
    if (dx && (rc = check_matrix(dx, "dx", dx_stride, rows, cols, es))) return rc;
    if (!rstd || !aligned_to(rstd, 4)) return set_error(ALAMD_ERR_INVALID_ARG, "rstd is null or not aligned to fp32");
    if (dweight && (!workspace || !aligned_to(workspace, 4)))
      return set_error(ALAMD_ERR_INVALID_ARG, "dweight needs a workspace aligned to fp32 (alamd_rms_norm_grad_workspace)");
    m[n++] = {"x", x, x_stride * es, cols * es, READ_REPLACEABLE};
    m[n++] = {"dsum", dsum, dsum_stride * es, cols * es, READ_REPLACEABLE};
    m[n++] = {"rstd", rstd, 4, 4, READ};
    m[n++] = {"the weight", weight, 0, cols * wes, READ};
    m[n++] = {"dx", dx, dx_stride * es, cols * es, WRITTEN_IN_PLACE};
    m[n++] = {"dweight", dweight, 0, cols * wes, WRITTEN};
    if (dweight) {
      // the workspace has rows of its own: as one stretch of bytes
      const size_t bytes = alamd_rms_norm_grad_workspace(rows, cols);
      m[n++] = {"the workspace", workspace, 0, bytes, WRITTEN};
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
    p.dweight = static_cast<char *>(dweight);
    p.dw32 = weight_dtype == ALAMD_F32;
    p.replaces_dsum = dsum && dx == dsum && cols % (16 / es) != 0;
    p.dy_pitch = dy_stride * es;
    p.x_pitch = x_stride * es;
    p.dsum_pitch = dsum_stride * es;
    p.dx_pitch = dx_stride * es;
    p.rows = rows;
    p.cols = (unsigned)cols;
    p.P = P;
    p.w32 = weight && weight_dtype == ALAMD_F32;
    p.inv_n = 1.0f / (float)cols;
    const size_t moved = rows * cols * es * ((size_t)P + 1 + (dsum ? 1 : 0) + (dx ? 1 : 0));
    p.policy = {moved >= kGradStreamFromBytes,
                moved >= kGradStreamFromBytes && whole_lines(dx, p.dx_pitch, cols * es)};
    switch (dtype) {
    case ALAMD_F16: rc = grad_rows<f16_t>(p, &parts, as_stream(stream)); break;
    case ALAMD_BF16: rc = grad_rows<bf16_t>(p, &parts, as_stream(stream)); break;
    default: rc = grad_rows<float>(p, &parts, as_stream(stream)); break;
    }
    if (rc) return rc;
  }
  if (!dweight || (rows > 0 && parts == 0)) return ALAMD_OK;
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
