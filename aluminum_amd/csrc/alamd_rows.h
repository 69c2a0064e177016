// Rows of a matrix held in the registers of a team of lanes: loads, stores and sums over the team.
#pragma once

#include "alamd_tile.h"

namespace alamd {

// Element access of a row's type: a 128-bit vector as floats and back (rounded to nearest, ties to even),
// and single elements.
template <typename T> struct Row {
  static constexpr int VE = 16 / sizeof(T);  // elements of a vector
  static __device__ __forceinline__ void unpack(float (&x)[VE], u32x4 v) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(v[j]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[2 * j] = widen(T{(uint16_t)(v[j] & 0xffffu)});
        x[2 * j + 1] = widen(T{(uint16_t)(v[j] >> 16)});
      }
    }
  }
  static __device__ __forceinline__ u32x4 pack(const float (&x)[VE]) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (std::is_same<T, float>::value) v[j] = __float_as_uint(x[j]);
      else if constexpr (std::is_same<T, bf16_t>::value) v[j] = narrow_bf16x2(x[2 * j], x[2 * j + 1]);
      else v[j] = (uint32_t)narrow<T>(x[2 * j]).b | ((uint32_t)narrow<T>(x[2 * j + 1]).b << 16);
    }
    return v;
  }
  static __device__ __forceinline__ float get(const char *row, unsigned c) {
    if constexpr (std::is_same<T, float>::value) return reinterpret_cast<const float *>(row)[c];
    else return widen(reinterpret_cast<const T *>(row)[c]);
  }
  static __device__ __forceinline__ void put(char *row, unsigned c, float x) {
    if constexpr (std::is_same<T, float>::value) reinterpret_cast<float *>(row)[c] = x;
    else reinterpret_cast<T *>(row)[c] = narrow<T>(x);
  }
};

// ---- sums over a team -------------------------------------------------------
//
// Butterflies: every lane ends with the same bits, and the order of the additions depends on the team's
// size alone.  Within 16 lanes the partner comes through a data-parallel move (lanes swapped in pairs,
// pairs in fours, then mirrored halves of 8 and of 16, whose members already agree), across 16 and 32
// lanes through the row swaps; the waves of a larger team meet in LDS.

template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140;

template <int LANES> __device__ __forceinline__ float lanes_sum(float x) {
  x += __uint_as_float(dpp<kSwap1>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kSwap2>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kMirror8>(__float_as_uint(x)));
  x += __uint_as_float(dpp<kMirror16>(__float_as_uint(x)));
  if constexpr (LANES > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (LANES > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// The largest of `lanes` neighbouring lanes (a power of two, the same for the whole wave).
__device__ __forceinline__ uint32_t group_max(uint32_t x, unsigned lanes) {
  if (lanes > 1) x = umax(x, dpp<kSwap1>(x));
  if (lanes > 2) x = umax(x, dpp<kSwap2>(x));
  if (lanes > 4) x = umax(x, dpp<kMirror8>(x));
  if (lanes > 8) x = umax(x, dpp<kMirror16>(x));
  if (lanes > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = umax(r[0], r[1]);
  }
  if (lanes > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    x = umax(r[0], r[1]);
  }
  return x;
}

// The waves of a workgroup of up to 1024 threads meet in `lds`, kWaves * words floats.  A caller that comes back
// needs another place the next time and may use the first again the time after (a wave that writes there has
// met all others since).
constexpr int kWaves = 16;
template <int TEAM> __device__ __forceinline__ float team_sum(float x, float *lds) {
  x = lanes_sum<(TEAM ? TEAM : 64)>(x);
  if constexpr (TEAM == 0) {
    const unsigned waves = blockDim.x >> 6;
    if (waves == 1) return x;
    if ((threadIdx.x & 63u) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    x = lds[0];
    for (unsigned k = 1; k < waves; ++k) x += lds[k];
  }
  return x;
}
// A sum and a largest word in one meeting.
template <int TEAM> __device__ __forceinline__ void team_sum_max(float &x, uint32_t &m, float *lds) {
  x = lanes_sum<(TEAM ? TEAM : 64)>(x);
  m = group_max(m, TEAM ? TEAM : 64);
  if constexpr (TEAM == 0) {
    const unsigned waves = blockDim.x >> 6;
    if (waves == 1) return;
    if ((threadIdx.x & 63u) == 0) {
      lds[2 * (threadIdx.x >> 6)] = x;
      lds[2 * (threadIdx.x >> 6) + 1] = __uint_as_float(m);
    }
    __syncthreads();
    x = lds[0];
    m = __float_as_uint(lds[1]);
    for (unsigned k = 1; k < waves; ++k) {
      x += lds[2 * k];
      m = umax(m, __float_as_uint(lds[2 * k + 1]));
    }
  }
}

// ---- a row in registers -------------------------------------------------------

// A team is the whole workgroup (TEAM = 0: as many waves as the row needs) or one of its waves (64).  Lane l of
// a team of n lanes holds the vectors l, n + l, 2 n + l, ..: vector i covers the elements [i * VE, ..) of the row.
// Where the row does not end with a whole vector, the last one is moved back to end with it: its first `skip`
// elements are then the lane's before it too.  cols >= VE.
template <typename T, int TEAM, int NV> struct RowTeam {
  static_assert(TEAM == 0 || TEAM == 64, "a wave's lanes belong to one row");
  static constexpr int VE = Row<T>::VE;
  static constexpr unsigned kNowhere = 0x7ffffff0u;  // an offset behind every row
  unsigned lane, index, size;
  unsigned cols;
  bool ragged;        // the last vector was moved back
  unsigned off[NV];   // byte offset in the row of the lane's vectors
  unsigned skip[NV];  // elements of each that another lane counts

  __device__ __forceinline__ explicit RowTeam(unsigned n) : cols(n) {
    size = TEAM ? (unsigned)TEAM : blockDim.x;
    lane = TEAM ? threadIdx.x % 64u : threadIdx.x;
    index = TEAM ? (unsigned)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64u)) : 0u;
    const unsigned full = n / VE, rem = n % VE;
    ragged = rem != 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const unsigned i = (unsigned)v * size + lane;
      const bool last = ragged && i == full;
      off[v] = i < full ? i * 16u : last ? (n - VE) * (unsigned)sizeof(T) : kNowhere;
      skip[v] = last ? VE - rem : 0u;
    }
  }
  // The first element of vector v, counted as if every vector were in its place.
  __device__ __forceinline__ unsigned element(int v) const { return ((unsigned)v * size + lane) * VE; }
  // Whether element j of vector v is this lane's to count (elements of no row are zeros and may be counted).
  __device__ __forceinline__ bool counts(int v, int j) const { return (unsigned)j >= skip[v]; }

  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const char *base, unsigned long long pitch, unsigned long long row,
                                                         bool live, unsigned bytes) const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base + row * pitch), 0, live ? (int)bytes : 0, kRsrcFlags);
  }
  __device__ __forceinline__ void load(u32x4 (&raw)[NV], const char *base, unsigned long long pitch, unsigned long long row,
                                       bool live) const {
    const auto r = rsrc(base, pitch, row, live, cols * (unsigned)sizeof(T));
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = __builtin_amdgcn_raw_buffer_load_b128(r, off[v], 0, kAuxLoadStream);
  }
  __device__ __forceinline__ void store(const u32x4 (&raw)[NV], char *base, unsigned long long pitch, unsigned long long row,
                                        bool live) const {
    const auto r = rsrc(base, pitch, row, live, cols * (unsigned)sizeof(T));
#pragma unroll
    for (int v = 0; v < NV; ++v) __builtin_amdgcn_raw_buffer_store_b128(raw[v], r, off[v], 0, kAuxStoreStream);
  }
  __device__ __forceinline__ void load_weight(float (&w)[VE], int v, const char *weight, int w32) const {
    if constexpr (!std::is_same<T, float>::value) {
      if (w32) {
        const auto r = rsrc(weight, 0, 0, true, cols * 4u);
        const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, off[v] * 2u, 0, 0);
        const u32x4 b = __builtin_amdgcn_raw_buffer_load_b128(r, off[v] * 2u + 16u, 0, 0);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = __uint_as_float(a[j]);
          w[4 + j] = __uint_as_float(b[j]);
        }
        return;
      }
    }
    const auto r = rsrc(weight, 0, 0, true, cols * (unsigned)sizeof(T));
    Row<T>::unpack(w, __builtin_amdgcn_raw_buffer_load_b128(r, off[v], 0, 0));
  }
  // x * by in e4m3, a byte each.  The elements that the lane before has too are left to that lane, whose group's
  // scale may be another.
  __device__ __forceinline__ void store_e4m3(const float (&x)[VE], int v, float by, char *base, unsigned long long pitch,
                                             unsigned long long row, bool live) const {
    uint32_t q[VE / 4];
#pragma unroll
    for (int j = 0; j < VE / 4; ++j) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * by, x[4 * j + 1] * by, 0, false);
      q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * by, x[4 * j + 3] * by, lo, true);
    }
    const unsigned at = off[v] / (unsigned)sizeof(T);
    const unsigned whole = ragged && skip[v] ? kNowhere : at;
    const auto r = rsrc(base, pitch, row, live, cols);
    if constexpr (VE == 8) {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 both = {q[0], q[1]};
      __builtin_amdgcn_raw_buffer_store_b64(both, r, whole, 0, kAuxStoreStream);
    } else {
      __builtin_amdgcn_raw_buffer_store_b32(q[0], r, whole, 0, kAuxStoreStream);
    }
    if (ragged && skip[v] && live) {
      char *o = base + row * pitch + at;
#pragma unroll
      for (int j = 1; j < VE; ++j)
        if (counts(v, j)) o[j] = (char)(q[j / 4] >> (8 * (j % 4)));
    }
  }
  // x to elements of an fp32 row.
  __device__ __forceinline__ void store_f32(const float (&x)[VE], int v, float *row) const {
    if (off[v] == kNowhere) return;
    float *o = row + off[v] / (unsigned)sizeof(T);
#pragma unroll
    for (int j = 0; j < VE; ++j) o[j] = x[j];
  }
};

}  // namespace alamd
