// Rows of a matrix held in the registers of a team of lanes: loads, stores and sums over the team.
#pragma once

#include "alamd_tile.h"

namespace alamd {

constexpr int kAuxStoreRow = 2;  // nt

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
// A team is a run of whole waves of a workgroup that hold one row together.  Sums and maxima are butterflies:
// every lane ends with the same bits, and the order of the additions depends on the team's size alone.
// Within 16 lanes the partner comes through a data-parallel move (lanes swapped in pairs, pairs in fours,
// then mirrored halves of 8 and of 16, whose members already agree), across 16 and 32 lanes through the row
// swaps; the waves of a larger team meet in LDS, where the lanes of every wave read one wave's part each.

template <int CTRL> __device__ __forceinline__ float dpp(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E, kMirror8 = 0x141, kMirror16 = 0x140, kFromLaneBehind = 0x130;

// The larger magnitude; a NaN is larger than every number.
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_elementwise_maximum(__builtin_fabsf(a), __builtin_fabsf(b));
}
__device__ __forceinline__ float lanes16_sum(float x) {
  x += dpp<kSwap1>(x);
  x += dpp<kSwap2>(x);
  x += dpp<kMirror8>(x);
  return x + dpp<kMirror16>(x);
}
__device__ __forceinline__ float wave_sum(float x) {
  x = lanes16_sum(x);
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The largest magnitude of `lanes` neighbouring lanes: 4, 8, 16, 32 or 64, the same for the whole wave.
__device__ __forceinline__ float lanes_max(float x, unsigned lanes) {
  x = larger(x, dpp<kSwap1>(x));
  x = larger(x, dpp<kSwap2>(x));
  if (lanes > 4) {
    x = larger(x, dpp<kMirror8>(x));
    if (lanes > 8) {
      x = larger(x, dpp<kMirror16>(x));
      if (lanes > 16) {
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
        if (lanes > 32) {
          r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
          x = larger(__uint_as_float(r[0]), __uint_as_float(r[1]));
        }
      }
    }
  }
  return x;
}

constexpr unsigned kMaxWaves = 16;  // of a workgroup

// ---- a row in registers -------------------------------------------------------

// The workgroup's teams: `teams` of them, `waves` waves each.
struct TeamShape { unsigned waves, teams; };
// How rows are read and written (alamd_tile.h says what the policies are): loads past the caches or through
// them, stores written through or, like the loads past the caches, not kept.
struct RowPolicy { bool stream_loads, write_through; };

// Vector i of a row covers its elements [i * VE, ..); every wave of a team holds NV runs of 64 vectors, one a
// lane, and the waves' runs follow one another.  Where the row does not end with a whole vector, the last one
// is moved back to end with it: its first `skip` elements are then the lane's before it too.  cols >= VE.
//
// HALVES: rows of 16-bit elements may start in the middle of a dword, as every other row of an odd number of
// columns does, and every load of such a row would split dwords (forward pass over 16384 rows of 5125 bf16 to
// rows of an even pitch: one stream 73 us, two 117 us; from rows of an even pitch 63 and 84).  It is read from
// the dword it starts in instead - the two bytes before it that come along share that dword -, and `settle`
// moves every lane's elements down by one, the last coming from the next lane, or, at the end of a wave's run,
// from a dword that the wave reads as a scalar: 65 and 93 us.  The backward pass lets loads split dwords, which costs it
// a quarter (16384 rows of 5125 bf16 126 us, from inputs of an even pitch 93, dx at either): what these moves cost (12
// a vector and stream) is what the loads gain (121 us either way), and with the next row's scalars under way every
// meeting of a team would wait for them besides (207 us).  What needs no moves is not built: rows that lie an even
// number apart have one parity, so that a team of odd rows could begin its vectors at the row's second element.
template <typename T, int NV, bool HALVES> struct RowTeam {
  static_assert(!HALVES || sizeof(T) == 2, "only 16-bit elements start in the middle of a dword");
  static constexpr int VE = Row<T>::VE;
  static constexpr unsigned kNowhere = 0x7ffffff0u;  // an offset behind every row
  unsigned wave, waves, index;  // the wave in the workgroup; waves of the team; which team
  unsigned lane, size;          // in the team
  unsigned cols;
  RowPolicy policy;
  bool ragged;        // a lane of this wave holds a vector that was moved back
  unsigned off[NV];   // byte offset in the row of the lane's vectors
  unsigned skip[NV];  // elements of each that another lane counts

  __device__ __forceinline__ RowTeam(unsigned n, TeamShape shape, RowPolicy how) : cols(n), policy(how) {
    wave = (unsigned)__builtin_amdgcn_readfirstlane((int)(threadIdx.x / 64u));
    waves = shape.waves;
    index = shape.teams == 1 ? 0u : wave / waves;
    size = waves * 64u;
    lane = threadIdx.x - index * size;
    const unsigned full = n / VE, rem = n % VE;
    ragged = rem != 0 && full % size / 64u == wave - index * waves;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const unsigned i = vector(v);
      const bool last = rem != 0 && i == full;
      off[v] = i < full ? i * 16u : last ? (n - VE) * (unsigned)sizeof(T) : kNowhere;
      skip[v] = last ? VE - rem : 0u;
    }
  }
  // The vector that the lane holds as its v-th, counted as if every one were in its place.
  __device__ __forceinline__ unsigned vector(int v) const { return (unsigned)v * size + lane; }
  // Whether element j of vector v is this lane's to count (elements of no row are zeros and may be counted).
  __device__ __forceinline__ bool counts(int v, int j) const { return (unsigned)j >= skip[v]; }

  // The sum over the team.  `lds`: a word for each wave; a caller that comes back needs other words the next
  // time and may use the first again the time after (a wave that writes there has met all others since).
  // Every wave of the workgroup has to come.
  __device__ __forceinline__ float sum(float x, float *lds) const {
    x = wave_sum(x);
    if (waves == 1) return x;
    if ((threadIdx.x & 63u) == 0) lds[wave] = x;
    __syncthreads();
    const unsigned k = threadIdx.x & 15u;
    return lanes16_sum(k < waves ? lds[index * waves + k] : 0.0f);
  }
  // A sum and a largest magnitude in one meeting; `lds`: two words for each wave.
  __device__ __forceinline__ void sum_max(float &x, float &m, float *lds) const {
    x = wave_sum(x);
    m = lanes_max(m, 64);
    if (waves == 1) return;
    if ((threadIdx.x & 63u) == 0) {
      lds[wave] = x;
      lds[kMaxWaves + wave] = m;
    }
    __syncthreads();
    const unsigned k = threadIdx.x & 15u;
    x = lanes16_sum(k < waves ? lds[index * waves + k] : 0.0f);
    m = lanes_max(k < waves ? lds[kMaxWaves + index * waves + k] : 0.0f, 16);
  }

  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const char *base, unsigned long long pitch, unsigned long long row,
                                                         bool live, unsigned bytes) const {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(base + row * pitch), 0, live ? (int)bytes : 0, kRsrcFlags);
  }
  // A lane's part of a row as it is in memory, and the dwords behind the wave's runs.
  struct Loaded {
    u32x4 raw[NV];
    uint32_t more[HALVES ? NV : 1];
  };
  static __device__ __forceinline__ bool split(const char *base, unsigned long long pitch, unsigned long long row) {
    return HALVES && ((reinterpret_cast<uintptr_t>(base) + row * pitch) & 2u) != 0;
  }
  __device__ __forceinline__ void load(Loaded &to, const char *base, unsigned long long pitch, unsigned long long row,
                                       bool live) const {
    const unsigned back = split(base, pitch, row) ? 2u : 0u;
    const auto r = rsrc(base - back, pitch, row, live, cols * (unsigned)sizeof(T) + back);
    unsigned at[NV];  // (the vector that was moved back is read from where it begins)
#pragma unroll
    for (int v = 0; v < NV; ++v) at[v] = HALVES && skip[v] ? off[v] + back : off[v];
    if (policy.stream_loads) {
#pragma unroll
      for (int v = 0; v < NV; ++v) to.raw[v] = __builtin_amdgcn_raw_buffer_load_b128(r, at[v], 0, kAuxLoadStream);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) to.raw[v] = __builtin_amdgcn_raw_buffer_load_b128(r, at[v], 0, kAuxLoadCached);
    }
    if constexpr (HALVES) {
      typedef const __attribute__((address_space(4))) uint32_t *Scalar;
      const uintptr_t from = (reinterpret_cast<uintptr_t>(base) + (live ? row : 0u) * pitch) & ~(uintptr_t)3;
#pragma unroll
      for (int v = 0; v < NV; ++v) to.more[v] = *reinterpret_cast<Scalar>(from + (back && live ? run_end(v) : 0u));
    }
  }
  // Where the wave's run of vectors v ends, in bytes from the dword that a split row starts in; 0: it holds none.
  // (The dword there holds the last element of the run's last vector.)
  __device__ __forceinline__ unsigned run_end(int v) const {
    const unsigned whole = cols / VE, from = (unsigned)v * size + (wave - index * waves) * 64u, end = from + 64u;
    return from < whole ? (end < whole ? end : whole) * 16u : 0u;
  }
  __device__ __forceinline__ void settle(Loaded &l, const char *base, unsigned long long pitch, unsigned long long row) const {
    if constexpr (HALVES) {
      if (!split(base, pitch, row)) return;
      // in the wave where the row ends there are lanes before the last whose next lane holds no neighbour
      const unsigned whole = cols / VE;
      const bool edge = ragged || (whole % 64u != 0 && (whole - 1u) % size / 64u == wave - index * waves);
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const u32x4 a = l.raw[v];
        // the next lane's first dword; the last lane keeps `more`, and lanes that hold nothing keep to zeros
        const uint32_t more = run_end(v) ? l.more[v] : 0u;
        uint32_t fifth = (uint32_t)__builtin_amdgcn_update_dpp((int)more, (int)a[0], kFromLaneBehind, 0xf, 0xf, false);
        if (edge) fifth = off[v] == kNowhere ? 0u : vector(v) + 1u >= whole ? more : fifth;
        u32x4 b;
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = __builtin_amdgcn_alignbit(j < 3 ? a[j < 3 ? j + 1 : 3] : fifth, a[j], 16);
        if (edge && skip[v]) b = a;
        l.raw[v] = b;
      }
    }
  }
  __device__ __forceinline__ void store(const u32x4 (&raw)[NV], char *base, unsigned long long pitch, unsigned long long row,
                                        bool live) const {
    const auto r = rsrc(base, pitch, row, live, cols * (unsigned)sizeof(T));
    if (policy.write_through) {
#pragma unroll
      for (int v = 0; v < NV; ++v) __builtin_amdgcn_raw_buffer_store_b128(raw[v], r, off[v], 0, kAuxStoreStream);
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v) __builtin_amdgcn_raw_buffer_store_b128(raw[v], r, off[v], 0, kAuxStoreRow);
    }
  }
  // A row of weights, of the rows' type or (w32) of fp32; it is read again and again.
  __device__ __forceinline__ void load_weight(float (&w)[VE], int v, const char *weight, int w32) const {
    if constexpr (!std::is_same<T, float>::value) {
      if (w32) {
        const auto r = rsrc(weight, 0, 0, true, cols * 4u);
        const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, off[v] * 2u, 0, kAuxLoadCached);
        const u32x4 b = __builtin_amdgcn_raw_buffer_load_b128(r, off[v] * 2u + 16u, 0, kAuxLoadCached);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[j] = __uint_as_float(a[j]);
          w[4 + j] = __uint_as_float(b[j]);
        }
        return;
      }
    }
    const auto r = rsrc(weight, 0, 0, true, cols * (unsigned)sizeof(T));
    Row<T>::unpack(w, __builtin_amdgcn_raw_buffer_load_b128(r, off[v], 0, kAuxLoadCached));
  }

  // x * by in e4m3, a byte each.  `apart`: what a vector that was moved back shares with the lane before belongs
  // to that lane's group, whose scale is another, and is left to that lane.  (8191 rows of f16
  // in groups of 128: 26.2 us at 4099 columns, where stores of eight bytes a lane split dwords in three rows of four, 24.8
  // at 4104, 22.3 at 4096.  Whole dwords put together across lanes, with single bytes at both ends of a wave's run, were
  // slower by half than such stores when both were tried, 51 us against 35.)
  __device__ __forceinline__ void store_e4m3(const float (&x)[VE], int v, float by, bool apart, char *base, unsigned long long pitch,
                                             unsigned long long row, bool live) const {
    uint32_t q[VE / 4];
#pragma unroll
    for (int j = 0; j < VE / 4; ++j) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j] * by, x[4 * j + 1] * by, 0, false);
      q[j] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * j + 2] * by, x[4 * j + 3] * by, lo, true);
    }
    const auto r = rsrc(base, pitch, row, live, cols);
    const unsigned at = off[v] / (unsigned)sizeof(T);
    if (!(apart && ragged)) {
      store_dwords(q, r, at);
    } else {
      store_dwords(q, r, skip[v] ? kNowhere : at);
      // the rem bytes behind the last whole vector, moved down, in pieces of four, two and one
      const unsigned rem = cols % VE;
      unsigned long long tail = VE == 8 ? (unsigned long long)q[VE / 4 - 1] << 32 | q[0] : q[0];
      tail >>= 8u * (VE - rem);
      unsigned o = skip[v] ? cols - rem : kNowhere;
      if (rem & 4u) {
        __builtin_amdgcn_raw_buffer_store_b32((uint32_t)tail, r, o, 0, 0);
        tail >>= 32;
        o += 4u;
      }
      if (rem & 2u) {
        __builtin_amdgcn_raw_buffer_store_b16((uint16_t)tail, r, o, 0, 0);
        tail >>= 16;
        o += 2u;
      }
      if (rem & 1u) __builtin_amdgcn_raw_buffer_store_b8((uint8_t)tail, r, o, 0, 0);
    }
  }
  __device__ __forceinline__ void store_dwords(const uint32_t (&d)[VE / 4], __amdgpu_buffer_rsrc_t r, unsigned at) const {
    if constexpr (VE == 8) {
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
      const u32x2 both = {d[0], d[1]};
      if (policy.write_through) __builtin_amdgcn_raw_buffer_store_b64(both, r, at, 0, kAuxStoreStream);
      else __builtin_amdgcn_raw_buffer_store_b64(both, r, at, 0, kAuxStoreRow);
    } else {
      if (policy.write_through) __builtin_amdgcn_raw_buffer_store_b32(d[0], r, at, 0, kAuxStoreStream);
      else __builtin_amdgcn_raw_buffer_store_b32(d[0], r, at, 0, kAuxStoreRow);
    }
  }
  // x as a vector of a row that is the team's alone.
  __device__ __forceinline__ void store_vector(const float (&x)[VE], int v, char *base) const {
    const auto r = rsrc(base, 0, 0, true, cols * (unsigned)sizeof(T));
    __builtin_amdgcn_raw_buffer_store_b128(Row<T>::pack(x), r, off[v], 0, 0);
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
