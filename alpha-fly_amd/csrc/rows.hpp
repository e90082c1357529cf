// Rows of float32, float16 or bfloat16 in 16-byte pieces, and sums and maxima over a workgroup.
#pragma once

#include "common.hpp"

#include <type_traits>

namespace fly {

typedef __bf16 bhalf;

// 16 bytes at any 2-byte alignment: rows of an odd length start anywhere, and the hardware loads and stores dwords
// at any address, so one path serves every row.
struct __attribute__((packed, aligned(2))) Raw16 {
  uint32_t v[4];
};

template <typename T>
struct Piece {
  static constexpr int N = 16 / (int)sizeof(T);
  float v[N];
};

template <typename T>
__device__ __forceinline__ float to_float(uint32_t bits) {   // the low bits hold a T
  if constexpr (std::is_same_v<T, float>) return __uint_as_float(bits);
  else if constexpr (std::is_same_v<T, bhalf>) return __uint_as_float(bits << 16);
  else return static_cast<float>(__builtin_bit_cast(_Float16, (uint16_t)bits));
}

// Elements [i N, i N + N) of a row of `cols`; `fill` past its end.
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T *__restrict__ row, int64_t i, int64_t cols, float fill) {
  constexpr int N = Piece<T>::N;
  Piece<T> p;
  const int64_t c = i * N;
  if (c + N <= cols) {
    const Raw16 raw = *reinterpret_cast<const Raw16 *>(row + c);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if constexpr (N == 4) p.v[e] = __uint_as_float(raw.v[e]);
      else p.v[e] = to_float<T>((e & 1) ? raw.v[e / 2] >> 16 : raw.v[e / 2] & 0xffffu);
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = c + e < cols ? static_cast<float>(row[c + e]) : fill;
  }
  return p;
}

template <typename T>
__device__ __forceinline__ void store_piece(T *__restrict__ row, int64_t i, int64_t cols, const Piece<T> &p) {
  constexpr int N = Piece<T>::N;
  const int64_t c = i * N;
  if (c + N <= cols) {
    Raw16 raw;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if constexpr (N == 4) raw.v[w] = __float_as_uint(p.v[w]);
      else
        raw.v[w] = (uint32_t)__builtin_bit_cast(uint16_t, static_cast<T>(p.v[2 * w])) |
                   (uint32_t)__builtin_bit_cast(uint16_t, static_cast<T>(p.v[2 * w + 1])) << 16;
    }
    *reinterpret_cast<Raw16 *>(row + c) = raw;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < cols) row[c + e] = static_cast<T>(p.v[e]);
  }
}

// Columns whose byte in `seen` (a row of the mask, any alignment) is 0 become -inf.
template <typename T>
__device__ __forceinline__ void mask_piece(Piece<T> &p, const uint8_t *__restrict__ seen, int64_t i, int64_t cols) {
  constexpr int N = Piece<T>::N;
  struct __attribute__((packed)) Bytes {
    uint32_t w[N / 4];
  };
  const int64_t c = i * N;
  if (c + N <= cols) {
    const Bytes b = *reinterpret_cast<const Bytes *>(seen + c);
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (!((b.w[e / 4] >> (8 * (e & 3))) & 0xffu)) p.v[e] = -INFINITY;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < cols && !seen[c + e]) p.v[e] = -INFINITY;
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {   // NaN where any lane has one
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float o = __shfl_xor(v, d);
    v = (o > v || o != o) ? o : v;
  }
  return v;
}

// C values over the workgroup, in every thread; `share` holds C * (waves) floats.  Sums add in wave order.
template <int C>
__device__ __forceinline__ void block_sum(float (&v)[C], float *share) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = wave_sum(v[c]);
  if (waves == 1) return;
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int c = 0; c < C; ++c) share[c * waves + wave] = v[c];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float s = share[c * waves];
    for (int w = 1; w < waves; ++w) s += share[c * waves + w];
    v[c] = s;
  }
}
template <int C>
__device__ __forceinline__ void block_max(float (&v)[C], float *share) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = (blockDim.x + 63) >> 6;
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = wave_max(v[c]);
  if (waves == 1) return;
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int c = 0; c < C; ++c) share[c * waves + wave] = v[c];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float s = share[c * waves];
    for (int w = 1; w < waves; ++w) {
      const float o = share[c * waves + w];
      s = (o > s || o != o) ? o : s;
    }
    v[c] = s;
  }
}

}  // namespace fly
