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
constexpr uint32_t kLowest = std::is_same_v<T, float> ? 0xff800000u : std::is_same_v<T, bhalf> ? 0xff80u : 0xfc00u;   // -inf

template <typename T>
__device__ __forceinline__ float to_float(uint32_t bits) {   // the low bits hold a T
  if constexpr (std::is_same_v<T, float>) return __uint_as_float(bits);
  else if constexpr (std::is_same_v<T, bhalf>) return __uint_as_float(bits << 16);
  else return static_cast<float>(__builtin_bit_cast(_Float16, (uint16_t)bits));
}
template <typename T>
__device__ __forceinline__ uint32_t to_bits(T v) {
  if constexpr (std::is_same_v<T, float>) return __float_as_uint(v);
  else return __builtin_bit_cast(uint16_t, v);
}

// Element e of a piece, and -inf in its place.
template <typename T>
__device__ __forceinline__ float element(const Raw16 &p, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(p.v[e]);
  else if constexpr (std::is_same_v<T, bhalf>)
    return __uint_as_float((e & 1) ? p.v[e / 2] & 0xffff0000u : p.v[e / 2] << 16);
  else return to_float<T>((e & 1) ? p.v[e / 2] >> 16 : p.v[e / 2] & 0xffffu);
}
template <typename T>
__device__ __forceinline__ void erase(Raw16 &p, int e) {
  if constexpr (sizeof(T) == 4) p.v[e] = kLowest<T>;
  else if (e & 1) p.v[e / 2] = (p.v[e / 2] & 0xffffu) | kLowest<T> << 16;
  else p.v[e / 2] = (p.v[e / 2] & 0xffff0000u) | kLowest<T>;
}

// Whole piece i of a row, and the `left` < N elements of its last one, -inf behind them.
template <typename T>
__device__ __forceinline__ Raw16 load_whole(const T *__restrict__ row, int i) {
  return *reinterpret_cast<const Raw16 *>(row + (int64_t)i * Piece<T>::N);
}
template <typename T>
__device__ __forceinline__ Raw16 load_last(const T *__restrict__ row, int i, int left) {
  constexpr int N = Piece<T>::N;
  Raw16 p;
#pragma unroll
  for (int w = 0; w < 4; ++w) p.v[w] = sizeof(T) == 4 ? kLowest<T> : kLowest<T> * 0x10001u;
#pragma unroll
  for (int e = 0; e < N - 1; ++e)
    if (e < left) {
      const uint32_t b = to_bits(row[(int64_t)i * N + e]);
      if constexpr (sizeof(T) == 4) p.v[e] = b;
      else p.v[e / 2] = (e & 1) ? (p.v[e / 2] & 0xffffu) | b << 16 : (p.v[e / 2] & 0xffff0000u) | b;
    }
  return p;
}

// Elements [i N, i N + N) of a row of `cols` as floats, `fill` past its end.
template <typename T>
__device__ __forceinline__ Piece<T> load_piece(const T *__restrict__ row, int64_t i, int64_t cols, float fill) {
  constexpr int N = Piece<T>::N;
  Piece<T> p;
  const int64_t c = i * N;
  if (c + N <= cols) {
    const Raw16 raw = *reinterpret_cast<const Raw16 *>(row + c);
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = element<T>(raw, e);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = c + e < cols ? static_cast<float>(row[c + e]) : fill;
  }
  return p;
}

// PAST: around the caches.
template <typename T, bool PAST>
__device__ __forceinline__ void store_whole(T *__restrict__ row, int i, const Piece<T> &p) {
  constexpr int N = Piece<T>::N;
  Raw16 raw;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (N == 4) raw.v[w] = __float_as_uint(p.v[w]);
    else raw.v[w] = to_bits(static_cast<T>(p.v[2 * w])) | to_bits(static_cast<T>(p.v[2 * w + 1])) << 16;
  }
  typedef uint32_t words __attribute__((ext_vector_type(4), aligned(2)));
  if constexpr (PAST)
    __builtin_nontemporal_store(words{raw.v[0], raw.v[1], raw.v[2], raw.v[3]},
                                reinterpret_cast<words *>(row + (int64_t)i * N));
  else *reinterpret_cast<Raw16 *>(row + (int64_t)i * N) = raw;
}
template <typename T>
__device__ __forceinline__ void store_last(T *__restrict__ row, int i, int left, const Piece<T> &p) {
#pragma unroll
  for (int e = 0; e < Piece<T>::N - 1; ++e)
    if (e < left) row[(int64_t)i * Piece<T>::N + e] = static_cast<T>(p.v[e]);
}

// Columns whose byte in `seen` (a row of the mask, any alignment) is 0 become -inf.
template <typename T>
__device__ __forceinline__ void mask_whole(Raw16 &p, const uint8_t *__restrict__ seen, int i) {
  constexpr int N = Piece<T>::N;
  struct __attribute__((packed)) Bytes {
    uint32_t w[N / 4];
  };
  const Bytes b = *reinterpret_cast<const Bytes *>(seen + (int64_t)i * N);
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (!((b.w[e / 4] >> (8 * (e & 3))) & 0xffu)) erase<T>(p, e);
}
template <typename T>
__device__ __forceinline__ void mask_last(Raw16 &p, const uint8_t *__restrict__ seen, int i, int left) {
#pragma unroll
  for (int e = 0; e < Piece<T>::N - 1; ++e)
    if (e < left && !seen[(int64_t)i * Piece<T>::N + e]) erase<T>(p, e);
}

// The hardware's 2^x and log2 (within an ulp or so; 2^x of less than -126 is 0).
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_of(float x) { return __builtin_amdgcn_logf(x); }

// x from lane ^ 1, ^ 2 (within 4 lanes), rotated by 4 and 8 within 16, and across the 16- and 32-lane halves: six steps
// on the vector ALU that leave a whole wave's sum or maximum in every lane.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <typename F>
__device__ __forceinline__ float reduce16(float v, F &&f) {   // over each 16 lanes
  v = f(v, dpp<0xB1>(v));    // quad_perm 1 0 3 2
  v = f(v, dpp<0x4E>(v));    // quad_perm 2 3 0 1
  v = f(v, dpp<0x124>(v));   // row_ror:4
  return f(v, dpp<0x128>(v));   // row_ror:8
}
template <typename F>
__device__ __forceinline__ float wave_reduce(float v, F &&f) {
  v = reduce16(v, f);
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
  v = f(__int_as_float(h[0]), __int_as_float(h[1]));
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return f(__int_as_float(w[0]), __int_as_float(w[1]));
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(v, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float wave_max(float v) {   // of numbers: NaN only where every lane has one
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float nan_max(float a, float b) { return b > a || b != b ? b : a; }

// sum exp2((x - top) scale): a part of a log-sum-exp.  Of nothing: {-inf, 0}.  NaN among the terms makes the sum NaN whatever
// top is.  The maximum is taken off before the scale is put on: a type's lowest value, which masks are made of, would
// pass the range otherwise.
struct PartSum {
  float top, sum;
  __device__ __forceinline__ bool empty() const { return top == -INFINITY && sum == 0.0f; }
};
__device__ __forceinline__ float base_of(float top) { return top == -INFINITY ? 0.0f : top; }   // no inf - inf
__device__ __forceinline__ PartSum wave_part(PartSum p, float scale) {
  const float top = wave_max(p.top);
  p.sum = wave_sum(p.sum * exp2_of((p.top - base_of(top)) * scale));
  p.top = top;
  return p;
}

// x joins a part
__device__ __forceinline__ void join(PartSum &p, float x, float scale) {
  const float top = fmaxf(p.top, x), base = base_of(top);
  p.sum = p.sum * exp2_of((p.top - base) * scale) + exp2_of((x - base) * scale);
  p.top = top;
}

// C parts over the workgroup of at most 16 waves, in every thread; `share` holds 2 C * 16 floats.  Parts from c = 1 on
// come from the first `few` waves alone.  The waves' shares lie in 16 lanes each for the second step.
template <int C>
__device__ __forceinline__ void block_part(PartSum (&p)[C], float scale, float *share, int few = 16) {
  const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6;
#pragma unroll
  for (int c = 0; c < C; ++c)
    if (c == 0 || wave < few) p[c] = wave_part(p[c], scale);
  if (waves == 1) return;
  float2 *all = reinterpret_cast<float2 *>(share);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int c = 0; c < C; ++c) all[c * 16 + wave] = make_float2(p[c].top, p[c].sum);
  __syncthreads();
  const int l = threadIdx.x & 15;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    const float2 v = l < waves ? all[c * 16 + l] : make_float2(-INFINITY, 0.0f);
    const float top = reduce16(v.x, [](float a, float b) { return fmaxf(a, b); });
    p[c] = {top, reduce16(v.y * exp2_of((v.x - base_of(top)) * scale), [](float a, float b) { return a + b; })};
  }
}

}  // namespace fly
