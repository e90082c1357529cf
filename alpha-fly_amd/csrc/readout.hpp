// What the two ways of the read-out loss share: its arguments, targets and rows.
#pragma once

#include "readout_rules.hpp"
#include "rows.hpp"

namespace fly {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Targets {
  const void *index;
  int wide;               // index of 8 bytes
  const float *weight;    // null: 1
  int k;
  const uint8_t *legal;
  int64_t ldl;
  int cols;
};
__device__ __forceinline__ int64_t target_at(const Targets &t, int64_t at) {
  return t.wide ? static_cast<const int64_t *>(t.index)[at] : static_cast<const int32_t *>(t.index)[at];
}
// Whether entry j of a row counts: -1 none, -2 it lies past the columns, else its column.
__device__ __forceinline__ int target_of(const Targets &t, int64_t row, int j, float &weight) {
  const int64_t c = target_at(t, row * t.k + j);
  weight = t.weight ? t.weight[row * t.k + j] : 1.0f;
  if (c < 0 || weight == 0.0f) return -1;
  if (c >= t.cols) return -2;
  return t.legal && !t.legal[row * t.ldl + c] ? -1 : (int)c;
}

struct Given {
  const void *x, *w, *bias;
  int64_t ldx, ldw;
  int32_t bias_type;
  Targets targets;
  const float *row_scale;
  float grad_scale;
  float *loss;
  void *gx, *gw, *gb;
  int64_t ldgx, ldgw;
};

// Piece i of a row of `cols` as it lies in memory, zeros past its end.
template <typename T>
__device__ __forceinline__ Raw16 load_raw(const T *__restrict__ row, int i, int64_t cols) {
  constexpr int N = Piece<T>::N;
  if ((int64_t)i * N + N <= cols) return load_whole(row, i);
  Raw16 p = {};
#pragma unroll
  for (int e = 0; e < N - 1; ++e)
    if ((int64_t)i * N + e < cols) {
      const uint32_t b = to_bits(row[(int64_t)i * N + e]);
      if constexpr (sizeof(T) == 4) p.v[e] = b;
      else p.v[e / 2] |= b << (16 * (e & 1));
    }
  return p;
}

// The same in two steps, for loads that are to be in flight together: with a branch around its tail, each load is waited for where
// the branches meet.  Rows have a whole piece at least; a piece past the end holds the row's last elements until it is settled.
template <typename T>
__device__ __forceinline__ Raw16 load_clamped(const T *__restrict__ row, int i, int cols) {
  return *reinterpret_cast<const Raw16 *>(row + min(i * Piece<T>::N, cols - Piece<T>::N));
}
template <typename T>
__device__ __forceinline__ void settle(Raw16 &p, int i, int cols) {
  const int past = i * Piece<T>::N + Piece<T>::N - cols;   // elements
  if (past <= 0) return;
  const int bits = past * 8 * (int)sizeof(T);
  uint64_t lo = p.v[0] | (uint64_t)p.v[1] << 32, hi = p.v[2] | (uint64_t)p.v[3] << 32;
  if (bits >= 128) lo = hi = 0;
  else if (bits >= 64) lo = hi >> (bits - 64), hi = 0;
  else lo = lo >> bits | hi << (64 - bits), hi >>= bits;
  p.v[0] = (uint32_t)lo;
  p.v[1] = (uint32_t)(lo >> 32);
  p.v[2] = (uint32_t)hi;
  p.v[3] = (uint32_t)(hi >> 32);
}

// The sum or maximum over the four lanes that hold a row of a matrix instruction's result (lane & 15 alike), in each of them.
template <typename F>
__device__ __forceinline__ float over_four(float x, F &&f) {
  const auto h = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
  x = f(__int_as_float(h[0]), __int_as_float(h[1]));
  const auto w = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
  return f(__int_as_float(w[0]), __int_as_float(w[1]));
}

__device__ __forceinline__ float bias_at(const void *bias, int type, int64_t c) {
  if (type == FLY_F32) return static_cast<const float *>(bias)[c];
  if (type == FLY_F16) return static_cast<float>(static_cast<const _Float16 *>(bias)[c]);
  return static_cast<float>(static_cast<const bhalf *>(bias)[c]);
}

template <typename F>
inline void by_type(int32_t type, const char *what, F &&f) {
  switch (type) {
    case FLY_F32: f(float{}); break;
    case FLY_F16: f(_Float16{}); break;
    case FLY_BF16: f(bhalf{}); break;
    default: FLY_REQUIRE(false, what);
  }
}

// Few rows, without laying the operands out (readout_few.hip): what a call takes, and the call.
size_t few_ws(const Call &c);
void run_few(const Call &c, const Given &g, char *ws, hipStream_t st);

}  // namespace fly
