// Matrix product in 8-bit integers with a scale for each token (row of x) and channel (row of w).
//
//   a_m = max_k |x_mk|,  s_m = a_m / 127,  q_mk = rint(x_mk (127 / a_m))      (each step rounded to float32)
//   y_mn = (sum_k q_mk w_nk) (s_m t_n) + b_n
// The products sum exactly in int32 (k below 2^17 keeps 127 * 127 * k below 2^31) and are scaled in float32.  A row that
// holds an infinity or NaN has the scale NaN, so its outputs are NaN; a row below 2^-120 everywhere counts as zero.
//
// Both operands lie in blocks of 16 rows x 64 k, in the order in which the matrix cores take them: 1 KB, lane l's 16
// bytes at 16 l hold row l & 15, k 16 (l >> 4) .. + 15.  A wave loads a block as one contiguous kilobyte, from memory or
// LDS, without bank conflicts.  Weights are laid out once, in the plan; tokens by the kernel that quantises them.
#include "rows.hpp"

#include <cmath>

struct fly_int8 {
  int device = -1;
  int64_t n = 0, k = 0, nb = 0, kb = 0;   // channels and k, and their blocks of 16 and 64
  fly::DevArray<uint32_t> w;              // nb x kb blocks of 256 words
  fly::DevArray<float> scale, bias;       // 16 nb each, zero past n
};

namespace fly {
namespace {

typedef int int4v __attribute__((ext_vector_type(4)));
constexpr int64_t kMostK = 1 << 17;

// Where 16-byte piece c (k 16 c .. + 15) of row r lies among the blocks.
__device__ __forceinline__ int64_t block_piece(int64_t r, int64_t c, int64_t kb) {
  return (((r >> 4) * kb + (c >> 2)) << 6) + ((c & 3) << 4) + (r & 15);
}

// int8 rows into blocks, zero past k and past the rows; one thread per 16-byte piece.
__global__ __launch_bounds__(256) void k_int8_pack(const int8_t *__restrict__ src, int64_t ld, int64_t rows, int64_t k,
                                                   int64_t kb, int64_t pieces, int4v *__restrict__ out) {
  const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (i >= pieces) return;
  const int64_t r = i / (4 * kb), c = i - r * 4 * kb;
  uint32_t w[4] = {0, 0, 0, 0};
  if (r < rows)
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (16 * c + e < k) w[e / 4] |= (uint32_t)(uint8_t)src[r * ld + 16 * c + e] << (8 * (e & 3));
  out[block_piece(r, c, kb)] = int4v{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
}

// max |v| of a row piece into a running maximum that keeps NaN
__device__ __forceinline__ float abs_max(float m, float v) {
  const float x = fabsf(v);
  return x > m || x != x ? x : m;
}

struct RowScale {
  float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale(float top) {
  RowScale s;
  if (!(top <= 3.4028234663852886e38f)) {   // an infinity or NaN
    s.scale = __builtin_nanf("");
    s.inverse = 0.0f;
  } else if (top < 7.5231638452626401e-37f) {   // 2^-120: 127 / top may overflow
    s.scale = s.inverse = 0.0f;
  } else {
    s.scale = top / 127.0f;
    s.inverse = 127.0f / top;
  }
  return s;
}
// rint(v * inverse) as the low byte; 0 for the infinities and NaN of a row whose inverse is 0
__device__ __forceinline__ uint32_t quantised(float v, float inverse) {
  const float q = inverse == 0.0f ? 0.0f : rintf(v * inverse);
  return (uint32_t)(int)q & 0xffu;
}

// A wave per row.  PACKED: into blocks, zero past k; else row-major bytes at ldq.
template <typename T, bool PACKED>
__global__ __launch_bounds__(256) void k_quantize(const T *__restrict__ x, int64_t ldx, int64_t rows, int64_t k,
                                                  int64_t kb, int8_t *__restrict__ q, int64_t ldq,
                                                  float *__restrict__ scale) {
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const T *xr = x + row * ldx;
  constexpr int N = Piece<T>::N;
  float top = 0.0f;
  for (int64_t i = lane; i * N < k; i += 64) {
    const Piece<T> p = load_piece(xr, i, k, 0.0f);
#pragma unroll
    for (int e = 0; e < N; ++e) top = abs_max(top, p.v[e]);
  }
  top = wave_reduce(top, [](float a, float b) { return nan_max(a, b); });
  const RowScale s = row_scale(top);
  if (lane == 0) scale[row] = s.scale;
  const int64_t chunks = PACKED ? 4 * kb : (k + 15) / 16;
  for (int64_t c = lane; c < chunks; c += 64) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16 / N; ++j) {
      const int64_t i = c * (16 / N) + j;
      if (i * N >= k) continue;
      const Piece<T> p = load_piece(xr, i, k, 0.0f);
#pragma unroll
      for (int e = 0; e < N; ++e) w[(j * N + e) / 4] |= quantised(p.v[e], s.inverse) << (8 * (e & 3));
    }
    if constexpr (PACKED) {
      reinterpret_cast<int4v *>(q)[block_piece(row, c, kb)] = int4v{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    } else {
      for (int e = 0; e < 16; ++e)
        if (16 * c + e < k) q[row * ldq + 16 * c + e] = (int8_t)(w[e / 4] >> (8 * (e & 3)));
    }
  }
}

// One wave: 16 tokens x 64 channels, fragments straight from the blocks.
template <typename T>
__global__ __launch_bounds__(256) void k_int8_gemm(const int4v *__restrict__ w, const int4v *__restrict__ q,
                                                   const float *__restrict__ row_scale,
                                                   const float *__restrict__ scale, const float *__restrict__ bias,
                                                   int64_t rows, int64_t n, int64_t nb, int64_t kb, T *__restrict__ y,
                                                   int64_t ldy) {
  const int lane = threadIdx.x & 63;
  const int64_t nb0 = (blockIdx.x * (int64_t)4 + (threadIdx.x >> 6)) * 4, mb = blockIdx.y;
  if (nb0 >= nb) return;
  int4v acc[4] = {};
  for (int64_t b = 0; b < kb; ++b) {
    const int4v fq = q[((mb * kb + b) << 6) + lane];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int4v fw = w[((min(nb0 + j, nb - 1) * kb + b) << 6) + lane];
      acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw, fq, acc[j], 0, 0, 0);
    }
  }
  const int64_t m = 16 * mb + (lane & 15);
  if (m >= rows) return;
  const float sm = row_scale[m];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t c = 16 * (nb0 + j) + 4 * (lane >> 4) + r;
      if (c < n) y[m * ldy + c] = static_cast<T>((float)acc[j][r] * (sm * scale[c]) + bias[c]);
    }
}

template <typename F>
void by_float(int32_t type, const char *what, F &&f) {
  switch (type) {
    case FLY_F32: f(float{}); break;
    case FLY_F16: f(_Float16{}); break;
    case FLY_BF16: f(bhalf{}); break;
    default: FLY_REQUIRE(false, what);
  }
}

void pack(const int8_t *src, int64_t ld, int64_t rows, int64_t k, int64_t kb, void *out, hipStream_t st) {
  const int64_t pieces = round_up(rows, 16) * 4 * kb;
  FLY_REQUIRE(pieces / 256 < INT32_MAX, "operand too large");
  hipLaunchKernelGGL(k_int8_pack, dim3(blocks_for(pieces, 256)), dim3(256), 0, st, src, ld, rows, k, kb, pieces,
                     static_cast<int4v *>(out));
  check_launch("8-bit blocks");
}

size_t token_bytes(const fly_int8 &p, int64_t rows) { return (size_t)round_up(rows, 16) * p.kb * 64; }

size_t int8_ws(const fly_int8 &p, int64_t rows) {
  return align256(token_bytes(p, rows)) + align256((size_t)rows * sizeof(float));
}

}  // namespace
}  // namespace fly

using namespace fly;

extern "C" int fly_quantize_rows(const void *x, int32_t x_type, int64_t ldx, int64_t rows, int64_t cols, int8_t *q,
                                 int64_t ldq, float *scale, void *stream) {
  return guard([&] {
    FLY_REQUIRE(rows >= 0 && cols >= 0 && rows < (int64_t)INT32_MAX && ldx >= cols && ldq >= cols, "bad size");
    FLY_REQUIRE(!rows || (scale && (!cols || (x && q))), "null pointer");
    by_float(x_type, "x must be float32, float16 or bfloat16", [&](auto t) {
      using T = decltype(t);
      if (!rows) return;
      hipLaunchKernelGGL((k_quantize<T, false>), dim3(blocks_for(rows, 4)), dim3(256), 0, as_stream(stream),
                         static_cast<const T *>(x), ldx, rows, cols, (int64_t)0, q, ldq, scale);
      check_launch("quantised rows");
    });
  });
}

extern "C" int fly_int8_create(const int8_t *w, int64_t ldw, const float *scale, const float *bias, int64_t n,
                               int64_t k, void *stream, fly_int8 **out) {
  return guard([&] {
    FLY_REQUIRE(out != nullptr, "out is null");
    *out = nullptr;
    FLY_REQUIRE(n >= 1 && k >= 1 && k < kMostK && n < (int64_t)INT32_MAX && ldw >= k, "bad size");
    FLY_REQUIRE(w && scale, "null pointer");
    hipStream_t st = as_stream(stream);
    auto p = std::make_unique<fly_int8>();
    p->device = current_device();
    p->n = n;
    p->k = k;
    p->nb = (n + 15) / 16;
    p->kb = (k + 63) / 64;
    p->w.alloc((size_t)p->nb * p->kb * 256);
    pack(w, ldw, n, k, p->kb, p->w.p, st);
    p->scale.alloc((size_t)p->nb * 16);
    p->bias.alloc((size_t)p->nb * 16);
    FLY_HIP(hipMemsetAsync(p->scale.p, 0, p->nb * 16 * sizeof(float), st));
    FLY_HIP(hipMemsetAsync(p->bias.p, 0, p->nb * 16 * sizeof(float), st));
    FLY_HIP(hipMemcpyAsync(p->scale.p, scale, n * sizeof(float), hipMemcpyDeviceToDevice, st));
    if (bias) FLY_HIP(hipMemcpyAsync(p->bias.p, bias, n * sizeof(float), hipMemcpyDeviceToDevice, st));
    FLY_HIP(hipStreamSynchronize(st));
    *out = p.release();
  });
}

extern "C" int fly_int8_destroy(fly_int8 *p) {
  return guard([&] { delete p; });
}

extern "C" size_t fly_int8_workspace(const fly_int8 *p, int64_t rows) { return p && rows > 0 ? int8_ws(*p, rows) : 0; }

extern "C" int fly_int8_linear(const fly_int8 *p, const void *x, int32_t x_type, int64_t ldx, const float *x_scale,
                               int64_t rows, void *y, int32_t y_type, int64_t ldy, void *ws, size_t ws_bytes,
                               void *stream) {
  return guard([&] {
    FLY_REQUIRE(p != nullptr, "the 8-bit plan is null");
    FLY_REQUIRE(current_device() == p->device, "the 8-bit plan lives on another device");
    FLY_REQUIRE(rows >= 0 && rows < (int64_t)65535 * 16, "rows out of range");
    FLY_REQUIRE((x_type == FLY_I8) == (x_scale != nullptr), "8-bit rows come with their scales, other rows without");
    if (!rows) return;
    FLY_REQUIRE(x && y && ldx >= p->k && ldy >= p->n, "bad argument");
    FLY_REQUIRE(ws && ws_bytes >= int8_ws(*p, rows) && aligned(ws, 256), "workspace too small or misaligned");
    hipStream_t st = as_stream(stream);
    float *made = reinterpret_cast<float *>(static_cast<char *>(ws) + align256(token_bytes(*p, rows)));
    if (x_type == FLY_I8) {
      pack(static_cast<const int8_t *>(x), ldx, rows, p->k, p->kb, ws, st);
    } else {
      by_float(x_type, "x must be float32, float16, bfloat16 or int8", [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((k_quantize<T, true>), dim3(blocks_for(rows, 4)), dim3(256), 0, st,
                           static_cast<const T *>(x), ldx, rows, p->k, p->kb, static_cast<int8_t *>(ws), (int64_t)0,
                           made);
        check_launch("quantised tokens");
      });
    }
    by_float(y_type, "y must be float32, float16 or bfloat16", [&](auto t) {
      using T = decltype(t);
      hipLaunchKernelGGL(k_int8_gemm<T>, dim3(blocks_for(p->nb, 16), blocks_for(rows, 16)), dim3(256), 0, st,
                         reinterpret_cast<const int4v *>(p->w.p), static_cast<const int4v *>(ws),
                         x_scale ? x_scale : made, p->scale.p, p->bias.p, rows, p->n, p->nb, p->kb,
                         static_cast<T *>(y), ldy);
      check_launch("8-bit product");
    });
  });
}
