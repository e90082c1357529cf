// Softmax cross entropy of a read-out and its gradients, without keeping the logits.
//
//   z_rv = sum_d x_rd w_vd + b_v over the row's visible columns,   p_r = softmax(z_r)
//   loss_r = sum_j a_rj (log sum_v exp z_rv - z_r,t_rj)            a list of targets t with weights a; one with weight 1
//   u_rv = (A_r p_rv - sum_{j: t_rj = v} a_rj) / B_r               A = sum_j a, B = sum_j |a|: |u| <= 2 whatever the weights
//   dx_r = f_r sum_v u_rv w_v,  dw_v = sum_r f_r u_rv x_r,  db_v = sum_r f_r u_rv,   f = B row_scale grad_scale
//
// Rows run in pieces whose logits and u fit a bounded workspace.
#include "blocks.hpp"

#include <cmath>

namespace fly {
namespace {

constexpr float kUnit = 16384.0f;            // u is multiplied as 2^14 u: float16 then holds it from 2^-28 on without loss
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int64_t kPieceBytes = (int64_t)1 << 31;   // of a piece of rows: its logits, u, and x laid out
constexpr int64_t kPieceRows = (int64_t)1 << 19;    // a piece at most: tiles of rows are counted in 16 bits

// Maxima over all rows that the scales of products over rows are taken by: bits of floats that are not negative.
struct Maxima {
  uint32_t weight, row;
};
__device__ __forceinline__ void raise(uint32_t *to, float v) {
  if (v > 0.0f && v <= 3.4028234663852886e38f) atomicMax(to, __float_as_uint(v));
}

__global__ void k_clear(Maxima *m) { *m = Maxima{0u, 0u}; }
__global__ void k_clear_row(Maxima *m) { m->row = 0u; }

// ---- targets ---------------------------------------------------------------------------------------------------------

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

// ---- operands into blocks --------------------------------------------------------------------------------------------

// 2^e with max |row| 2^e in [2^13, 2^14) for rows held as two halves, and its inverse; 1 of a row of zeros or with infinities.
__device__ __forceinline__ float unit_of(float top) {
  if (!(top > 0.0f) || !(top <= 3.4028234663852886e38f)) return 1.0f;
  int e;
  (void)frexpf(top, &e);                  // top = m 2^e, m in [1/2, 1)
  return ldexpf(1.0f, max(e - 14, -120));
}

template <typename T>
struct Lay {
  const T *src;
  int64_t ld, rows, cols;
  int kb, kt;             // blocks of 32 columns, and of 32 rows
  int4v *out, *turned;    // (rows, columns), and (columns, rows) or null
  float *unit;            // of two planes: each row's
  uint32_t *top;          // the largest unit, or null
  const void *bias;
  int bias_type;
  float *bias_out;        // bias as float32, or null: no bias wanted
  Targets targets;        // of the rows (index null: none): one without any left counts as zeros, whatever it holds
};

constexpr int kSlab = 512;   // columns that pass through LDS at a time

// 16 rows, a wave each; rows past the last are zero.
template <typename T>
__global__ __launch_bounds__(1024) void k_lay(const Lay<T> o) {
  using H = typename Multiplied<T>::H;
  constexpr int P = Multiplied<T>::P, N = Piece<T>::N, PIECES = kSlab / (64 * N);
  __shared__ __attribute__((aligned(16))) uint16_t lds[P][16][kSlab + 8];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), group = blockIdx.x;
  const int64_t row = (int64_t)group * 16 + wave;
  bool in = row < o.rows;
  const T *src = o.src + (in ? row : 0) * o.ld;
  if (in && o.targets.index) {
    bool some = false;
    for (int j = lane; j < o.targets.k; j += 64) {
      float a;
      some |= target_of(o.targets, row, j, a) != -1;
    }
    in = __ballot(some) != 0;
  }
  float unit = 1.0f;
  if constexpr (P == 2) {
    float top = 0.0f;
    if (in)
      for (int64_t i = lane; i * N < o.cols; i += 64) {
        const Piece<T> p = load_piece(src, i, o.cols, 0.0f);
#pragma unroll
        for (int e = 0; e < N; ++e) top = __builtin_elementwise_maximum(top, fabsf(p.v[e]));
      }
    unit = unit_of(wave_reduce(top, [](float a, float b) { return nan_max(a, b); }));
    if (lane == 0) {
      o.unit[row] = unit;
      if (in && o.top) raise(o.top, unit);
    }
  }
  if (o.bias_out && lane == 0) {
    float b = 0.0f;
    if (in && o.bias) {
      if (o.bias_type == FLY_F32) b = static_cast<const float *>(o.bias)[row];
      else if (o.bias_type == FLY_F16) b = static_cast<float>(static_cast<const _Float16 *>(o.bias)[row]);
      else b = static_cast<float>(static_cast<const bhalf *>(o.bias)[row]);
    }
    o.bias_out[row] = b;
  }
  const float inverse = 1.0f / unit;
  for (int first = 0; first < o.kb * 32; first += kSlab) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int at = (lane + 64 * j) * N;
      Piece<T> p;
      if (in && first + at < o.cols) p = load_piece(src, (first + at) / N, o.cols, 0.0f);
      else
#pragma unroll
        for (int e = 0; e < N; ++e) p.v[e] = 0.0f;
#pragma unroll
      for (int e = 0; e < N; e += 2) {
        uint32_t a[P], b[P];
        planes_of<H, P>(P == 2 ? p.v[e] * inverse : p.v[e], a);
        planes_of<H, P>(P == 2 ? p.v[e + 1] * inverse : p.v[e + 1], b);
#pragma unroll
        for (int q = 0; q < P; ++q) *reinterpret_cast<uint32_t *>(&lds[q][wave][at + e]) = a[q] | b[q] << 16;
      }
    }
    __syncthreads();
    const int k = first / 32 + wave;
    if (k < o.kb) {
#pragma unroll
      for (int q = 0; q < P; ++q)
        o.out[(((int64_t)group * o.kb + k) * P + q) * 64 + lane] =
            *reinterpret_cast<const int4v *>(&lds[q][lane & 15][32 * wave + 8 * (lane >> 4)]);
      if (o.turned) {
        const int at = 32 * wave + 16 * (lane >> 5) + (lane & 15), eight = (lane >> 4) & 1;
        const int64_t block = ((int64_t)2 * k + (lane >> 5)) * o.kt + (group >> 1);
#pragma unroll
        for (int q = 0; q < P; ++q) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = lds[q][8 * eight + 2 * e][at] | (uint32_t)lds[q][8 * eight + 2 * e + 1][at] << 16;
          o.turned[(block * P + q) * 64 + 16 * (2 * (group & 1) + eight) + (lane & 15)] =
              int4v{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
        }
      }
    }
    __syncthreads();
  }
}

// ---- logits ----------------------------------------------------------------------------------------------------------

// Logits of a piece of rows, with each row's maximum and sum over a wave's columns.
struct LogitsOut {
  const float *unit_m, *unit_n;   // or null
  const float *bias;
  const uint8_t *legal;
  int64_t ldl;
  int rows, cols;
  float *z;
  int64_t ldz;
  float2 *parts;      // (column part, row)
  int64_t ld_parts;
  template <int FN, int FM>
  __device__ __forceinline__ void tile(float4v (&acc)[FN][FM], int m0, int n0, int lane, int part, float *turn) const {
    const int quad = 4 * (lane >> 4);
    float4v b[FN], un[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int c = n0 + 16 * j + quad;
      b[j] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
      un[j] = float4v{1.0f, 1.0f, 1.0f, 1.0f};
      if (c < cols) {   // the arrays are padded to a multiple of 32
        b[j] = *reinterpret_cast<const float4v *>(bias + c);
        if (unit_n) un[j] = *reinterpret_cast<const float4v *>(unit_n + c);
      }
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + 16 * i + (lane & 15);
      const float um = unit_m && m < rows ? unit_m[m] : 1.0f;
      const uint8_t *seen = legal && m < rows ? legal + m * ldl : nullptr;
      float4v v[FN];
      PartSum p{-INFINITY, 0.0f};
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int c = n0 + 16 * j + quad;
        float l[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // a load for each column, of one that is there where this one is not: no branch around each
          const uint8_t shown = seen ? seen[min(c + e, cols - 1)] : 1;
          const float x = (unit_n ? acc[j][i][e] * um * un[j][e] : acc[j][i][e]) + b[j][e];
          l[e] = c + e < cols && shown ? x : -INFINITY;
          p.top = fmaxf(p.top, l[e]);
        }
        v[j] = float4v{l[0], l[1], l[2], l[3]};
      }
      // over the four lanes of the row
      auto four = [](float x, auto &&f) {
        const auto h = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
        x = f(__int_as_float(h[0]), __int_as_float(h[1]));
        const auto w = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
        return f(__int_as_float(w[0]), __int_as_float(w[1]));
      };
      p.top = four(p.top, [](float x, float y) { return fmaxf(x, y); });
      const float base = base_of(p.top);
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) p.sum += exp2_of((v[j][e] - base) * kLog2e);
      p.sum = four(p.sum, [](float x, float y) { return x + y; });
      if (lane < 16 && m < rows) parts[part * ld_parts + m] = make_float2(p.top, p.sum);
      turn_over<FN>(v, turn, lane, [&](int row, int c, const float4v &four_) {
        const int mm = m0 + 16 * i + row;
        if (mm < rows && n0 + c < ldz) *reinterpret_cast<float4v *>(z + mm * ldz + n0 + c) = four_;
      });
    }
  }
};

// ---- rows ------------------------------------------------------------------------------------------------------------

// What a row's gradient is made of: p = exp2((z - top) log2 e - log_sum), u = share p - a / whole.
struct RowInfo {
  float top, log_sum, share, whole;
};

// A wave per row.
__global__ __launch_bounds__(256) void k_loss_rows(const float2 *__restrict__ parts, int64_t ld_parts, int count, int rows,
                                                   const Targets t, const float *__restrict__ z, int64_t ldz,
                                                   const float *__restrict__ unit, const float *__restrict__ row_scale,
                                                   float grad_scale, float *__restrict__ loss, RowInfo *__restrict__ info,
                                                   float *__restrict__ factor, float *__restrict__ turned_factor,
                                                   uint32_t *__restrict__ most) {
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  PartSum p{-INFINITY, 0.0f};
  for (int i = lane; i < count; i += 64) {
    const float2 v = parts[i * ld_parts + row];
    const float top = fmaxf(p.top, v.x), base = base_of(top);
    p.sum = p.sum * exp2_of((p.top - base) * kLog2e) + v.y * exp2_of((v.x - base) * kLog2e);
    p.top = top;
  }
  p = wave_part(p, kLog2e);
  const float log_sum = log2_of(p.sum);
  float sum = 0.0f, share = 0.0f, whole = 0.0f;
  for (int j = lane; j < t.k; j += 64) {
    float a;
    const int c = target_of(t, row, j, a);
    if (c == -1) continue;
    const float far = c == -2 ? __builtin_nanf("") : (p.top - z[row * ldz + c]) + kLn2 * log_sum;
    sum += a * far;
    share += c == -2 ? __builtin_nanf("") : a;
    whole += fabsf(a);
  }
  sum = wave_sum(sum);
  share = wave_sum(share);
  whole = wave_sum(whole);
  if (lane) return;
  const bool some = whole != 0.0f;   // NaN too
  if (loss) loss[row] = some ? sum : 0.0f;
  if (!info) return;
  info[row] = RowInfo{base_of(p.top), log_sum, some ? share / whole : 0.0f, whole};
  const float f = some ? whole * (row_scale ? row_scale[row] : 1.0f) * grad_scale : 0.0f, ft = unit ? f * unit[row] : f;
  factor[row] = f;
  turned_factor[row] = ft;
  raise(most, fabsf(ft));
}

// ---- the logits' gradient --------------------------------------------------------------------------------------------

constexpr int kGradRows = 64, kGradCols = 128, kGradPitch = 130;

// u of 64 rows x 128 columns into blocks, by rows (times the columns' units) and turned (times the rows' factors), and its
// columns' sums.
template <typename H, int P>
__global__ __launch_bounds__(256) void k_logits_grad(const float *__restrict__ z, int64_t ldz, int rows, const Targets t,
                                                     const RowInfo *__restrict__ info, const float *__restrict__ factor,
                                                     const float *__restrict__ turned_factor,
                                                     const float *__restrict__ unit_n, const Maxima *__restrict__ maxima,
                                                     int rb, int vb, int4v *__restrict__ out, int4v *__restrict__ turned,
                                                     float *__restrict__ sums, int64_t ld_sums) {
  __shared__ __attribute__((aligned(16))) float u[kGradRows][kGradPitch];
  __shared__ float col_sum[2][kGradCols], f_row[kGradRows], ft_row[kGradRows], un_col[kGradCols];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c0 = blockIdx.x * kGradCols, r0 = blockIdx.y * kGradRows, cols = t.cols;
  if (tid < kGradRows) {
    const int r = r0 + tid;
    const float most = __uint_as_float(maxima->row);
    f_row[tid] = r < rows ? factor[r] : 0.0f;
    ft_row[tid] = r < rows && most > 0.0f ? turned_factor[r] / most * kUnit : 0.0f;
  }
  if (tid >= 128) {
    const int c = c0 + tid - 128;
    un_col[tid - 128] = P == 2 && c < cols ? unit_n[c] / __uint_as_float(maxima->weight) * kUnit : kUnit;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = (tid >> 5) + 8 * i, c = 4 * (tid & 31);
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (r0 + r < rows && c0 + c < cols) {
      const RowInfo f = info[r0 + r];
      const float4v at = *reinterpret_cast<const float4v *>(z + (int64_t)(r0 + r) * ldz + c0 + c);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c0 + c + e < cols && f.share != 0.0f) v[e] = f.share * exp2_of((at[e] - f.top) * kLog2e - f.log_sum);
    }
    *reinterpret_cast<float2 *>(&u[r][c]) = make_float2(v[0], v[1]);
    *reinterpret_cast<float2 *>(&u[r][c + 2]) = make_float2(v[2], v[3]);
  }
  __syncthreads();
  {
    // the targets of a row, in their order, a thread for each quarter of its columns
    const int r = tid & 63, q0 = c0 + 32 * (tid >> 6);
    if (r0 + r < rows && info[r0 + r].whole != 0.0f) {
      const float whole = info[r0 + r].whole;
      for (int j = 0; j < t.k; ++j) {
        float a;
        const int64_t c = target_at(t, (int64_t)(r0 + r) * t.k + j);
        if (c >= q0 && c < q0 + 32 && target_of(t, r0 + r, j, a) >= 0) u[r][c - c0] -= a / whole;
      }
    }
  }
  __syncthreads();
  typedef uint32_t words[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = wave * 4 + i, rg = b >> 2, cg = b & 3;   // 16 rows, 32 columns
    const int gr = (r0 >> 4) + rg, gc = (c0 >> 5) + cg;
    if (out && gr < rb && gc < vb) {
      const int r = 16 * rg + (lane & 15), c = 32 * cg + 8 * (lane >> 4);
      words w[P];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 v = *reinterpret_cast<const float2 *>(&u[r][c + 2 * e]);
        uint32_t a[P], d[P];
        planes_of<H, P>(v.x * un_col[c + 2 * e], a);
        planes_of<H, P>(v.y * un_col[c + 2 * e + 1], d);
#pragma unroll
        for (int q = 0; q < P; ++q) w[q][e] = a[q] | d[q] << 16;
      }
#pragma unroll
      for (int q = 0; q < P; ++q)
        out[(((int64_t)gr * vb + gc) * P + q) * 64 + lane] = int4v{(int)w[q][0], (int)w[q][1], (int)w[q][2], (int)w[q][3]};
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = wave * 4 + i, cg = b >> 1, rg = b & 1;   // 16 columns, 32 rows
    const int gc = (c0 >> 4) + cg, gr = (r0 >> 5) + rg;
    if (turned && gc < 2 * vb && 2 * gr < rb) {
      const int c = 16 * cg + (lane & 15), r = 32 * rg + 8 * (lane >> 4);
      words w[P];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        uint32_t a[P], d[P];
        planes_of<H, P>(u[r + 2 * e][c] * ft_row[r + 2 * e], a);
        planes_of<H, P>(u[r + 2 * e + 1][c] * ft_row[r + 2 * e + 1], d);
#pragma unroll
        for (int q = 0; q < P; ++q) w[q][e] = a[q] | d[q] << 16;
      }
#pragma unroll
      for (int q = 0; q < P; ++q)
        turned[(((int64_t)gc * (rb / 2) + gr) * P + q) * 64 + lane] =
            int4v{(int)w[q][0], (int)w[q][1], (int)w[q][2], (int)w[q][3]};
    }
  }
  if (!sums) return;
  const int c = tid & 127, half = tid >> 7;
  float s = 0.0f;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) s = fmaf(u[32 * half + r][c], f_row[32 * half + r], s);
  col_sum[half][c] = s;
  __syncthreads();
  if (half == 0 && c0 + c < cols) sums[blockIdx.y * ld_sums + c0 + c] = s + col_sum[1][c];
}

// The columns' sums over all tiles of rows, after what earlier pieces of rows gave.
template <typename T>
__global__ __launch_bounds__(256) void k_bias_grad(const float *__restrict__ sums, int64_t ld_sums, int tiles, int cols,
                                                   const float *__restrict__ before, float *__restrict__ after,
                                                   T *__restrict__ out) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float s = before ? before[c] : 0.0f;
  for (int i = 0; i < tiles; ++i) s += sums[i * ld_sums + c];
  if (after) after[c] = s;
  else out[c] = static_cast<T>(s);
}

// ---- gradients -------------------------------------------------------------------------------------------------------

// out[m][n] = sum * row[m] * *scale / 2^14, after what earlier pieces of rows gave.
template <typename T>
struct GradOut {
  const float *row;          // or null
  const uint32_t *scale;     // a maximum's bits, or null
  int rows, cols;
  const float *before;
  float *after;              // or null: the last piece, into out
  int64_t ld_sum;
  T *out;
  int64_t ld;
  template <int FN, int FM>
  __device__ __forceinline__ void tile(float4v (&acc)[FN][FM], int m0, int n0, int lane, int, float *turn) const {
    const float s = (scale ? __uint_as_float(*scale) : 1.0f) / kUnit;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      float4v v[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) v[j] = acc[j][i];
      turn_over<FN>(v, turn, lane, [&](int r, int c, const float4v &four) {
        const int m = m0 + 16 * i + r, n = n0 + c;
        if (m >= rows || n >= cols) return;
        const float f = row ? s * row[m] : s;
        float4v w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = four[e] * f;
        if (before) w += *reinterpret_cast<const float4v *>(before + m * ld_sum + n);
        if (after) {
          *reinterpret_cast<float4v *>(after + m * ld_sum + n) = w;
          return;
        }
        struct __attribute__((packed, aligned(sizeof(T)))) Four {
          T v[4];
        };
        T *to = out + m * ld + n;
        if (n + 4 <= cols)
          *reinterpret_cast<Four *>(to) =
              Four{{static_cast<T>(w[0]), static_cast<T>(w[1]), static_cast<T>(w[2]), static_cast<T>(w[3])}};
        else
#pragma unroll
          for (int e = 0; e < 3; ++e)
            if (n + e < cols) to[e] = static_cast<T>(w[e]);
      });
    }
  }
};

template <typename T>
__global__ __launch_bounds__(256) void k_zeros(T *__restrict__ out, int64_t ld, int64_t rows, int64_t cols) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
    out[i / cols * ld + i % cols] = static_cast<T>(0.0f);
}

// ---- the call --------------------------------------------------------------------------------------------------------

struct Call {
  int32_t type;
  int64_t rows, d, v;
  bool gx, gw, gb;
  bool grads() const { return gx || gw || gb; }
};

template <typename H, int P, typename EP>
void product(const Blocks &o, const EP &ep, hipStream_t st) {
  if constexpr (P == 1) launch_blocks<H, P, 2, 4, 4, 2, 4>(o, ep, st);
  else launch_blocks<H, P, 2, 4, 4, 2, 3>(o, ep, st);
}
constexpr int kTileN = 128, kPartN = 64;

// Where everything lies in the workspace.
struct Space {
  int64_t piece;      // rows at a time
  int64_t db, vb, rb; // blocks of 32
  int parts;
  bool several;
  size_t x, xt, w, wt, z, g, gt, unit_x, unit_w, bias, stat, info, factor, turned, sums, maxima, acc_w, acc_b, bytes;
  Space(const Call &c, int planes) {
    db = (c.d + 31) / 32;
    vb = (c.v + 31) / 32;
    parts = (int)((vb * 32 + kTileN - 1) / kTileN * (kTileN / kPartN));
    const int64_t each = vb * 32 * (4 + 2 * planes * ((c.gx ? 1 : 0) + (c.gw ? 1 : 0))) + db * 64 * planes * (c.gw ? 2 : 1);
    piece = std::min({round_up(c.rows, 64), std::max<int64_t>(kPieceBytes / each / 64 * 64, 64), kPieceRows});
    several = piece < c.rows;
    rb = piece / 32;
    size_t at = 0;
    auto take = [&](int64_t n) {
      const size_t was = at;
      at += align256((size_t)n);
      return was;
    };
    const int64_t block = 2048 * planes;   // of 32 x 32
    x = take(rb * db * block);
    xt = c.gw ? take(rb * db * block) : 0;
    w = take(vb * db * block);
    wt = c.gx ? take(vb * db * block) : 0;
    z = take(piece * vb * 32 * 4);
    g = c.gx ? take(rb * vb * block) : 0;
    gt = c.gw ? take(rb * vb * block) : 0;
    unit_x = take(rb * 32 * 4);
    unit_w = take(vb * 32 * 4);
    bias = take(vb * 32 * 4);
    stat = take(piece * parts * 8);
    info = take(piece * sizeof(RowInfo));
    factor = take(piece * 4);
    turned = take(piece * 4);
    sums = c.gb ? take(piece / 64 * vb * 32 * 4) : 0;
    maxima = take(sizeof(Maxima));
    acc_w = several && c.gw ? take(c.v * db * 32 * 4) : 0;
    acc_b = several && c.gb ? take(vb * 32 * 4) : 0;
    bytes = at;
  }
};

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

template <typename F>
void by_type(int32_t type, const char *what, F &&f) {
  switch (type) {
    case FLY_F32: f(float{}); break;
    case FLY_F16: f(_Float16{}); break;
    case FLY_BF16: f(bhalf{}); break;
    default: FLY_REQUIRE(false, what);
  }
}

template <typename T>
void run(const Call &c, const Given &g, char *ws, hipStream_t st) {
  using H = typename Multiplied<T>::H;
  constexpr int P = Multiplied<T>::P;
  const Space s(c, P);
  auto at = [&](size_t offset) { return ws + offset; };
  auto blocks = [&](size_t offset) { return reinterpret_cast<int4v *>(ws + offset); };
  auto floats = [&](size_t offset) { return reinterpret_cast<float *>(ws + offset); };
  Maxima *maxima = reinterpret_cast<Maxima *>(at(s.maxima));
  float *unit_x = P == 2 ? floats(s.unit_x) : nullptr, *unit_w = P == 2 ? floats(s.unit_w) : nullptr;
  RowInfo *info = c.grads() ? reinterpret_cast<RowInfo *>(at(s.info)) : nullptr;
  hipLaunchKernelGGL(k_clear, dim3(1), dim3(1), 0, st, maxima);
  check_launch("read-out loss");
  auto lay = [&](const Lay<T> &l) {
    hipLaunchKernelGGL(k_lay<T>, dim3((unsigned)(2 * l.kt)), dim3(1024), 0, st, l);
    check_launch("read-out operands");
  };
  lay(Lay<T>{static_cast<const T *>(g.w), g.ldw, c.v, c.d, (int)s.db, (int)s.vb, blocks(s.w), c.gx ? blocks(s.wt) : nullptr,
             unit_w, P == 2 ? &maxima->weight : nullptr, g.bias, g.bias_type, floats(s.bias), Targets{}});
  for (int64_t first = 0; first < c.rows; first += s.piece) {
    const int rows = (int)std::min(s.piece, c.rows - first);
    const bool last = first + rows == c.rows;
    const int rb = (rows + 31) / 32, tiles = (rows + kGradRows - 1) / kGradRows;
    const int64_t ldz = s.vb * 32;
    if (first) {
      hipLaunchKernelGGL(k_clear_row, dim3(1), dim3(1), 0, st, maxima);
      check_launch("read-out loss");
    }
    Targets t = g.targets;
    t.index = static_cast<const char *>(t.index) + first * t.k * (t.wide ? 8 : 4);
    if (t.weight) t.weight += first * t.k;
    if (t.legal) t.legal += first * t.ldl;
    lay(Lay<T>{static_cast<const T *>(g.x) + first * g.ldx, g.ldx, rows, c.d, (int)s.db, rb, blocks(s.x),
               c.gw ? blocks(s.xt) : nullptr, unit_x, nullptr, nullptr, 0, nullptr, t});
    product<H, P>(Blocks{blocks(s.w), blocks(s.x), (int)(2 * s.vb), 2 * rb, (int)s.db, 0, 0, 0},
                  LogitsOut{unit_x, unit_w, floats(s.bias), t.legal, t.ldl, rows, (int)c.v, floats(s.z), ldz,
                            reinterpret_cast<float2 *>(at(s.stat)), s.piece},
                  st);
    hipLaunchKernelGGL(k_loss_rows, dim3(blocks_for(rows, 4)), dim3(256), 0, st, reinterpret_cast<const float2 *>(at(s.stat)),
                       s.piece, s.parts, rows, t, floats(s.z), ldz, unit_x,
                       g.row_scale ? g.row_scale + first : nullptr, g.grad_scale, g.loss ? g.loss + first : nullptr, info,
                       floats(s.factor), floats(s.turned), &maxima->row);
    check_launch("read-out loss");
    if (!c.grads()) continue;
    hipLaunchKernelGGL((k_logits_grad<H, P>), dim3(blocks_for(c.v, kGradCols), tiles), dim3(256), 0, st, floats(s.z), ldz,
                       rows, t, info, floats(s.factor), floats(s.turned), unit_w, maxima, 2 * rb, (int)s.vb,
                       c.gx ? blocks(s.g) : nullptr, c.gw ? blocks(s.gt) : nullptr, c.gb ? floats(s.sums) : nullptr, ldz);
    check_launch("read-out gradient");
    if (c.gb)
      by_type(g.bias_type, "the bias must be float32, float16 or bfloat16", [&](auto b) {
        using B = decltype(b);
        hipLaunchKernelGGL(k_bias_grad<B>, dim3(blocks_for(c.v, 256)), dim3(256), 0, st, floats(s.sums), ldz, tiles, (int)c.v,
                           first ? floats(s.acc_b) : nullptr, last ? nullptr : floats(s.acc_b), static_cast<B *>(g.gb));
        check_launch("read-out gradient");
      });
    if (c.gx)
      product<H, P>(Blocks{blocks(s.wt), blocks(s.g), (int)(2 * s.db), 2 * rb, (int)s.vb, 0, 0, 0},
                    GradOut<T>{floats(s.factor), P == 2 ? &maxima->weight : nullptr, rows, (int)c.d, nullptr, nullptr, 0,
                               static_cast<T *>(g.gx) + first * g.ldgx, g.ldgx},
                    st);
    if (c.gw)
      product<H, P>(Blocks{blocks(s.xt), blocks(s.gt), (int)(2 * s.db), (int)(2 * s.vb), rb, 0, 0, 0},
                    GradOut<T>{nullptr, &maxima->row, (int)c.v, (int)c.d, first ? floats(s.acc_w) : nullptr,
                               last ? nullptr : floats(s.acc_w), s.db * 32, static_cast<T *>(g.gw), g.ldgw},
                    st);
  }
}

void require_call(const Call &c) {
  FLY_REQUIRE(c.type >= FLY_F32 && c.type <= FLY_BF16, "x and w must be float32, float16 or bfloat16");
  FLY_REQUIRE(c.rows >= 0 && c.rows < (int64_t)1 << 40 && c.d >= 1 && c.d <= (int64_t)1 << 16 && c.v >= 1 &&
                  c.v <= (int64_t)1 << 20,
              "size out of range");
}
size_t call_ws(const Call &c) { return c.rows ? Space(c, c.type == FLY_F32 ? 2 : 1).bytes : 0; }

}  // namespace
}  // namespace fly

using namespace fly;

extern "C" size_t fly_readout_loss_workspace(int32_t type, int64_t rows, int64_t d, int64_t v, int32_t wanted) {
  const Call c{type, rows, d, v, (wanted & FLY_GRAD_X) != 0, (wanted & FLY_GRAD_W) != 0, (wanted & FLY_GRAD_B) != 0};
  size_t bytes = 0;
  guard([&] {
    require_call(c);
    bytes = call_ws(c);
  });
  return bytes;
}

extern "C" int fly_readout_loss(const void *x, int32_t type, int64_t ldx, int64_t rows, int64_t d, const void *w, int64_t ldw,
                                int64_t v, const void *bias, int32_t bias_type, const uint8_t *legal, int64_t ldl,
                                const void *index, int32_t index_type, const float *weight, int32_t k, float *loss,
                                const float *row_scale, float grad_scale, void *gx, int64_t ldgx, void *gw, int64_t ldgw,
                                void *gb, void *ws, size_t ws_bytes, void *stream) {
  return guard([&] {
    const Call c{type, rows, d, v, gx != nullptr, gw != nullptr, gb != nullptr};
    require_call(c);
    FLY_REQUIRE(bias_type >= FLY_F32 && bias_type <= FLY_BF16, "the bias must be float32, float16 or bfloat16");
    FLY_REQUIRE(index_type == FLY_I32 || index_type == FLY_I64, "the targets must be int32 or int64");
    FLY_REQUIRE(k >= 1 && k <= 1024, "k must lie in 1..1024");
    FLY_REQUIRE(w && (!rows || (x && index)), "null pointer");
    FLY_REQUIRE(!rows || loss || c.grads(), "neither loss nor gradients are wanted");
    FLY_REQUIRE(ldx >= d && ldw >= d && (!legal || ldl >= v) && (!gx || ldgx >= d) && (!gw || ldgw >= d), "rows overlap");
    hipStream_t st = as_stream(stream);
    if (!rows) {
      by_type(type, "", [&](auto t) {
        using T = decltype(t);
        if (gw) hipLaunchKernelGGL(k_zeros<T>, dim3(1024), dim3(256), 0, st, static_cast<T *>(gw), ldgw, v, d);
      });
      by_type(bias_type, "", [&](auto t) {
        using T = decltype(t);
        if (gb) hipLaunchKernelGGL(k_zeros<T>, dim3(64), dim3(256), 0, st, static_cast<T *>(gb), v, 1, v);
      });
      check_launch("read-out gradient");
      return;
    }
    FLY_REQUIRE(ws && ws_bytes >= call_ws(c) && aligned(ws, 256), "workspace too small or misaligned");
    const Given g{x, w, bias, ldx, ldw, bias_type,
                  Targets{index, index_type == FLY_I64, weight, k, legal, ldl, (int)v}, row_scale, grad_scale, loss, gx, gw, gb,
                  ldgx, ldgw};
    by_type(type, "", [&](auto t) { run<decltype(t)>(c, g, static_cast<char *>(ws), st); });
  });
}
