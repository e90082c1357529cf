// Softmax cross entropy of a read-out and its gradients, without keeping the logits.
//
//   z_rv = sum_d x_rd w_vd + b_v over the row's visible columns,   p_r = softmax(z_r)
//   loss_r = sum_j a_rj (log sum_v exp z_rv - z_r,t_rj)            a list of targets t with weights a; one with weight 1
//   u_rv = (A_r p_rv - sum_{j: t_rj = v} a_rj) / B_r               A = sum_j a, B = sum_j |a|: |u| <= 2 whatever the weights
//   dx_r = f_r sum_v u_rv w_v,  dw_v = sum_r f_r u_rv x_r,  db_v = sum_r f_r u_rv,   f = B row_scale grad_scale
//
// Rows run in pieces whose logits and u fit a bounded workspace.  A piece is six launches:
//   k_lay          the weight (once) and the rows into the matrix cores' blocks, for both directions; the rows' targets
//   k_blocks       logits, and what is kept of them (LogitsOut)
//   k_loss_rows    the rows' log-sum-exp and losses
//   k_logits_grad  u into blocks for both directions, its columns' sums
//   k_blocks       dx and dw side by side (GradOut)
//   k_finish       db, and the sums of products that ran in parts
// The loss alone is the first three.  Nothing depends on which workgroup comes first, so results repeat bit for bit.
#include "blocks.hpp"
#include "readout.hpp"

#include <cmath>

namespace fly {
namespace {

constexpr float kUnit = 16384.0f;            // u is multiplied as 2^14 u: float16 then holds it from 2^-28 on without loss

// ---- targets ---------------------------------------------------------------------------------------------------------

// A row's targets as the later kernels take them: each column once (-1: none) with its weights added up, and over the row the sum
// of the weights and of their sizes.
struct List {
  int *column;      // (k, row)
  float *weight;
  float *logit;     // filled in by the product
  float2 *sums;     // (row)
  int64_t ld;       // rows of a piece
  int k;
};

// By a wave; the sum of the weights' sizes, 0 of a row where no target counts.
__device__ __forceinline__ float list_row(const Targets &t, const List &l, int64_t row, int lane) {
  float share = 0.0f, whole = 0.0f;
  for (int first = 0; first < t.k; first += 64) {
    const int j = first + lane;
    float a = 0.0f;
    int c = j < t.k ? target_of(t, row, j, a) : -1;
    if (c == -2) share = whole = __builtin_nanf("");
    if (c < 0) a = 0.0f;
    share += a;
    whole += fabsf(a);
    float sum = a;
    bool again = c < 0;
    if (t.k > 1)
      for (int other = 0; other < t.k; other += 64) {
        float b = a;
        int d = c;
        if (other != first) {
          d = other + lane < t.k ? target_of(t, row, other + lane, b) : -1;
          if (d < 0) b = 0.0f;
        }
        const int n = min(64, t.k - other);
        for (int i = 0; i < n; ++i) {
          const int di = __builtin_amdgcn_readlane(d, i);
          const float bi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(b), i));
          again |= di == c && other + i < j;
          if (di == c && other + i > j) sum += bi;
        }
      }
    if (j < t.k) {
      l.column[j * l.ld + row] = again ? -1 : c;
      l.weight[j * l.ld + row] = sum;
    }
  }
  share = wave_sum(share);
  whole = wave_sum(whole);
  if (lane == 0) l.sums[row] = make_float2(share, whole);
  return whole;
}

// ---- operands into blocks --------------------------------------------------------------------------------------------

constexpr int kLeastUnit = -120;   // as a power of 2: its inverse and its products with a half stay in float32's range

// What a row held as two halves is divided by: 2^e with max |row| / 2^e in [2^13, 2^14).  Of a row with NaN or infinities 1, of a row
// of zeros the least there is: the units' maximum scales the other rows' products, and no bits of theirs may go to a row without any.
__device__ __forceinline__ float unit_of(float top) {
  if (top == 0.0f) return ldexpf(1.0f, kLeastUnit);
  if (!(top <= 3.4028234663852886e38f)) return 1.0f;
  int e;
  (void)frexpf(top, &e);                  // top = m 2^e, m in [1/2, 1)
  return ldexpf(1.0f, max(e - 14, kLeastUnit));
}

template <typename T>
struct Lay {
  const T *src;
  int64_t ld, rows, cols;
  int kb, kt;             // blocks of 32 columns, and of 32 rows
  int4v *out, *turned;    // (rows, columns), and (columns, rows) or null
  float *unit;            // of two planes: each row's
  const void *bias;
  int bias_type;
  float *bias_out;        // bias as float32, or null: no bias wanted
  Targets targets;        // of the rows (index null: none): one without any left counts as zeros, whatever it holds
  List list;
  const float *row_scale;
  float grad_scale;
  float *factor;           // B row_scale grad_scale of a row, or null
  double *turned_factor;   // and times its unit (0 of zeros held as halves)
};
template <typename T>
struct Lays {
  Lay<T> of[2];           // the weight and the rows, or the rows alone after nothing (kt 0)
};

constexpr int kSlab = 512;   // columns that pass through LDS at a time

// 16 rows, a wave each; rows past the last are zero.  SLABS > 0: the row stays in registers, all its loads in flight together, from
// its maximum to its planes; 0: rows of any length, read from memory once more for the maximum.
// Bound by memory: a float32 weight of 4,168 x 2,333 with 256 rows 27 us (41 MB in, 82 out: 4.5 TB/s), a bfloat16 one with 16,384 rows
// 67 us (96 MB in, 192 out).
// 64 registers at most, for two workgroups a CU: with 66 the calls of 256 and of 1,120 float32 positions take 3 us more.
template <typename T, int SLABS>
__global__ __launch_bounds__(1024, 8) void k_lay(const Lays<T> lays) {
  using H = typename Multiplied<T>::H;
  constexpr int P = Multiplied<T>::P, N = Piece<T>::N, PIECES = kSlab / (64 * N), HELD = SLABS ? SLABS : 1;
  __shared__ __attribute__((aligned(16))) uint16_t lds[2][P][16][kSlab + 8];
  __shared__ __attribute__((aligned(16))) uint16_t passed[16];   // all bits, or none: rows that count for dw
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool second = (int)blockIdx.x >= 2 * lays.of[0].kt;
  const Lay<T> &o = lays.of[second];
  const int group = blockIdx.x - (second ? 2 * lays.of[0].kt : 0);
  const int64_t row = (int64_t)group * 16 + wave;
  bool in = row < o.rows;
  const T *src = o.src + (in ? row : 0) * o.ld;
  float whole = 0.0f;
  if (in && o.targets.index) {
    whole = list_row(o.targets, o.list, row, lane);
    in = whole != 0.0f;   // NaN too
  }
  Raw16 held[HELD][PIECES];
  auto fetch = [&](Raw16 (&p)[PIECES], int first) {
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int i = first / N + lane + 64 * j;
      if constexpr (SLABS > 0) p[j] = load_clamped(src, i, (int)o.cols);
      else p[j] = in && (int64_t)i * N < o.cols ? load_raw(src, i, o.cols) : Raw16{};
    }
  };
  if constexpr (SLABS > 0)
#pragma unroll
    for (int s = 0; s < SLABS; ++s) fetch(held[s], s * kSlab);
  float unit = 1.0f;
  bool zeros = false;
  if constexpr (P == 2) {
    float top = 0.0f;
    if constexpr (SLABS > 0) {
#pragma unroll
      for (int s = 0; s < SLABS; ++s)
#pragma unroll
        for (int j = 0; j < PIECES; ++j)
#pragma unroll
          for (int e = 0; e < N; ++e) top = __builtin_elementwise_maximum(top, fabsf(element<T>(held[s][j], e)));
      if (!in) top = 0.0f;
    } else if (in) {
      for (int64_t i = lane; i * N < o.cols; i += 64) {
        const Raw16 p = load_raw(src, (int)i, o.cols);
#pragma unroll
        for (int e = 0; e < N; ++e) top = __builtin_elementwise_maximum(top, fabsf(element<T>(p, e)));
      }
    }
    top = wave_reduce(top, [](float a, float b) { return nan_max(a, b); });
    zeros = top == 0.0f;
    unit = unit_of(top);
    if (lane == 0) o.unit[row] = unit;
  }
  if (o.bias_out && lane == 0) {
    float b = 0.0f;
    if (row < o.rows && o.bias) b = bias_at(o.bias, o.bias_type, row);
    o.bias_out[row] = b;
  }
  float f = 0.0f;
  if (o.factor && lane == 0 && row < o.rows) {
    if (in) f = whole * (o.row_scale ? o.row_scale[row] : 1.0f) * o.grad_scale;
    o.factor[row] = f;
    o.turned_factor[row] = (double)f * (zeros ? 0.0f : unit);
  }
  if (lane == 0) passed[wave] = !o.factor || f != 0.0f ? 0xffff : 0;   // read behind the first slab's barrier
  const float inverse = 1.0f / unit;
  auto slab = [&](Raw16 (&p)[PIECES], int first, int turn) {
    auto &part = lds[turn];
    if constexpr (SLABS > 0) {
      if (first + kSlab > o.cols)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) settle<T>(p[j], first / N + lane + 64 * j, (int)o.cols);
      if (!in)
#pragma unroll
        for (int j = 0; j < PIECES; ++j) p[j] = Raw16{};
    }
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
      const int at = (lane + 64 * j) * N;
      if constexpr (P == 1) {
        *reinterpret_cast<int4v *>(&part[0][wave][at]) = int4v{(int)p[j].v[0], (int)p[j].v[1], (int)p[j].v[2], (int)p[j].v[3]};
      } else {
        uint32_t w[P][2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          uint32_t a[P], b[P];
          planes_of<H, P>(element<T>(p[j], 2 * e) * inverse, a);
          planes_of<H, P>(element<T>(p[j], 2 * e + 1) * inverse, b);
#pragma unroll
          for (int q = 0; q < P; ++q) w[q][e] = a[q] | b[q] << 16;
        }
#pragma unroll
        for (int q = 0; q < P; ++q) *reinterpret_cast<uint2 *>(&part[q][wave][at]) = make_uint2(w[q][0], w[q][1]);
      }
    }
    __syncthreads();   // one a slab: its halves of LDS take turns, and every wave has read the other one by now
    const int k = first / 32 + wave;
    if (k >= o.kb) return;
#pragma unroll
    for (int q = 0; q < P; ++q)
      o.out[(((int64_t)group * o.kb + k) * P + q) * 64 + lane] =
          *reinterpret_cast<const int4v *>(&part[q][lane & 15][32 * wave + 8 * (lane >> 4)]);
    if (!o.turned) return;
    const int at = 32 * wave + 16 * (lane >> 5) + (lane & 15), eight = (lane >> 4) & 1;
    const int64_t block = ((int64_t)2 * k + (lane >> 5)) * o.kt + (group >> 1);
    const int4v rows = *reinterpret_cast<const int4v *>(&passed[8 * eight]);
#pragma unroll
    for (int q = 0; q < P; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = (part[q][8 * eight + 2 * e][at] | (uint32_t)part[q][8 * eight + 2 * e + 1][at] << 16) & (uint32_t)rows[e];
      o.turned[(block * P + q) * 64 + 16 * (2 * (group & 1) + eight) + (lane & 15)] =
          int4v{(int)w[0], (int)w[1], (int)w[2], (int)w[3]};
    }
  };
  if constexpr (SLABS > 0) {
#pragma unroll
    for (int s = 0; s < SLABS; ++s)
      if (s * kSlab < o.kb * 32) slab(held[s], s * kSlab, s & 1);
  } else {
    for (int s = 0; s * kSlab < o.kb * 32; ++s) {
      fetch(held[0], s * kSlab);
      slab(held[0], s * kSlab, s & 1);
    }
  }
}

// ---- logits ----------------------------------------------------------------------------------------------------------

// How far a logit lies below its part's largest, in 65,535 steps up to 32, from where on it counts as none (its p is below 2e-14 of
// the part's largest).  The softmax errs by half a step, 2^-12 relative, about half of what the rounding of its gradient to float16
// may add.  v_cvt_pknorm makes two of them in an instruction.
constexpr float kSteps = 65535.0f / 32.0f;
constexpr uint32_t kNone = 65535;

// What is left of a piece of rows' logits: each row's maximum and sum over a wave's columns, its targets' logits, and for the
// gradients the logits themselves (Keep: float32, or their distance from the maximum in 16 bits).  Those lie in blocks of 16 rows x
// 16 columns as the lanes hold them (lane l: row l & 15, columns 4 (l >> 4) .. + 3), so a wave's 64 columns leave as whole kilobytes
// and are not turned over in LDS.
enum Keep { kNothing, kFloats, kCodes };
template <Keep KEEP>
struct LogitsOut {
  static constexpr bool kLogits = true;
  const float *unit_m, *unit_n;   // or null
  const float *bias;
  const uint8_t *legal;
  int64_t ldl;
  int rows, cols, padded;   // columns, and to a multiple of 32, as bias, units and logits are
  void *z;
  float2 *parts;      // (row, column part)
  int64_t ld_parts;
  List list;
  template <int FN, int FM>
  __device__ __forceinline__ void tile(float4v (&acc)[FN][FM], int m0, int n0, int lane, int part, int, float *turn) const {
    constexpr int PITCH = 16 * FN + 4;
    const int quad = 4 * (lane >> 4);
    // What 16 rows need from memory is loaded while the 16 before them are done, without branches: the bytes of the mask (the last
    // ones of a row moved down to their columns) and the first 32 entries of the lists.
    struct __attribute__((packed)) Bytes {
      uint32_t w;
    };
    struct Ahead {
      uint32_t shown[FN];
      int column[8];
      float unit;
    };
    auto entries = [&](int (&to)[8], int first, int64_t row) {
#pragma unroll
      for (int j = 0; j < 8; ++j) to[j] = list.column[min(first + 4 * j + (lane >> 4), list.k - 1) * list.ld + row];
    };
    auto fetch = [&](int i) {
      Ahead a;
      const int64_t row = min(m0 + 16 * i + (lane & 15), rows - 1);
      a.unit = unit_m ? unit_m[row] : 1.0f;
      if (legal) {
        const uint8_t *seen = legal + row * ldl;
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int c = n0 + 16 * j + quad, most = max(cols - 4, 0);
          if (cols >= 4) {
            const int past = c - most;   // columns
            const uint32_t w = reinterpret_cast<const Bytes *>(seen + min(c, most))->w;
            a.shown[j] = past <= 0 ? w : past < 4 ? w >> (8 * past) : 0u;
          } else {
            a.shown[j] = 0u;
            for (int e = 0; e < cols; ++e)
              if (c == 0 && seen[e]) a.shown[j] |= 1u << (8 * e);
          }
        }
      }
      entries(a.column, 0, row);
      return a;
    };
    constexpr bool AHEAD = FM < 4;   // 16 waves of 64 x 64 have no registers for it: the loads of 16 rows go together, and are waited for
    Ahead next;
    if constexpr (AHEAD) next = fetch(0);
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = m0 + 16 * i + (lane & 15);
      const Ahead mine = AHEAD ? next : fetch(i);
      if (AHEAD && i + 1 < FM) next = fetch(i + 1);
      float4v v[FN];
      PartSum p{-INFINITY, 0.0f};
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int c = n0 + 16 * j + quad, at = min(c, padded - 4);
        v[j] = acc[j][i];
        if (unit_n) {
          const float4v un = *reinterpret_cast<const float4v *>(unit_n + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[j][e] *= mine.unit * un[e];   // powers of 2, whose product is no larger than a logit needs
        }
        v[j] += *reinterpret_cast<const float4v *>(bias + at);
        if (legal || n0 + 16 * FN > cols) {
          const uint32_t shown = legal ? mine.shown[j] : 0x01010101u;
          float l[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) l[e] = c + e < cols && (shown & (0xffu << (8 * e))) ? v[j][e] : -INFINITY;
          v[j] = float4v{l[0], l[1], l[2], l[3]};
        }
        p.top = fmaxf(p.top, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
      }
      p.top = over_four(p.top, [](float x, float y) { return fmaxf(x, y); });
      const float base = base_of(p.top);
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) p.sum += exp2_of((v[j][e] - base) * kLog2e);
      p.sum = over_four(p.sum, [](float x, float y) { return x + y; });
      if (lane < 16 && m < rows) parts[m * ld_parts + part] = make_float2(p.top, p.sum);
      if constexpr (KEEP != kNothing) {
        const int64_t block = ((int64_t)(m0 >> 4) + i) * (padded >> 4) + (n0 >> 4);
        if (m0 + 16 * i < rows)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            if (n0 + 16 * j < padded) {
              if constexpr (KEEP == kFloats) {
                static_cast<float4v *>(z)[(block + j) * 64 + lane] = v[j];
              } else {
                float g[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) g[e] = (p.top - v[j][e]) * (1.0f / 32.0f);
                static_cast<uint2 *>(z)[(block + j) * 64 + lane] =
                    make_uint2(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(g[0], g[1])),
                               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pknorm_u16(g[2], g[3])));
              }
            }
      }
#pragma unroll
      for (int j = 0; j < FN; ++j) *reinterpret_cast<float4v *>(turn + (lane & 15) * PITCH + 16 * j + quad) = v[j];
      asm volatile("" ::: "memory");   // other lanes read what this one wrote: a wave's LDS accesses keep their order
      // the targets among these columns: 4 entries of 16 rows in a load, 8 loads in flight
      const int64_t row = min(m, rows - 1);
      auto found = [&](const int (&column)[8], int first) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int entry = first + 4 * j + (lane >> 4), at = column[j] - n0;
          if (m < rows && entry < list.k && at >= 0 && at < 16 * FN)
            list.logit[entry * list.ld + row] = turn[(lane & 15) * PITCH + at];
        }
      };
      found(mine.column, 0);
      for (int first = 32; first < list.k; first += 32) {
        int column[8];
        entries(column, first, row);
        found(column, first);
      }
      asm volatile("" ::: "memory");
    }
  }
};

// ---- rows ------------------------------------------------------------------------------------------------------------

// A wave per row; a first workgroup finds the largest factors.
__global__ __launch_bounds__(256) void k_loss_rows(const float2 *__restrict__ parts, int64_t ld_parts, int count, int rows,
                                                   const List l, float *__restrict__ loss, RowInfo *__restrict__ info,
                                                   const float *__restrict__ factor, const double *__restrict__ turned_factor,
                                                   const float *__restrict__ unit_n, int cols, Maxima *__restrict__ maxima) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (info && blockIdx.x == 0) {
    __shared__ float weight[4];
    __shared__ double factors[4];
    float w = 0.0f;
    double r = 0.0;
    auto raise = [](auto &most, auto v) {   // finite ones
      v = v < 0 ? -v : v;
      if (v > most && v < INFINITY) most = v;
    };
    if (unit_n)
#pragma unroll 8
      for (int c = threadIdx.x; c < cols; c += 256) raise(w, unit_n[c]);
#pragma unroll 8
    for (int i = threadIdx.x; i < rows; i += 256) raise(r, turned_factor[i]);
    w = wave_max(w);
    for (int d = 1; d < 64; d <<= 1) raise(r, __shfl_xor(r, d));
    if (lane == 0) weight[wave] = w, factors[wave] = r;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int i = 1; i < 4; ++i) raise(w, weight[i]), raise(r, factors[i]);
      int e;
      const double fraction = frexp(r, &e);
      *maxima = Maxima{r, w, ldexpf(1.0f, e), (float)fraction};
    }
    return;
  }
  const int64_t row = (blockIdx.x - (info ? 1 : 0)) * (int64_t)4 + wave;
  if (row >= rows) return;
  const float2 sums = l.sums[row];
  PartSum p{-INFINITY, 0.0f};
  for (int i = lane; i < count; i += 64) {
    const float2 v = parts[row * ld_parts + i];
    const float top = fmaxf(p.top, v.x), base = base_of(top);
    p.sum = p.sum * exp2_of((p.top - base) * kLog2e) + v.y * exp2_of((v.x - base) * kLog2e);
    p.top = top;
  }
  p = wave_part(p, kLog2e);
  const float log_sum = log2_of(p.sum);
  float sum = 0.0f;
  for (int j = lane; j < l.k; j += 64)
    if (l.column[j * l.ld + row] >= 0)
      sum += l.weight[j * l.ld + row] * ((p.top - l.logit[j * l.ld + row]) + kLn2 * log_sum);
  sum = wave_sum(sum);
  if (lane) return;
  const bool some = sums.y != 0.0f;   // NaN too
  if (loss) loss[row] = !some ? 0.0f : sums.y == sums.y ? sum : sums.y;
  if (!info) return;
  const bool passes = some && factor[row] != 0.0f;   // else u is 0, whatever the row holds
  info[row] = RowInfo{base_of(p.top), log_sum, passes ? sums.x / sums.y : 0.0f, passes ? sums.y : 0.0f};
}

// ---- the logits' gradient --------------------------------------------------------------------------------------------

constexpr int kGradRows = 64, kGradCols = 128, kGradPitch = 130;

// u of 64 rows x 128 columns into blocks, by rows (times the columns' units) and turned (times the rows' factors), and its columns'
// sums.  With 16-bit operands u is rounded to their type: both sides of a matrix instruction have one, two planes of u would double the
// gradients' products (590 us of 1,044 at 16,384 bfloat16 rows), and the outputs' own rounding is as large.  Parts of 2^shift columns.  Bound by memory and by the way there: all loads go first, then the tile passes through
// LDS (16,384 x 4,168 bfloat16 110 us, 137 MB in and 273 out; with each load behind the step before it 170).
template <typename H, int P, Keep KEEP>
__global__ __launch_bounds__(256) void k_logits_grad(const void *__restrict__ z, int64_t ldz, int rows, int cols, const List l,
                                                     const float2 *__restrict__ parts, int64_t ld_parts, int shift,
                                                     const RowInfo *__restrict__ info, const float *__restrict__ factor,
                                                     const double *__restrict__ turned_factor,
                                                     const float *__restrict__ unit_n, const Maxima *__restrict__ maxima,
                                                     int rb, int vb, int4v *__restrict__ out, int4v *__restrict__ turned,
                                                     float *__restrict__ sums, int64_t ld_sums) {
  __shared__ __attribute__((aligned(16))) float u[kGradRows][kGradPitch];
  __shared__ float col_sum[2][kGradCols], f_row[kGradRows], ft_row[kGradRows], un_col[kGradCols], f_part[kGradRows][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c0 = blockIdx.x * kGradCols, r0 = blockIdx.y * kGradRows;
  // 4 x 8 blocks of 16 x 16 logits, 8 for each wave; all loads first, without branches, then what is made of them
  using Kept = std::conditional_t<KEEP == kFloats, float4v, uint2>;
  const int row_blocks = (rows + 15) >> 4;   // that were stored
  const int64_t block0 = (int64_t)min((r0 >> 4) + wave, row_blocks - 1) * (ldz >> 4);
  Kept kept[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    kept[i] = static_cast<const Kept *>(z)[(block0 + min((c0 >> 4) + i, (int)(ldz >> 4) - 1)) * 64 + lane];
  const int64_t list_row = min(r0 + lane, rows - 1);
  int column[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) column[j] = l.column[min(wave + 4 * j, l.k - 1) * l.ld + list_row];
  const RowInfo mine = info[list_row];   // of a row of the lists
  const double most = maxima->row;
  const float most_weight = maxima->weight;
  if (tid < kGradRows) {
    const bool in = r0 + tid < rows;
    const float f = factor[list_row];
    const double ft = turned_factor[list_row];
    f_row[tid] = in ? f : 0.0f;
    ft_row[tid] = in ? (float)(most > 0.0 ? ft / most : ft) * kUnit : 0.0f;
  }
  if (tid >= 128) {
    const int c = c0 + tid - 128;
    un_col[tid - 128] = P == 2 && c < cols ? unit_n[c] / most_weight * kUnit : kUnit;
  }
  if constexpr (KEEP == kCodes) {
    // a part's largest p, times the share
    const int r = tid >> 2, q = tid & 3;
    float f = 0.0f;
    if (r0 + r < rows && c0 + (q << shift) < cols && (q << shift) < kGradCols) {
      const RowInfo i = info[r0 + r];
      const float top = parts[(r0 + r) * ld_parts + (c0 >> shift) + q].x;
      if (i.share != 0.0f) f = i.share * exp2_of((top - i.top) * kLog2e - i.log_sum);
    }
    f_part[r][q] = f;
    __syncthreads();
  }
  const int r16 = 16 * wave + (lane & 15);
  RowInfo row{};
  if constexpr (KEEP == kFloats) row = info[min(r0 + r16, rows - 1)];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = 16 * i + 4 * (lane >> 4);
    const bool in = r0 + r16 < rows && c0 + c < ldz;
    float v[4];
    if constexpr (KEEP == kFloats) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float p = row.share * exp2_of((kept[i][e] - row.top) * kLog2e - row.log_sum);
        v[e] = in && row.share != 0.0f ? p : 0.0f;
      }
    } else {
      const float f = in ? f_part[r16][c >> shift] : 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t code = e < 2 ? (kept[i].x >> (16 * e)) & 0xffffu : (kept[i].y >> (16 * (e - 2))) & 0xffffu;
        v[e] = f * (code == kNone ? 0.0f : exp2_of((float)code * (-kLog2e / kSteps)));
      }
    }
    *reinterpret_cast<float2 *>(&u[r16][c]) = make_float2(v[0], v[1]);
    *reinterpret_cast<float2 *>(&u[r16][c + 2]) = make_float2(v[2], v[3]);
  }
  __syncthreads();
  // the targets among these columns, each once
  auto aim = [&](int j, int c) {
    if (r0 + lane >= rows || j >= l.k || c < c0 || c >= c0 + kGradCols || mine.whole == 0.0f) return;
    const int64_t from = j * l.ld + r0 + lane;
    u[lane][c - c0] = mine.share * exp2_of((l.logit[from] - mine.top) * kLog2e - mine.log_sum) - l.weight[from] / mine.whole;
  };
#pragma unroll
  for (int j = 0; j < 8; ++j) aim(wave + 4 * j, column[j]);
  for (int j = wave + 32; j < l.k; j += 4) aim(j, l.column[j * l.ld + list_row]);
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

// ---- gradients -------------------------------------------------------------------------------------------------------

// out[m][n] = sum * *power / 2^14 * row[m] * *times, after what earlier pieces of rows gave.  The power of 2 comes first: with the row's
// factor it may pass float32's range where the gradient does not.  Where k runs in parts, the sums of each go to `share` and k_finish
// adds them up.
template <typename T>
struct GradOut {
  static constexpr bool kLogits = false;
  const float *row, *power, *times;   // or null: 1
  int rows, cols;
  const float *before;
  float *after;              // or null: the last piece, into out
  int64_t ld_sum;            // columns, to a multiple of 32
  T *out;
  int64_t ld;
  float *share;              // (part, row, column) or null
  __device__ __forceinline__ float2 scale() const { return make_float2((power ? *power : 1.0f) / kUnit, times ? *times : 1.0f); }
  __device__ __forceinline__ void put(int m, int n, const float4v &sum, float2 scale) const {
    const float f = row ? row[m] : scale.y;
    float4v w;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = sum[e] * scale.x * f;
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
  }
  template <int FN, int FM>
  __device__ __forceinline__ void tile(float4v (&acc)[FN][FM], int m0, int n0, int lane, int, int split, float *turn) const {
    const float2 s = scale();
    float *to = share ? share + (int64_t)split * rows * ld_sum : nullptr;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      float4v v[FN];
#pragma unroll
      for (int j = 0; j < FN; ++j) v[j] = acc[j][i];
      turn_over<FN>(v, turn, lane, [&](int r, int c, const float4v &four) {
        const int m = m0 + 16 * i + r, n = n0 + c;
        if (m >= rows || n >= cols) return;
        if (to) *reinterpret_cast<float4v *>(to + m * ld_sum + n) = four;
        else put(m, n, four, s);
      });
    }
  }
};

// The last of a piece of rows, in one launch: the columns' sums over all tiles of rows, after what earlier pieces gave (workgroups of 32
// columns, 32 lanes of tiles), and the parts of the products' k.
template <typename B>
struct BiasOut {
  const float *sums;         // (tile, column) or null
  int64_t ld;
  int tiles, cols;
  const float *before;
  float *after;
  B *out;
};
template <typename T>
struct Join {
  GradOut<T> out;
  int splits, groups;        // workgroups, 0 without parts
};
template <typename T, typename B>
__global__ __launch_bounds__(1024) void k_finish(const BiasOut<B> b, int bias_groups, const Join<T> x, const Join<T> w) {
  __shared__ float share[32][33];
  if ((int)blockIdx.x < bias_groups) {
    const int lane = threadIdx.x & 31, part = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < b.cols)
      for (int i = part; i < b.tiles; i += 32) s += b.sums[i * b.ld + c];
    share[part][lane] = s;
    __syncthreads();
    if (part || c >= b.cols) return;
    s = b.before ? b.before[c] : 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += share[i][lane];
    if (b.after) b.after[c] = s;
    else b.out[c] = static_cast<B>(s);
    return;
  }
  int group = blockIdx.x - bias_groups;
  const Join<T> &j = group < x.groups ? x : w;
  if (group >= x.groups) group -= x.groups;
  const GradOut<T> &g = j.out;
  const int64_t per = g.ld_sum / 4, all = g.rows * per, stride = g.rows * g.ld_sum;
  const float2 s = g.scale();
  for (int64_t i = group * (int64_t)1024 + threadIdx.x; i < all; i += (int64_t)j.groups * 1024) {
    const int m = (int)(i / per), n = 4 * (int)(i % per);
    if (n >= g.cols) continue;
    const float *from = g.share + m * g.ld_sum + n;
    float4v sum = *reinterpret_cast<const float4v *>(from);
    for (int p = 1; p < j.splits; ++p) sum += *reinterpret_cast<const float4v *>(from + p * stride);
    g.put(m, n, sum, s);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_zeros(T *__restrict__ out, int64_t ld, int64_t rows, int64_t cols) {
  for (int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x; i < rows * cols; i += (int64_t)gridDim.x * 256)
    out[i / cols * ld + i % cols] = static_cast<T>(0.0f);
}

// ---- the call --------------------------------------------------------------------------------------------------------

template <typename H, int P, typename EP, int COUNT>
void product(Shape shape, const Products<EP, COUNT> &p, hipStream_t st) {
  if (shape == kSmall) launch_blocks<H, P, 2, 2, 2, 2, 4>(p, st);
  else if constexpr (P == 2) {
    if constexpr (EP::kLogits) {   // the gradients' products never take it
      if (shape == kLarge) return launch_blocks<H, P, 2, 4, 4, 3, 3>(p, st);
    }
    launch_blocks<H, P, 4, 4, 2, 2, 4>(p, st);
  } else if (shape == kMedium) launch_blocks<H, P, 2, 4, 4, 2, 4>(p, st);
  else launch_blocks<H, P, 4, 4, 4, 4, 4>(p, st);
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
  const int padded = (int)s.vb * 32;
  for (int64_t first = 0; first < c.rows; first += s.piece) {
    const int rows = (int)std::min(s.piece, c.rows - first);
    const bool last = first + rows == c.rows;
    const int rb = (rows + 31) / 32, tiles = (rows + kGradRows - 1) / kGradRows;
    Targets t = g.targets;
    t.index = static_cast<const char *>(t.index) + first * t.k * (t.wide ? 8 : 4);
    if (t.weight) t.weight += first * t.k;
    if (t.legal) t.legal += first * t.ldl;
    const List list{reinterpret_cast<int *>(at(s.column)), floats(s.weight), floats(s.logit),
                    reinterpret_cast<float2 *>(at(s.list_sums)), s.piece, t.k};
    Lays<T> lays{};
    if (!first)
      lays.of[0] = Lay<T>{static_cast<const T *>(g.w), g.ldw, c.v, c.d, (int)s.db, (int)s.vb, blocks(s.w),
                          c.gx ? blocks(s.wt) : nullptr, unit_w, g.bias, g.bias_type, floats(s.bias), Targets{}, List{}, nullptr,
                          0.0f, nullptr, nullptr};
    lays.of[1] = Lay<T>{static_cast<const T *>(g.x) + first * g.ldx, g.ldx, rows, c.d, (int)s.db, rb, blocks(s.x),
                        c.gw ? blocks(s.xt) : nullptr, unit_x, nullptr, 0, nullptr, t, list,
                        g.row_scale ? g.row_scale + first : nullptr, g.grad_scale, c.grads() ? floats(s.factor) : nullptr,
                        reinterpret_cast<double *>(at(s.turned))};
    const unsigned groups = (unsigned)(2 * (lays.of[0].kt + rb));
    auto lay = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(groups), dim3(1024), 0, st, lays); };
    const int64_t slabs = (s.db * 32 + kSlab - 1) / kSlab;   // up to six slabs of a row stay in registers
    if (c.d < Piece<T>::N) lay(k_lay<T, 0>);
    else if (slabs <= 2) lay(k_lay<T, 2>);
    else if (slabs <= 6) lay(k_lay<T, 6>);
    else lay(k_lay<T, 0>);
    check_launch("read-out operands");
    const Shape wide = logits_shape(P, rows, c.v);
    const int parts = parts_of(P, wide, padded);
    const float2 *stat = reinterpret_cast<const float2 *>(at(s.stat));
    auto logits = [&](auto keep) {
      constexpr Keep KEEP = decltype(keep)::value;
      product<H, P>(wide,
                    Products<LogitsOut<KEEP>, 1>{
                        {Blocks{blocks(s.w), blocks(s.x), (int)(2 * s.vb), 2 * rb, (int)s.db, 1, 0, 0, 0}},
                        {LogitsOut<KEEP>{unit_x, unit_w, floats(s.bias), t.legal, t.ldl, rows, (int)c.v, padded, at(s.z),
                                         reinterpret_cast<float2 *>(at(s.stat)), s.parts, list}}},
                    st);
    };
    constexpr Keep KEPT = P == 1 ? kCodes : kFloats;
    if (c.grads()) logits(std::integral_constant<Keep, KEPT>{});
    else logits(std::integral_constant<Keep, kNothing>{});
    hipLaunchKernelGGL(k_loss_rows, dim3(blocks_for(rows, 4) + c.grads()), dim3(256), 0, st, stat, s.parts, parts, rows, list,
                       g.loss ? g.loss + first : nullptr, info, floats(s.factor), reinterpret_cast<double *>(at(s.turned)), unit_w,
                       (int)c.v, maxima);
    check_launch("read-out loss");
    if (!c.grads()) continue;
    hipLaunchKernelGGL((k_logits_grad<H, P, KEPT>), dim3(blocks_for(c.v, kGradCols), tiles), dim3(256), 0, st, at(s.z),
                       (int64_t)padded, rows, (int)c.v, list, stat, s.parts, part_shift(P, wide), info, floats(s.factor),
                       reinterpret_cast<double *>(at(s.turned)), unit_w, maxima, 2 * rb, (int)s.vb, c.gx ? blocks(s.g) : nullptr,
                       c.gw ? blocks(s.gt) : nullptr, c.gb ? floats(s.sums) : nullptr, (int64_t)padded);
    check_launch("read-out gradient");
    const Shape shape = grad_shape(P, c, rows);
    const Splits splits = splits_of(P, c, rows);
    const int64_t ld_sum = s.db * 32;
    const Blocks by_rows{blocks(s.wt), blocks(s.g), (int)(2 * s.db), 2 * rb, (int)s.vb, splits.x, 0, 0, 0};
    const Blocks by_columns{blocks(s.xt), blocks(s.gt), (int)(2 * s.db), (int)(2 * s.vb), rb, splits.w, 0, 0, 0};
    const GradOut<T> to_x{floats(s.factor), P == 2 ? &maxima->weight : nullptr, nullptr, rows, (int)c.d, nullptr, nullptr, ld_sum,
                          c.gx ? static_cast<T *>(g.gx) + first * g.ldgx : nullptr, g.ldgx,
                          splits.x > 1 ? floats(s.share_x) : nullptr};
    const GradOut<T> to_w{nullptr, &maxima->power, &maxima->fraction, (int)c.v, (int)c.d, first ? floats(s.acc_w) : nullptr,
                          last ? nullptr : floats(s.acc_w), ld_sum, static_cast<T *>(g.gw), g.ldgw,
                          splits.w > 1 ? floats(s.share_w) : nullptr};
    if (c.gx && c.gw)   // the longer sums first
      product<H, P>(shape,
                    s.vb / splits.x >= rb / splits.w ? Products<GradOut<T>, 2>{{by_rows, by_columns}, {to_x, to_w}}
                                                     : Products<GradOut<T>, 2>{{by_columns, by_rows}, {to_w, to_x}},
                    st);
    else if (c.gx) product<H, P>(shape, Products<GradOut<T>, 1>{{by_rows}, {to_x}}, st);
    else if (c.gw) product<H, P>(shape, Products<GradOut<T>, 1>{{by_columns}, {to_w}}, st);
    auto join = [&](const GradOut<T> &o, int parts_of_k) {
      return Join<T>{o, parts_of_k, o.share ? (int)std::min<int64_t>((o.rows * ld_sum / 4 + 1023) / 1024, 1024) : 0};
    };
    const Join<T> join_x = join(to_x, splits.x), join_w = join(to_w, splits.w);
    const int bias_groups = c.gb ? (int)blocks_for(c.v, 32) : 0;
    if (bias_groups + join_x.groups + join_w.groups)
      by_type(g.bias_type, "the bias must be float32, float16 or bfloat16", [&](auto b) {
        using B = decltype(b);
        const BiasOut<B> bias{floats(s.sums), padded, tiles, (int)c.v, first ? floats(s.acc_b) : nullptr,
                              last ? nullptr : floats(s.acc_b), static_cast<B *>(g.gb)};
        hipLaunchKernelGGL((k_finish<T, B>), dim3((unsigned)(bias_groups + join_x.groups + join_w.groups)), dim3(1024), 0, st, bias,
                           bias_groups, join_x, join_w);
        check_launch("read-out gradient");
      });
  }
}

void require_call(const Call &c) {
  FLY_REQUIRE(c.type >= FLY_F32 && c.type <= FLY_BF16, "x and w must be float32, float16 or bfloat16");
  FLY_REQUIRE(c.rows >= 0 && c.rows < (int64_t)1 << 40 && c.d >= 1 && c.d <= (int64_t)1 << 16 && c.v >= 1 &&
                  c.v <= (int64_t)1 << 20,
              "size out of range");
  FLY_REQUIRE(c.k >= 1 && c.k <= 1024, "k must lie in 1..1024");
}
size_t call_ws(const Call &c) {
  return !c.rows ? 0 : few_rows(c) ? few_ws(c) : Space(c, c.type == FLY_F32 ? 2 : 1).bytes;
}

}  // namespace
}  // namespace fly

using namespace fly;

extern "C" size_t fly_readout_loss_workspace(int32_t type, int64_t rows, int64_t d, int64_t v, int32_t k, int32_t wanted) {
  const Call c{type, rows, d, v, k, (wanted & FLY_GRAD_X) != 0, (wanted & FLY_GRAD_W) != 0, (wanted & FLY_GRAD_B) != 0};
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
    const Call c{type, rows, d, v, k, gx != nullptr, gw != nullptr, gb != nullptr};
    require_call(c);
    FLY_REQUIRE(bias_type >= FLY_F32 && bias_type <= FLY_BF16, "the bias must be float32, float16 or bfloat16");
    FLY_REQUIRE(index_type == FLY_I32 || index_type == FLY_I64, "the targets must be int32 or int64");
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
    if (few_rows(c)) run_few(c, g, static_cast<char *>(ws), st);
    else by_type(type, "", [&](auto t) { run<decltype(t)>(c, g, static_cast<char *>(ws), st); });
  });
}
