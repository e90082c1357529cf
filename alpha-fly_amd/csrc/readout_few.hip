// The read-out loss of few rows, where laying the weight out would cost more than the products: both operands come from memory as
// they lie.
//
//   k_few_logits   z = x w^T + b by blocks of 16 columns, the sums over d shared among a workgroup's 8 waves
//   k_few_rows     each row's log-sum-exp, targets and loss
//   k_few_u        g = f u in float32, and its columns' sums
//   k_few_grads    dx = g w in parts of the columns, dw = g^T x, side by side in one launch; k_few_join adds the parts up
//
// 16-bit operands are multiplied as such in the logits; everything else runs on float32 matrix instructions (16 x 16 x 4, products
// and sums in float32).  In those a lane holds one k of a row, so an operand whose k runs down the rows of a matrix is read as it
// lies too: 4 neighbours of a lane's 16-byte load go to 4 blocks, whose rows then are every fourth.
#include "blocks.hpp"
#include "readout.hpp"

#include <cmath>

namespace fly {
namespace {

constexpr int kWaves = 8;   // of k_few_logits, that share the sums over d

__device__ __forceinline__ float4v product4(float a, float b, float4v c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// 16 columns x 16 MB rows.  Rounds of BYTES of each row pass through LDS, so that a wave loads whole kilobytes of a row: read as the
// matrix cores take them, 64 bytes of 16 rows at a time, 4,168 x 2,333 float32 took 18 us at best.  Of the weights two rounds are
// in flight while a third is multiplied, of the rows, which the L2 holds, one.  Bound by the weight's bytes: 39 MB 15 us, 131 MB (32,000
// x 1,024) 40 us.
template <typename T, int MB, int BYTES>
__global__ __launch_bounds__(64 * kWaves) void k_few_logits(const T *__restrict__ x, int64_t ldx, int rows,
                                                            const T *__restrict__ w, int64_t ldw, int v, int d,
                                                            const void *__restrict__ bias, int bias_type,
                                                            const uint8_t *__restrict__ legal, int64_t ldl,
                                                            float *__restrict__ z, int64_t ldz, float2 *__restrict__ parts,
                                                            int64_t ld_parts) {
  constexpr int N = Piece<T>::N, PER = BYTES / 16, PITCH = BYTES + 16;   // pieces of a row in a round
  constexpr int LOADS = 16 * PER / (64 * kWaves), STEPS = PER / 4 / kWaves;   // a thread's of 16 rows; a wave's steps of 4 pieces
  static_assert(LOADS >= 1 && STEPS >= 1, "a round is shared by all waves");
  __shared__ __attribute__((aligned(16))) char lds[16 * (1 + MB) * PITCH];
  static_assert(sizeof(lds) >= kWaves * MB * 1024, "the sums fit in the operands' place");
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int v0 = blockIdx.x * 16, r0 = blockIdx.y * 16 * MB;
  float4v acc[MB];
#pragma unroll
  for (int m = 0; m < MB; ++m) acc[m] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  const int rounds = (d + PER * N - 1) / (PER * N);
  auto piece = [&](const T *base, int64_t ld, int row, int last, int at) {   // rows past the last repeat it
    return load_clamped(base + min(row, last) * ld, at, d);
  };
  Raw16 a[2][LOADS], b[MB][LOADS];
  auto load_w = [&](Raw16 (&to)[LOADS], int round) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = tid + 64 * kWaves * i;
      to[i] = piece(w, ldw, v0 + at / PER, v - 1, round * PER + at % PER);
    }
  };
  auto load_x = [&](int round) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int at = tid + 64 * kWaves * i;
        b[m][i] = piece(x, ldx, r0 + 16 * m + at / PER, rows - 1, round * PER + at % PER);
      }
  };
  auto put = [&](Raw16 (&from)[LOADS], int block, int round) {
    if (round == rounds - 1)
#pragma unroll
      for (int i = 0; i < LOADS; ++i) settle<T>(from[i], round * PER + (tid + 64 * kWaves * i) % PER, d);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int at = tid + 64 * kWaves * i;
      *reinterpret_cast<int4v *>(lds + (16 * block + at / PER) * PITCH + 16 * (at % PER)) = __builtin_bit_cast(int4v, from[i]);
    }
  };
  auto get = [&](int block, int step) {
    return *reinterpret_cast<const int4v *>(lds + (16 * block + (lane & 15)) * PITCH + 64 * (wave * STEPS + step) + 16 * (lane >> 4));
  };
  load_w(a[0], 0);
  load_x(0);
  load_w(a[1], 1);
  auto round_of = [&](Raw16 (&mine)[LOADS], int round) {
    put(mine, 0, round);
#pragma unroll
    for (int m = 0; m < MB; ++m) put(b[m], 1 + m, round);
    __syncthreads();
    load_x(round + 1);   // first: loads retire in order, and a wait for these must not wait for the weights behind them
    load_w(mine, round + 2);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int4v p = get(0, s);
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        const int4v q = get(1 + m, s);
        if constexpr (N == 4) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m] = product4(__int_as_float(p[e]), __int_as_float(q[e]), acc[m]);
        } else {
          acc[m] = product16<T>(p, q, acc[m]);
        }
      }
    }
    __syncthreads();
  };
  for (int round = 0; round < rounds; round += 2) {
    round_of(a[0], round);
    if (round + 1 < rounds) round_of(a[1], round + 1);
  }
  float4v(*sums)[MB][64] = reinterpret_cast<float4v(*)[MB][64]>(lds);
#pragma unroll
  for (int m = 0; m < MB; ++m) sums[wave][m][lane] = acc[m];
  __syncthreads();
  if (wave >= MB) return;
  float4v sum = sums[0][wave][lane];
#pragma unroll
  for (int o = 1; o < kWaves; ++o) sum += sums[o][wave][lane];
  const int r = r0 + 16 * wave + (lane & 15), c = v0 + 4 * (lane >> 4);
  float l[4];
  PartSum p{-INFINITY, 0.0f};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int at = min(c + e, v - 1);
    const uint8_t shown = legal && r < rows ? legal[r * ldl + at] : 1;
    const float value = sum[e] + (bias ? bias_at(bias, bias_type, at) : 0.0f);
    l[e] = c + e < v && shown ? value : -INFINITY;
    p.top = fmaxf(p.top, l[e]);
  }
  p.top = over_four(p.top, [](float q, float y) { return fmaxf(q, y); });
  const float base = base_of(p.top);
#pragma unroll
  for (int e = 0; e < 4; ++e) p.sum += exp2_of((l[e] - base) * kLog2e);
  p.sum = over_four(p.sum, [](float q, float y) { return q + y; });
  if (r >= rows) return;
  if (lane < 16) parts[r * ld_parts + blockIdx.x] = make_float2(p.top, p.sum);
  *reinterpret_cast<float4v *>(z + r * ldz + c) = float4v{l[0], l[1], l[2], l[3]};
}

struct Factors {
  const float *row_scale;
  float grad_scale;
};

// What a wave finds out about a row: its softmax's maximum and sum, its targets' weights and, where `loss` is not null, its loss.
__device__ __forceinline__ RowInfo few_row(const float2 *__restrict__ parts, int64_t ld_parts, int count,
                                           const float *__restrict__ z, int64_t ldz, const Targets &t, int64_t row, int lane,
                                           float *__restrict__ loss) {
  PartSum p{-INFINITY, 0.0f};
  for (int i = lane; i < count; i += 64) {
    const float2 v = parts[row * ld_parts + i];
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
    if (c == -2) share = whole = sum = __builtin_nanf("");
    if (c < 0) continue;
    share += a;
    whole += fabsf(a);
    if (loss) sum += a * ((p.top - z[row * ldz + c]) + kLn2 * log_sum);
  }
  share = wave_sum(share);
  whole = wave_sum(whole);
  if (loss) {
    sum = wave_sum(sum);
    if (lane == 0) loss[row] = whole != 0.0f ? sum : 0.0f;
  }
  return RowInfo{base_of(p.top), log_sum, whole != 0.0f ? share / whole : 0.0f, whole};
}

__device__ __forceinline__ float factor_of(const Factors &f, const RowInfo &i, int64_t row) {
  return i.whole != 0.0f ? i.whole * (f.row_scale ? f.row_scale[row] : 1.0f) * f.grad_scale : 0.0f;
}

// A wave per row.
__global__ __launch_bounds__(256) void k_few_rows(const float2 *__restrict__ parts, int64_t ld_parts, int count,
                                                  const float *__restrict__ z, int64_t ldz, const Targets t, int rows,
                                                  float *__restrict__ loss, RowInfo *__restrict__ info) {
  const int lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x * (int64_t)4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const RowInfo i = few_row(parts, ld_parts, count, z, ldz, t, row, lane, loss);
  if (info && lane == 0) info[row] = i;
}

// 64 columns of all rows: a wave takes every 16th row, a lane a column.  Rows' infos from k_few_rows, or (info null) found here by
// every workgroup, which saves the launch where there are few parts.
template <typename B>
__global__ __launch_bounds__(1024) void k_few_u(const float2 *__restrict__ parts, int64_t ld_parts, int count,
                                                const float *__restrict__ z, int64_t ldz, const Targets t, int rows,
                                                const RowInfo *__restrict__ info, const Factors f, float *__restrict__ loss,
                                                float *__restrict__ g, float *__restrict__ factor, B *__restrict__ gb) {
  __shared__ float share[16][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = blockIdx.x * 64;
  const int c = c0 + lane;
  float sum = 0.0f;
  for (int64_t row = wave; row < rows; row += 16) {
    const float at = c < ldz ? z[row * ldz + c] : -INFINITY;
    RowInfo i;
    if (info) i = info[row];
    else i = few_row(parts, ld_parts, count, z, ldz, t, row, lane, blockIdx.x == row % gridDim.x ? loss : nullptr);
    float u = i.share != 0.0f ? i.share * exp2_of((at - i.top) * kLog2e - i.log_sum) : 0.0f;
    if (i.whole != 0.0f)
      for (int first = 0; first < t.k; first += 64) {
        float a = 0.0f;
        const int to = first + lane < t.k ? target_of(t, row, first + lane, a) : -1;
        // the targets among these columns, in their order
        for (uint64_t hit = __ballot(to >= c0 && to < c0 + 64); hit; hit &= hit - 1) {
          const int j = __builtin_ctzll(hit);
          const float b = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), j));
          if (c == __builtin_amdgcn_readlane(to, j)) u -= b / i.whole;
        }
      }
    const float s = factor_of(f, i, row), value = s == 0.0f ? 0.0f : s * u;   // a row left out may hold anything
    if (c < ldz) g[row * ldz + c] = c < t.cols ? value : 0.0f;
    if (blockIdx.x == 0 && lane == 0) factor[row] = s;
    sum += value;
  }
  if (!gb) return;
  share[wave][lane] = sum;
  __syncthreads();
  if (wave || c >= t.cols) return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += share[i][lane];
  gb[c] = static_cast<B>(sum);
}

// 4 neighbours of a row, loaded without a branch (see load_clamped) and settled to floats, zeros past the row's end.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Four {
  T v[4];
};
template <typename T>
__device__ __forceinline__ Four<T> four_at(const T *__restrict__ row, int at, int cols) {
  return *reinterpret_cast<const Four<T> *>(row + min(at, cols - 4));
}
template <typename T>
__device__ __forceinline__ float4v settled(const Four<T> &p, int at, int cols) {
  float4v f;
#pragma unroll
  for (int e = 0; e < 4; ++e) f[e] = static_cast<float>(p.v[e]);
  const int past = at + 4 - cols;   // elements
  if (past > 0) {
    const float a = past == 1 ? f[1] : past == 2 ? f[2] : f[3], b = past == 1 ? f[2] : f[3];
    f = float4v{past < 4 ? a : 0.0f, past < 3 ? b : 0.0f, past < 2 ? f[3] : 0.0f, 0.0f};
  }
  return f;
}

template <typename T>
struct FewGrads {
  const float *g;         // (rows, ldz)
  int64_t ldz;
  const float *factor;
  const T *x, *w;
  int64_t ldx, ldw;
  int rows, d, v;
  int nd;                 // blocks of 64 of d
  int jobs_x, splits, chunk, row_blocks;   // of dx: parts of `chunk` columns, blocks of 16 MB rows
  float *share;           // (part, row, d)
  int64_t ld_share;
  int jobs;
  T *gw;
  int64_t ldgw;
};

// A job to each wave.  dx: 64 of d, 16 MB rows and a part of the columns.  dw: 64 x 64 over all rows.  Bound by memory, the weight read
// for dx and dw written: 13 rows of 2,333 into 4,168, 78 MB, 21 us.
template <typename T, int MB>
__global__ __launch_bounds__(256) void k_few_grads(const FewGrads<T> o) {
  const int lane = threadIdx.x & 63, low = lane & 15, high = lane >> 4;
  int job = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (job >= o.jobs) return;
  if (job < o.jobs_x) {
    const int d0 = 64 * (job % o.nd), part = job / o.nd % o.splits, r0 = 16 * MB * (job / o.nd / o.splits);
    const int end = min(o.v, (part + 1) * o.chunk), last = (int)o.ldz - 4 - 4 * high;   // the last 4 of a row of g
    const float *gr[MB];
#pragma unroll
    for (int m = 0; m < MB; ++m) gr[m] = o.g + min(r0 + 16 * m + low, o.rows - 1) * o.ldz + 4 * high;
    float4v acc[MB][4];
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][e] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int U = MB == 1 ? 4 : MB == 2 ? 2 : 1;
    for (int c = part * o.chunk; c < end; c += 16 * U) {
      float4v a[U][MB];
      Four<T> b[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = c + 16 * u;
#pragma unroll
        for (int m = 0; m < MB; ++m) a[u][m] = *reinterpret_cast<const float4v *>(gr[m] + min(at, last));
#pragma unroll
        for (int t = 0; t < 4; ++t) b[u][t] = four_at(o.w + min(at + 4 * high + t, o.v - 1) * o.ldw, d0 + 4 * low, o.d);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + 16 * u >= end) break;
        if (c + 16 * u > last)   // g is 0 past the columns, but may end within the 16
#pragma unroll
          for (int m = 0; m < MB; ++m) a[u][m] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const float4v w = settled(b[u][t], d0 + 4 * low, o.d);
#pragma unroll
          for (int m = 0; m < MB; ++m)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[m][e] = product4(a[u][m][t], w[e], acc[m][e]);
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int r = r0 + 16 * m + 4 * high + q;
        if (r < o.rows && d0 + 4 * low < o.d)
          *reinterpret_cast<float4v *>(o.share + ((int64_t)part * o.rows + r) * o.ld_share + d0 + 4 * low) =
              float4v{acc[m][0][q], acc[m][1][q], acc[m][2][q], acc[m][3][q]};
      }
    return;
  }
  job -= o.jobs_x;
  const int d0 = 64 * (job % o.nd), v0 = 64 * (job / o.nd);
  float4v acc[4][4];
#pragma unroll
  for (int f = 0; f < 4; ++f)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[f][e] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int U = 4;
  for (int r0 = 0; r0 < o.rows; r0 += 4 * U) {
    float4v a[U];
    Four<T> b[U];
    float factor[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = min(r0 + 4 * u + high, o.rows - 1);
      factor[u] = o.factor[r];
      a[u] = *reinterpret_cast<const float4v *>(o.g + r * o.ldz + min(v0 + 4 * low, (int)o.ldz - 4));   // columns past the end go nowhere
      b[u] = four_at(o.x + r * o.ldx, d0 + 4 * low, o.d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (r0 + 4 * u >= o.rows) break;
      const bool in = r0 + 4 * u + high < o.rows && factor[u] != 0.0f;   // rows left out count as zeros, whatever they hold
      const float4v x = settled(b[u], d0 + 4 * low, o.d);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float xe = in ? x[e] : 0.0f;
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f][e] = product4(in ? a[u][f] : 0.0f, xe, acc[f][e]);
      }
    }
  }
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int c = v0 + 4 * (4 * high + q) + f, at = d0 + 4 * low;
      if (c >= o.v || at >= o.d) continue;
      T *to = o.gw + c * o.ldgw + at;
      const Four<T> four{{static_cast<T>(acc[f][0][q]), static_cast<T>(acc[f][1][q]), static_cast<T>(acc[f][2][q]),
                       static_cast<T>(acc[f][3][q])}};
      if (at + 4 <= o.d) *reinterpret_cast<Four<T> *>(to) = four;
      else
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (at + e < o.d) to[e] = four.v[e];
    }
}

template <typename T>
__global__ __launch_bounds__(256) void k_few_join(const float *__restrict__ share, int64_t ld_share, int splits, int rows, int d,
                                                  T *__restrict__ gx, int64_t ldgx) {
  const int at = 4 * (blockIdx.x * 64 + (threadIdx.x & 63)), row = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (row >= rows || at >= d) return;
  const float *from = share + row * ld_share + at;
  float4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
  for (int p = 0; p < splits; ++p) sum += *reinterpret_cast<const float4v *>(from + (int64_t)p * rows * ld_share);
  for (int e = 0; e < 4 && at + e < d; ++e) gx[row * ldgx + at + e] = static_cast<T>(sum[e]);
}

struct Few {
  int64_t ldz, ld_share;
  int parts, nd, splits, chunk, mb, row_blocks;
  size_t z, g, stat, info, factor, share, bytes;
  explicit Few(const Call &c) {
    ldz = round_up(c.v, 32);
    parts = (int)(ldz / 16);
    nd = (int)((c.d + 63) / 64);
    ld_share = round_up(c.d, 4);
    mb = c.rows <= 16 ? 1 : c.rows <= 32 ? 2 : 4;
    row_blocks = (int)((c.rows + 16 * mb - 1) / (16 * mb));
    // about 1,200 waves of dx, each with 64 columns at least
    const int64_t want = std::max<int64_t>(1, 1200 / (nd * row_blocks));
    chunk = (int)round_up(std::max<int64_t>((c.v + want - 1) / want, 64), 16);
    splits = (int)((c.v + chunk - 1) / chunk);
    size_t at = 0;
    auto take = [&](int64_t n) {
      const size_t was = at;
      at += align256((size_t)n);
      return was;
    };
    z = take(c.rows * ldz * 4);
    stat = take(c.rows * parts * 8);
    g = c.grads() ? take(c.rows * ldz * 4) : 0;
    info = c.grads() ? take(c.rows * sizeof(RowInfo)) : 0;
    factor = c.grads() ? take(c.rows * 4) : 0;
    share = c.gx ? take(splits * c.rows * ld_share * 4) : 0;
    bytes = at;
  }
};

template <typename T>
void few(const Call &c, const Given &g, char *ws, hipStream_t st) {
  const Few s(c);
  auto floats = [&](size_t offset) { return reinterpret_cast<float *>(ws + offset); };
  float2 *stat = reinterpret_cast<float2 *>(ws + s.stat);
  const T *x = static_cast<const T *>(g.x), *w = static_cast<const T *>(g.w);
  const int rows = (int)c.rows, v = (int)c.v, d = (int)c.d;
  auto logits = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks_for(c.v, 16), blocks_for(c.rows, 16 * s.mb)), dim3(64 * kWaves), 0, st, x, g.ldx, rows,
                       w, g.ldw, v, d, g.bias, g.bias_type, g.targets.legal, g.targets.ldl, floats(s.z), s.ldz, stat,
                       (int64_t)s.parts);
    check_launch("read-out logits");
  };
  if (s.mb == 1) logits(k_few_logits<T, 1, 2048>);
  else if (s.mb == 2) logits(k_few_logits<T, 2, 1024>);
  else logits(k_few_logits<T, 4, 1024>);
  const int parts = (v + 15) / 16;
  RowInfo *info = nullptr;
  if (!c.grads() || c.rows * parts > 8192) {
    info = c.grads() ? reinterpret_cast<RowInfo *>(ws + s.info) : nullptr;
    hipLaunchKernelGGL(k_few_rows, dim3(blocks_for(c.rows, 4)), dim3(256), 0, st, stat, (int64_t)s.parts, parts, floats(s.z),
                       s.ldz, g.targets, rows, g.loss, info);
    check_launch("read-out loss");
    if (!c.grads()) return;
  }
  by_type(g.bias_type, "the bias must be float32, float16 or bfloat16", [&](auto b) {
    using B = decltype(b);
    hipLaunchKernelGGL(k_few_u<B>, dim3(blocks_for(s.ldz, 64)), dim3(1024), 0, st, stat, (int64_t)s.parts, parts, floats(s.z),
                       s.ldz, g.targets, rows, info, Factors{g.row_scale, g.grad_scale}, g.loss, floats(s.g),
                       floats(s.factor), static_cast<B *>(g.gb));
    check_launch("read-out gradient");
  });
  if (!c.gx && !c.gw) return;
  FewGrads<T> o{floats(s.g), s.ldz, floats(s.factor), x, w, g.ldx, g.ldw, rows, d, v, s.nd,
                c.gx ? s.nd * s.splits * s.row_blocks : 0, s.splits, s.chunk, s.row_blocks, floats(s.share), s.ld_share, 0,
                static_cast<T *>(g.gw), g.ldgw};
  o.jobs = o.jobs_x + (c.gw ? s.nd * ((v + 63) / 64) : 0);
  auto grads = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(blocks_for(o.jobs, 4)), dim3(256), 0, st, o); };
  if (s.mb == 1) grads(k_few_grads<T, 1>);
  else if (s.mb == 2) grads(k_few_grads<T, 2>);
  else grads(k_few_grads<T, 4>);
  check_launch("read-out gradient");
  if (!c.gx) return;
  hipLaunchKernelGGL(k_few_join<T>, dim3(blocks_for(c.d, 256), blocks_for(c.rows, 4)), dim3(256), 0, st, floats(s.share),
                     s.ld_share, s.splits, rows, d, static_cast<T *>(g.gx), g.ldgx);
  check_launch("read-out gradient");
}

}  // namespace

size_t few_ws(const Call &c) { return Few(c).bytes; }

void run_few(const Call &c, const Given &g, char *ws, hipStream_t st) {
  by_type(c.type, "", [&](auto t) { few<decltype(t)>(c, g, ws, st); });
}

}  // namespace fly
