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
#include "device.hpp"
#include "rows.hpp"

#include <cmath>

struct fly_int8 {
  int device = -1;
  int64_t n = 0, k = 0, nb = 0, kb = 0;   // channels and k, and their blocks of 16 and 64
  fly::DevArray<uint32_t> mem;            // nb x kb blocks of 256 words; scales and bias, 16 nb each, zero past n
  const void *w() const { return mem.p; }
  float *scale() const { return reinterpret_cast<float *>(mem.p + nb * kb * 256); }
  float *bias() const { return scale() + 16 * nb; }
};

namespace fly {
namespace {

typedef int int4v __attribute__((ext_vector_type(4)));
constexpr int64_t kMostK = 1 << 17;   // sums below 2^31
// A launch holds less than 2^32 threads: 64 for each block of an operand that is laid out, 256 for 16 channels of few rows.
constexpr int64_t kMostBlocks = (int64_t)1 << 26, kMostChannels = (int64_t)1 << 28;
constexpr int kFewBlocks = 12;   // blocks of k that a wave of k_int8_few holds
constexpr int kFewSpan = 48;     // and that a row has at most where the product quantises it

// Where 16-byte piece c (k 16 c .. + 15) of row r lies among the blocks.
__device__ __forceinline__ int64_t block_piece(int64_t r, int64_t c, int64_t kb) {
  return (((r >> 4) * kb + (c >> 2)) << 6) + ((c & 3) << 4) + (r & 15);
}

// int8 rows into blocks, zero past k and past the rows; a wave for each block, which leaves as one contiguous kilobyte (4,168
// x 2,333: 8.4 us against 11.6 with a thread for each piece of a row).
__global__ __launch_bounds__(256) void k_int8_pack(const int8_t *__restrict__ src, int64_t ld, int64_t rows, int64_t k,
                                                   uint32_t kb, uint32_t blocks, int4v *__restrict__ out) {
  struct __attribute__((packed)) Bytes {
    uint32_t w[4];
  };
  const uint32_t b = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (b >= blocks) return;
  const uint32_t rb = b / kb;
  const int64_t r = 16 * (int64_t)rb + (lane & 15), at = 64 * (int64_t)(b - rb * kb) + 16 * (lane >> 4);
  Bytes p = {};
  if (r < rows && at + 16 <= k) {
    p = *reinterpret_cast<const Bytes *>(src + r * ld + at);
  } else if (r < rows) {
#pragma unroll
    for (int e = 0; e < 15; ++e)
      if (at + e < k) p.w[e / 4] |= (uint32_t)(uint8_t)src[r * ld + at + e] << (8 * (e & 3));
  }
  out[(int64_t)b * 64 + lane] = int4v{(int)p.w[0], (int)p.w[1], (int)p.w[2], (int)p.w[3]};
}

// A plan's scales and bias (zero without one), zero past n.
__global__ __launch_bounds__(256) void k_int8_scales(const float *__restrict__ scale, const float *__restrict__ bias,
                                                     int64_t n, int64_t padded, float *__restrict__ out_scale,
                                                     float *__restrict__ out_bias) {
  const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
  if (i >= padded) return;
  out_scale[i] = i < n ? scale[i] : 0.0f;
  out_bias[i] = bias && i < n ? bias[i] : 0.0f;
}

// max |v| of a row piece into a running maximum that keeps NaN
__device__ __forceinline__ float abs_max(float m, float v) {
  const float x = fabsf(v);
  return x > m || x != x ? x : m;
}

struct RowScale {
  float scale, inverse;
};
__device__ __forceinline__ RowScale row_scale_of(float top) {
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
  const RowScale s = row_scale_of(top);
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
    } else if (16 * c + 16 <= k) {
      struct __attribute__((packed)) Bytes {
        uint32_t w[4];
      };
      *reinterpret_cast<Bytes *>(q + row * ldq + 16 * c) = Bytes{{w[0], w[1], w[2], w[3]}};
    } else {
      for (int e = 0; e < 15; ++e)
        if (16 * c + e < k) q[row * ldq + 16 * c + e] = (int8_t)(w[e / 4] >> (8 * (e & 3)));
    }
  }
}

// Tokens into blocks: a workgroup takes the 16 rows of a block column, a wave each, held in registers from the maximum to
// the rounding (NP pieces of 16 bytes a lane: k up to 1,024 NP / sizeof(T)); the blocks go through LDS, so that they leave
// as whole kilobytes.  Rows past the last are zero.  Bound by memory, 16,384 float32 rows of 2,333 41 us (4.7 TB/s in and
// out); few rows by a row's chain of load, maximum and store (21 rows 5 us).
template <typename T, int NP>
__global__ __launch_bounds__(1024) void k_quantize_blocks(const T *__restrict__ x, int64_t ldx, int rows, int k, int kb,
                                                          int4v *__restrict__ out, float *__restrict__ scale) {
  constexpr int N = Piece<T>::N;
  extern __shared__ __attribute__((aligned(16))) int8_t lds8[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pitch = kb * 64 + 16;   // 16 rows in distinct banks
  const int64_t row = blockIdx.x * (int64_t)16 + wave;
  const T *xr = x + row * ldx;
  Piece<T> p[NP];
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int i = lane + 64 * j;
    if (i * N < k && row < rows) p[j] = load_piece(xr, i, k, 0.0f);
    else
#pragma unroll
      for (int e = 0; e < N; ++e) p[j].v[e] = 0.0f;
  }
#pragma unroll
  for (int j = 0; j < NP; ++j)
#pragma unroll
    for (int e = 0; e < N; ++e) top = __builtin_elementwise_maximum(top, fabsf(p[j].v[e]));
  top = wave_reduce(top, [](float a, float b) { return nan_max(a, b); });
  const RowScale s = row_scale_of(top);
  if (lane == 0 && row < rows) scale[row] = s.scale;
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int i = lane + 64 * j;
    if (i * N < kb * 64) {
      uint32_t w[N / 4] = {};
#pragma unroll
      for (int e = 0; e < N; ++e) w[e / 4] |= quantised(p[j].v[e], s.inverse) << (8 * (e & 3));
      uint32_t *to = reinterpret_cast<uint32_t *>(lds8 + wave * pitch + i * N);
#pragma unroll
      for (int d = 0; d < N / 4; ++d) to[d] = w[d];
    }
  }
  __syncthreads();
  for (int b = wave; b < kb; b += 16)
    out[((int64_t)blockIdx.x * kb + b) * 64 + lane] =
        *reinterpret_cast<const int4v *>(lds8 + (lane & 15) * pitch + b * 64 + (lane >> 4) * 16);
}

// An output in float32, from which it rounds to its type.  The value stands for itself: the compiler would round some kernels'
// float16 outputs from the exact product and sum instead, and a row's bits would depend on the batch around it.
__device__ __forceinline__ float scaled(int sum, float scale, float bias) {
  float v = fmaf((float)sum, scale, bias);
  asm("" : "+v"(v));
  return v;
}

// 16 bytes a lane from memory into LDS at `to` + 16 lane, without passing through registers.
__device__ __forceinline__ void to_lds(const int4v *from, int4v *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
// All but the last N of this wave's loads have landed, and all but the last R of its LDS reads are done.
template <int N, int R>
__device__ __forceinline__ void wait_for() {
  static_assert(N < 64 && R < 16, "the counters' range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(%1)" ::"n"(N), "n"(R) : "memory");
}
__device__ __forceinline__ void meet() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Workgroup L runs on XCD L mod 8: each XCD gets a contiguous run of tiles, in groups of 8 token tiles whose channel tiles
// follow one another, so that the tiles it runs together share operands in its L2.
__device__ __forceinline__ void int8_tile(int tiles, int mt, int nt, int &m, int &n) {
  const int L = blockIdx.x, xcd = L & 7, slot = L >> 3, per = tiles >> 3, rem = tiles & 7;
  const int q = xcd * per + min(xcd, rem) + slot, group = q / (8 * nt), first = group * 8, rows = min(mt - first, 8);
  const int in = q - group * 8 * nt;
  m = first + in % rows;
  n = in / rows;
}

template <int N>
using Stages = std::integral_constant<int, N>;

// WN x WM waves, each FN x FM blocks of channels x tokens; S stages of one block of k in LDS, loaded S - 1 ahead.  16,384 rows
// of 2,333 into 4,168 run at 1.79e15 operations a second, 178 us.  The main loop alone on a long k reaches 2.83e15 with random
// operands, by the matrix cores' clock (3.52e15 with constant ones): 113 of the 178 us.  The other 65 are the tiles' filling,
// emptying and stores, which only the CU's second workgroup covers.  Small products are bound by that chain alone: 1,120
// rows 20 us, where the bytes take 7.6.
template <typename T, int WN, int WM, int FN, int FM, int S>
__global__ __launch_bounds__(64 * WN * WM) void k_int8_gemm(const int4v *__restrict__ w, const int4v *__restrict__ q,
                                                            const float *__restrict__ row_scale,
                                                            const float *__restrict__ scale, const float *__restrict__ bias,
                                                            int rows, int n, int nb, int mb, int kb, int tiles, int mt,
                                                            int nt, T *__restrict__ y, int64_t ldy) {
  constexpr int WAVES = WN * WM, BN = WN * FN, BM = WM * FM;
  constexpr int LOADS = (BN + BM + WAVES - 1) / WAVES;
  constexpr int FEWER = (WAVES - (BN + BM) % WAVES) % WAVES;   // waves with one load less
  __shared__ __attribute__((aligned(16))) int4v lds[S][BN + BM][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int tm, tn;
  int8_tile(tiles, mt, nt, tm, tn);
  const int n0 = tn * BN, m0 = tm * BM, wn = wave % WN, wm = wave / WN;
  const int4v *src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    // blocks past the operands' ends load their last one, whose products go nowhere
    const int b = min(wave + i * WAVES, BN + BM - 1);
    src[i] = (b < BN ? w + (int64_t)min(n0 + b, nb - 1) * kb * 64 : q + (int64_t)min(m0 + b - BN, mb - 1) * kb * 64) + lane;
  }
  const bool fewer = FEWER > 0 && wave >= WAVES - FEWER;
  auto load = [&](int s) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < LOADS - 1 || !fewer) {
        to_lds(src[i], &lds[s][wave + i * WAVES][0]);
        src[i] += 64;
      }
  };
  // all but the last `stages` of this wave's stages are in LDS, all but its last block's operands out of it, and every wave
  // has come this far.  The products need those operands anyway, but nothing else keeps them on this side of the barrier.
  auto landed = [&](auto stages) {
    constexpr int n = decltype(stages)::value;
    if constexpr (FEWER > 0 && n > 0) {
      if (fewer) wait_for<n * (LOADS - 1), FN + FM>();
      else wait_for<n * LOADS, FN + FM>();
    } else {
      wait_for<n * LOADS, FN + FM>();
    }
    meet();
  };
  int4v acc[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) acc[j][i] = int4v{0, 0, 0, 0};
  struct Operands {
    int4v w[FN], q[FM];
  };
  auto read = [&](Operands &o, int s) {
#pragma unroll
    for (int i = 0; i < FM; ++i) o.q[i] = lds[s][BN + wm * FM + i][lane];
#pragma unroll
    for (int j = 0; j < FN; ++j) o.w[j] = lds[s][wn * FN + j][lane];
  };
  const int ahead = min(S - 1, kb);
  for (int s = 0; s < ahead; ++s) load(s);
  // Step k multiplies block k from registers while block k + 1 comes out of LDS and block k + S - 1 goes there, in the place
  // of block k - 1: every wave has read that one when it passes the barrier of step k.
  auto multiply = [&](const Operands &o) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(o.w[j], o.q[i], acc[j][i], 0, 0, 0);
  };
  Operands even, odd;
  int k = 0;
  if (kb >= S) {
    landed(Stages<S - 2>{});
    read(even, 0);
    for (; k + S < kb; k += 2) {   // two steps, without a branch: the reads stay in flight over the products
      landed(Stages<S - 3>{});
      load((k + S - 1) % S);
      read(odd, (k + 1) % S);
      multiply(even);
      landed(Stages<S - 3>{});
      load((k + S) % S);
      read(even, (k + 2) % S);
      multiply(odd);
    }
    if (k + S == kb) {
      landed(Stages<S - 3>{});
      load((k + S - 1) % S);
      read(odd, (k + 1) % S);
      multiply(even);
      even = odd;
      ++k;
    }
    static_for<S - 2>([&](auto j) {   // the last steps, with ever fewer loads behind them
      landed(Stages<S - 3 - decltype(j)::value>{});
      read(odd, (k + 1) % S);
      multiply(even);
      even = odd;
      ++k;
    });
    multiply(even);
  } else {
    landed(Stages<0>{});
    for (; k < kb; ++k) {
      read(even, k);
      multiply(even);
    }
  }
  // Each wave turns its 16 tokens x 16 FN channels at a time over in LDS, so that a token's channels leave side by side: with
  // every lane storing its own 4, the 16,384-row product into float16 spent 100 us of 237 on 32-byte pieces of rows.
  constexpr int PITCH = 16 * FN * sizeof(T) + 16, PER = 16 / sizeof(T), LANES = 16 * FN / PER;   // lanes for a token's channels
  static_assert(WAVES * 16 * PITCH <= sizeof(lds), "the tile's turn fits in the stages");
  wait_for<0, 0>();
  meet();   // every wave has read its last operands
  char *turn = reinterpret_cast<char *>(lds) + wave * 16 * PITCH;
  float4 t[FN], b[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    const int c = 16 * min(n0 + wn * FN + j, nb - 1) + 4 * (lane >> 4);
    t[j] = *reinterpret_cast<const float4 *>(scale + c);
    b[j] = *reinterpret_cast<const float4 *>(bias + c);
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int first = 16 * (m0 + wm * FM + i);
    const float sm = row_scale[min(first + (lane & 15), rows - 1)];
    struct __attribute__((aligned(4 * sizeof(T)))) Four {
      T v[4];
    };
#pragma unroll
    for (int j = 0; j < FN; ++j)
      *reinterpret_cast<Four *>(turn + (lane & 15) * PITCH + (16 * j + 4 * (lane >> 4)) * sizeof(T)) =
          Four{{static_cast<T>(scaled(acc[j][i][0], sm * t[j].x, b[j].x)),
                static_cast<T>(scaled(acc[j][i][1], sm * t[j].y, b[j].y)),
                static_cast<T>(scaled(acc[j][i][2], sm * t[j].z, b[j].z)),
                static_cast<T>(scaled(acc[j][i][3], sm * t[j].w, b[j].w))}};
    asm volatile("" ::: "memory");   // other lanes read what this one wrote: a wave's LDS accesses keep their order
#pragma unroll
    for (int r = 0; r < 16 * LANES; r += 64) {
      const int token = (r + lane) / LANES, piece = (r + lane) % LANES, m = first + token;
      const int c = 16 * (n0 + wn * FN) + piece * PER;
      if (token >= 16 || m >= rows || c >= n) continue;
      const Raw16 v = *reinterpret_cast<const Raw16 *>(turn + token * PITCH + piece * 16);
      T *out = y + m * ldy + c;
      if (c + PER <= n) *reinterpret_cast<Raw16 *>(out) = v;
      else
#pragma unroll
        for (int e = 0; e < PER; ++e)
          if (c + e < n)
            out[e] = __builtin_bit_cast(T, (std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>)(
                                               v.v[e * sizeof(T) / 4] >> (8 * (e * sizeof(T) % 4))));
    }
    asm volatile("" ::: "memory");
  }
}

template <typename T, int WN, int WM, int FN, int FM, int S>
void int8_gemm(const fly_int8 &p, const int4v *q, const float *row_scale, int64_t rows, T *y, int64_t ldy, hipStream_t st) {
  const int mb = (int)((rows + 15) / 16), mt = (mb + WM * FM - 1) / (WM * FM), nt = (int)((p.nb + WN * FN - 1) / (WN * FN));
  FLY_REQUIRE((int64_t)mt * nt < (int64_t)1 << 32 >> 9, "product too large");   // at up to 512 threads
  hipLaunchKernelGGL((k_int8_gemm<T, WN, WM, FN, FM, S>), dim3(mt * nt), dim3(64 * WN * WM), 0, st,
                     reinterpret_cast<const int4v *>(p.w()), q, row_scale, p.scale(), p.bias(), (int)rows, (int)p.n,
                     (int)p.nb, mb, (int)p.kb, mt * nt, mt, nt, y, ldy);
  check_launch("8-bit product");
}

// Few rows, R blocks of 16 of them: a workgroup has C blocks of 16 channels, 4 waves for each, and a wave every fourth block
// of k, whose weights go straight from memory to the matrix cores; the waves' integer sums meet in LDS.  The work is the
// weights' way here, so their loads go first.  X = void: the rows come quantised from the workspace.  Else every workgroup
// quantises them for itself, a wave per row, while its weights are on their way: one launch, and no workspace.  C = 1 up to 4
// rows, one for each wave, 261 workgroups for 4,168 channels (1 row of 2,333 4.9 us, C = 4 5.2; 4 rows of 3,000 into 500 4.9
// against 5.3); C = 4 past that, whose 16 waves share the rows (8 rows of 2,333 6.0 us against 7.1, 16 rows 7.7 against 10.3).
template <typename X, typename T, int C, int R>
__global__ __launch_bounds__(256 * C) void k_int8_few(const int4v *__restrict__ w, const void *__restrict__ in, int64_t ldx,
                                                      const float *__restrict__ row_scale,
                                                      const float *__restrict__ scale, const float *__restrict__ bias,
                                                      int rows, int n, int k, int nb, int kb, T *__restrict__ y,
                                                      int64_t ldy) {
  constexpr bool kQuantise = !std::is_void_v<X>;
  extern __shared__ int4v blocks[];   // the quantised rows, R x kb blocks
  __shared__ int4v sums[C][4][R][64];
  __shared__ float s_scale[16 * R];
  // one number for the wave: its loads and products stand behind scalar branches.  The matrix cores do not look at exec, so a
  // product behind a mask is skipped only where the compiler happens to keep a branch over it.
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = wave & 3, cb = blockIdx.x * C + (wave >> 2);
  const int4v *wb = w + (int64_t)min(cb, nb - 1) * kb * 64 + lane;
  int4v fw[kFewBlocks];
  auto fetch = [&](int b0) {
#pragma unroll
    for (int j = 0; j < kFewBlocks; ++j)
      if (b0 + 4 * j < kb) fw[j] = wb[(b0 + 4 * j) * 64];
  };
  fetch(part);
  if constexpr (kQuantise) {
    constexpr int N = Piece<X>::N, kPieces = 48 / N;   // of a row, that a lane holds
    char *bytes = reinterpret_cast<char *>(blocks);
    for (int row = wave; row < rows; row += 4 * C) {
      const X *xr = static_cast<const X *>(in) + row * ldx;
      Piece<X> p[kPieces];
      float top = 0.0f;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int i = lane + 64 * j;
        if (i * N < k) p[j] = load_piece(xr, i, k, 0.0f);
        else
#pragma unroll
          for (int e = 0; e < N; ++e) p[j].v[e] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < kPieces; ++j)
#pragma unroll
        for (int e = 0; e < N; ++e) top = __builtin_elementwise_maximum(top, fabsf(p[j].v[e]));
      top = wave_reduce(top, [](float a, float b) { return nan_max(a, b); });
      const RowScale s = row_scale_of(top);
      if (lane == 0) s_scale[row] = s.scale;
      char *to_row = bytes + (row >> 4) * kb * 1024 + (row & 15) * 16;
#pragma unroll
      for (int j = 0; j < kPieces; ++j) {
        const int at = (lane + 64 * j) * N;   // k of the piece's first element
        if (at < kb * 64) {
          uint32_t q[N / 4] = {};
#pragma unroll
          for (int e = 0; e < N; ++e) q[e / 4] |= quantised(p[j].v[e], s.inverse) << (8 * (e & 3));
          uint32_t *to = reinterpret_cast<uint32_t *>(to_row + (at >> 6) * 1024 + ((at >> 4) & 3) * 256 + (at & 15));
#pragma unroll
          for (int d = 0; d < N / 4; ++d) to[d] = q[d];
        }
      }
    }
    __syncthreads();
  }
  int4v acc[R];
#pragma unroll
  for (int i = 0; i < R; ++i) acc[i] = int4v{0, 0, 0, 0};
  for (int b0 = part; b0 < kb; b0 += 4 * kFewBlocks) {
    if (b0 != part) fetch(b0);
#pragma unroll
    for (int j = 0; j < kFewBlocks; ++j)
      if (b0 + 4 * j < kb)
#pragma unroll
        for (int i = 0; i < R; ++i) {
          const int at = (i * kb + b0 + 4 * j) * 64 + lane;
          int4v fq;
          if constexpr (kQuantise) fq = blocks[at];
          else fq = static_cast<const int4v *>(in)[at];
          acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(fw[j], fq, acc[i], 0, 0, 0);
        }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) sums[wave >> 2][part][i][lane] = acc[i];
  __syncthreads();
  const int m = 16 * part + (lane & 15), c = 16 * cb + 4 * (lane >> 4);   // a wave for each block of rows
  if (part >= R || cb >= nb || m >= rows) return;
  int4v sum = sums[wave >> 2][0][part][lane];
#pragma unroll
  for (int o = 1; o < 4; ++o) sum += sums[wave >> 2][o][part][lane];
  const float sm = kQuantise ? s_scale[m] : row_scale[m];
  const float4 t = *reinterpret_cast<const float4 *>(scale + c), b = *reinterpret_cast<const float4 *>(bias + c);
  const float v[4] = {scaled(sum[0], sm * t.x, b.x), scaled(sum[1], sm * t.y, b.y), scaled(sum[2], sm * t.z, b.z),
                      scaled(sum[3], sm * t.w, b.w)};
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (c + r < n) y[m * ldy + c + r] = static_cast<T>(v[r]);
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
  const int64_t blocks = (rows + 15) / 16 * kb;
  FLY_REQUIRE(blocks < kMostBlocks, "operand too large");
  hipLaunchKernelGGL(k_int8_pack, dim3(blocks_for(blocks, 4)), dim3(256), 0, st, src, ld, rows, k, (uint32_t)kb,
                     (uint32_t)blocks, static_cast<int4v *>(out));
  check_launch("8-bit blocks");
}

// Rows into blocks and their scales: from registers up to 3,072 columns, whose 16 rows also fit LDS (16,384 rows of 2,333
// float32 41 us against 87 by the kernel that reads them twice and stores 16 bytes at a time).
template <typename X>
void quantise_blocks(const fly_int8 &p, const X *x, int64_t ldx, int64_t rows, int4v *out, float *scale, hipStream_t st) {
  const int64_t per = 1024 / (int64_t)sizeof(X), span = p.kb * 64;   // elements of a wave's 64 pieces, and of a row
  auto held = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(blocks_for(rows, 16)), dim3(1024), 16 * (size_t)(span + 16), st, x, ldx, (int)rows,
                       (int)p.k, (int)p.kb, out, scale);
  };
  constexpr int kMost = sizeof(X) == 4 ? 12 : 6;
  if (span <= kMost / 3 * per) held(k_quantize_blocks<X, kMost / 3>);
  else if (span <= kMost * per) held(k_quantize_blocks<X, kMost>);
  else
    hipLaunchKernelGGL((k_quantize<X, true>), dim3(blocks_for(rows, 4)), dim3(256), 0, st, x, ldx, rows, p.k, p.kb,
                       reinterpret_cast<int8_t *>(out), (int64_t)0, scale);
  check_launch("quantised rows");
}

size_t token_bytes(const fly_int8 &p, int64_t rows) { return (size_t)round_up(rows, 16) * p.kb * 64; }

size_t int8_ws(const fly_int8 &p, int64_t rows) {
  return align256(token_bytes(p, rows)) + align256((size_t)rows * sizeof(float));
}

// Whether a call quantises its rows in the product itself (k_int8_few): up to 32 rows of at most 3,072 columns (a wave's
// registers; 96 KB of blocks) into at most 8,192 channels, over which every workgroup repeats the work.  Measured, us of the
// kernels in a graph against the two of the other path: 4,168 channels over 2,333: 1 row 4.9 against 8.6, 8 rows 6.0 against
// 8.9, 16 rows 7.7 against 9.6, 32 rows 10.6 against 12.3; the second launch costs the host another 4.  17,937 channels over
// 838: 1 row 7.1 against 5.9, 16 rows 11.3 against 7.0; 12,000 channels 1 row 4.5 against 5.9, 32 rows 8.8 against 8.1.
bool quantises_few(const fly_int8 &p, int32_t x_type, int64_t rows) {
  return x_type != FLY_I8 && rows <= 32 && p.nb <= 512 && p.kb <= kFewSpan;
}

template <typename X, typename T, int C, int R>
void int8_few(const fly_int8 &p, const void *x, int64_t ldx, const float *row_scale, int64_t rows, T *y, int64_t ldy,
              hipStream_t st) {
  const size_t lds = std::is_void_v<X> ? 0 : (size_t)R * p.kb * 1024;
  constexpr auto kernel = &k_int8_few<X, T, C, R>;
  if (lds > 32 * 1024) allow_lds(kernel, R * kFewSpan * 1024);
  hipLaunchKernelGGL(kernel, dim3(blocks_for(p.nb, C)), dim3(256 * C), lds, st, reinterpret_cast<const int4v *>(p.w()), x,
                     ldx, row_scale, p.scale(), p.bias(), (int)rows, (int)p.n, (int)p.k, (int)p.nb, (int)p.kb, y, ldy);
  check_launch("8-bit product of few rows");
}

// The product of rows in blocks.  Measured, us of the product (2,333 into 4,168 where nothing else is said):
// * up to 16 rows, a workgroup for each 16 channels (k_int8_few): 16 rows 5.2;
// * tiles of 64 x 64 while there are at most 512 of them: 384 rows 12.0 against 13.5 (128 x 128), 1,120 rows of 200 into 500
//   4.2 against 5.4; but 512 rows 14.7 against 13.5;
// * 128 x 128 while there are at most 256, one for each CU: 600 rows 14.0 against 17.6 (192 x 128); but 900 rows 20.2 against
//   19.2;
// * else 192 channels x 128 tokens (float32: 1,120 rows 19.4 against 21.2 with 128 x 128, 2,048 rows 28.9 against 31.9) or
//   128 x 192 (16 bits, so that a wave's share of a token is still 128 bytes: 517 rows of 838 into 17,937 16.6 against 17.6
//   with 192 x 128, 16,384 rows of 1,024 into 4,096 99 against 108), two workgroups of 8 waves per CU.  256 x 256 in one
//   workgroup of 16 waves: 16,384 rows 178 against 181, 4,096 rows 65 against 48.
template <typename T>
void int8_product(const fly_int8 &p, const int4v *q, const float *row_scale, int64_t rows, T *y, int64_t ldy,
                  hipStream_t st) {
  auto tiles = [&](int side) { return ((rows + side - 1) / side) * ((p.n + side - 1) / side); };
  if (rows <= 16) int8_few<void, T, 1, 1>(p, q, 0, row_scale, rows, y, ldy, st);
  else if (tiles(64) <= 512) int8_gemm<T, 2, 2, 2, 2, 6>(p, q, row_scale, rows, y, ldy, st);
  else if (tiles(128) <= 256) int8_gemm<T, 2, 4, 4, 2, 4>(p, q, row_scale, rows, y, ldy, st);
  else if constexpr (sizeof(T) == 4) int8_gemm<T, 4, 2, 3, 4, 4>(p, q, row_scale, rows, y, ldy, st);
  else int8_gemm<T, 2, 4, 4, 3, 4>(p, q, row_scale, rows, y, ldy, st);
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
      in_slices(rows, 64, [&](int64_t r, int64_t n) {
        hipLaunchKernelGGL((k_quantize<T, false>), dim3(blocks_for(n, 4)), dim3(256), 0, as_stream(stream),
                           cols ? static_cast<const T *>(x) + r * ldx : nullptr, ldx, n, cols, (int64_t)0,
                           cols ? q + r * ldq : nullptr, ldq, scale + r);
        check_launch("quantised rows");
      });
    });
  });
}

extern "C" int fly_int8_create(const int8_t *w, int64_t ldw, const float *scale, const float *bias, int64_t n,
                               int64_t k, void *stream, fly_int8 **out) {
  return guard([&] {
    FLY_REQUIRE(out != nullptr, "out is null");
    *out = nullptr;
    FLY_REQUIRE(n >= 1 && k >= 1 && k < kMostK && n < kMostChannels && ldw >= k, "bad size");
    FLY_REQUIRE((n + 15) / 16 * ((k + 63) / 64) < kMostBlocks, "bad size: the weight is too large");
    FLY_REQUIRE(w && scale, "null pointer");
    hipStream_t st = as_stream(stream);
    auto p = std::make_unique<fly_int8>();
    p->device = current_device();
    p->n = n;
    p->k = k;
    p->nb = (n + 15) / 16;
    p->kb = (k + 63) / 64;
    p->mem.alloc((size_t)p->nb * (p->kb * 256 + 32));
    pack(w, ldw, n, k, p->kb, p->mem.p, st);
    hipLaunchKernelGGL(k_int8_scales, dim3(blocks_for(p->nb * 16, 256)), dim3(256), 0, st, scale, bias, n, p->nb * 16,
                       p->scale(), p->bias());
    check_launch("8-bit scales");
    FLY_HIP(hipStreamSynchronize(st));
    *out = p.release();
  });
}

extern "C" int fly_int8_destroy(fly_int8 *p) {
  return guard([&] { delete p; });
}

extern "C" size_t fly_int8_workspace(const fly_int8 *p, int32_t x_type, int64_t rows) {
  return p && rows > 0 && !quantises_few(*p, x_type, rows) ? int8_ws(*p, rows) : 0;
}

extern "C" int fly_int8_linear(const fly_int8 *p, const void *x, int32_t x_type, int64_t ldx, const float *x_scale,
                               int64_t rows, void *y, int32_t y_type, int64_t ldy, void *ws, size_t ws_bytes,
                               void *stream) {
  return guard([&] {
    FLY_REQUIRE(p != nullptr, "the 8-bit plan is null");
    FLY_REQUIRE(current_device() == p->device, "the 8-bit plan lives on another device");
    FLY_REQUIRE(rows >= 0 && rows < (int64_t)1 << 24, "rows out of range");
    FLY_REQUIRE(x_type >= FLY_F32 && x_type <= FLY_I8, "x must be float32, float16, bfloat16 or int8");
    FLY_REQUIRE((x_type == FLY_I8) == (x_scale != nullptr), "8-bit rows come with their scales, other rows without");
    if (!rows) return;
    FLY_REQUIRE(x && y && ldx >= p->k && ldy >= p->n, "bad argument");
    hipStream_t st = as_stream(stream);
    by_float(y_type, "y must be float32, float16 or bfloat16", [&](auto yt) {
      using T = decltype(yt);
      if (quantises_few(*p, x_type, rows)) {
        by_float(x_type, "", [&](auto xt) {
          using X = decltype(xt);
          T *out = static_cast<T *>(y);
          if (rows <= 4) int8_few<X, T, 1, 1>(*p, x, ldx, nullptr, rows, out, ldy, st);
          else if (rows <= 16) int8_few<X, T, 4, 1>(*p, x, ldx, nullptr, rows, out, ldy, st);
          else int8_few<X, T, 4, 2>(*p, x, ldx, nullptr, rows, out, ldy, st);
        });
        return;
      }
      FLY_REQUIRE(ws && ws_bytes >= int8_ws(*p, rows) && aligned(ws, 256), "workspace too small or misaligned");
      float *made = reinterpret_cast<float *>(static_cast<char *>(ws) + align256(token_bytes(*p, rows)));
      if (x_type == FLY_I8) pack(static_cast<const int8_t *>(x), ldx, rows, p->k, p->kb, ws, st);
      else
        by_float(x_type, "", [&](auto xt) {
          quantise_blocks(*p, static_cast<const decltype(xt) *>(x), ldx, rows, static_cast<int4v *>(ws), made, st);
        });
      int8_product<T>(*p, static_cast<const int4v *>(ws), x_scale ? x_scale : made, rows, static_cast<T *>(y), ldy, st);
    });
  });
}
