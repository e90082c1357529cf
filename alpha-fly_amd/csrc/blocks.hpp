// Matrix products over operands laid out for the matrix cores: C[m][n] = sum_k B[m][k] A[n][k] in 16-bit floats, summed in
// float32.
//
// Both operands lie in blocks of 16 rows x 32 k in the order in which the matrix cores take them: 1 KB, lane l's 16 bytes at
// 16 l hold row l & 15, k 8 (l >> 4) .. + 7.  A wave loads a block as one contiguous kilobyte, from memory or LDS, without
// bank conflicts.  Block (r, k) of an operand lies at (r kb + k) planes; rows and k are padded with zeros to multiples of 32.
//
// Planes: 1, or 2 for float32 values v held as h + 2^-11 l with h = half(v) and l = half((v - h) 2^11), 22 bits of v where |v|
// is 2^-14 or more and an absolute 2^-36 below.  h h and h l + l h are summed apart, as their products' scales differ; l l
// is below float32's own rounding and left out.
#pragma once

#include "device.hpp"
#include "rows.hpp"

namespace fly {

typedef int int4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef bhalf bhalf8v __attribute__((ext_vector_type(8)));

template <typename H>
__device__ __forceinline__ float4v product16(int4v a, int4v b, float4v c) {
  if constexpr (std::is_same_v<H, bhalf>)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bhalf8v, a), __builtin_bit_cast(bhalf8v, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8v, a), __builtin_bit_cast(half8v, b), c, 0, 0, 0);
}

constexpr float kLow = 1.0f / 2048;   // a low plane's unit

// What a value of T is multiplied as: itself, or two halves.
template <typename T>
struct Multiplied {
  using H = T;
  static constexpr int P = 1;
};
template <>
struct Multiplied<float> {
  using H = _Float16;
  static constexpr int P = 2;
};

// v as plane `plane` of H holds it, in the low bits.
template <typename H, int P>
__device__ __forceinline__ void planes_of(float v, uint32_t (&out)[P]) {
  const H h = static_cast<H>(v);
  out[0] = to_bits(h);
  if constexpr (P == 2) out[1] = to_bits(static_cast<H>((v - static_cast<float>(h)) * 2048.0f));
}

// 16 bytes a lane from memory into LDS at `to` + 16 lane, without passing through registers.
__device__ __forceinline__ void block_to_lds(const int4v *from, int4v *to) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                   (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
// All but the last N of this wave's loads have landed, and all but the last R of its LDS reads are done.
template <int N, int R>
__device__ __forceinline__ void wait_for_blocks() {
  static_assert(N < 64 && R < 16, "the counters' range");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(%1)" ::"n"(N), "n"(R) : "memory");
}
__device__ __forceinline__ void meet_waves() {
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Workgroup L runs on XCD L mod 8: each XCD gets a contiguous run of tiles, in groups of 8 tiles of m whose tiles of n follow one
// another, so that the tiles it runs together share operands in its L2.
__device__ __forceinline__ void block_tile(int L, int tiles, int mt, int nt, int &m, int &n) {
  const int xcd = L & 7, slot = L >> 3, per = tiles >> 3, rem = tiles & 7;
  const int q = xcd * per + min(xcd, rem) + slot, group = q / (8 * nt), first = group * 8, rows = min(mt - first, 8);
  const int in = q - group * 8 * nt;
  m = first + in % rows;
  n = in / rows;
}

template <int N>
using Ahead = std::integral_constant<int, N>;

// One product's operands: blocks of 16 rows of m and n, blocks of 32 k.
struct Blocks {
  const int4v *a, *b;
  int na, mb, kb;       // blocks of n, of m and of k
  int splits;           // parts of k, each a job of its own
  int tiles, mt, nt;    // filled in at the launch
};

// The products of one launch, side by side: what one of them leaves idle at its end, the next one takes.
template <typename EP, int COUNT>
struct Products {
  Blocks of[COUNT];
  EP ep[COUNT];
};

// One plane: 16,384 x 2,333 into 4,168 270 us, 1.18e15 operations a second (the library 364 with k padded and 402 without), 256 x 256
// tiles.  The matrix cores' power is what bounds it: the gradients' products of a masked batch, whose u is mostly zeros, take a tenth
// less than those of the same batch without a mask.  Two planes: three products for one, both gradients of 4,096 rows 426 us, 1.12e15;
// there LDS bounds it as much, whose reads (two planes of both operands) take as long as the products.
//
// WN x WM waves, each FN x FM blocks of n x m; S stages of one block of k in LDS, loaded S - 1 ahead.  `ep` takes each wave's
// sums: ep.tile<FN, FM>(acc, m0, n0, lane, part, split, turn) with a wave's m0 and n0 in rows, its column part, its part of k, and
// 16 rows x 16 FN floats of LDS of its own to turn them over in.
template <typename H, int P, int WN, int WM, int FN, int FM, int S, typename EP, int COUNT>
__global__ __launch_bounds__(64 * WN * WM) void k_blocks(const Products<EP, COUNT> products) {
  constexpr int WAVES = WN * WM, BN = WN * FN, BM = WM * FM, ALL = (BN + BM) * P;
  constexpr int LOADS = (ALL + WAVES - 1) / WAVES;
  constexpr int FEWER = (WAVES - ALL % WAVES) % WAVES;   // waves with one load less
  constexpr int READS = (FN + FM) * P < 15 ? (FN + FM) * P : 15;
  __shared__ __attribute__((aligned(16))) int4v lds[S][ALL][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int index = blockIdx.x, which = 0;
  if constexpr (COUNT > 1)
    while (index >= products.of[which].tiles * products.of[which].splits) {
      index -= products.of[which].tiles * products.of[which].splits;
      ++which;
    }
  const Blocks &o = products.of[which];
  const int split = index / o.tiles, k0 = (int)((int64_t)o.kb * split / o.splits);
  int tm, tn;
  block_tile(index - split * o.tiles, o.tiles, o.mt, o.nt, tm, tn);
  const int n0 = tn * BN, m0 = tm * BM, wn = wave % WN, wm = wave / WN;
  const int kb = (int)((int64_t)o.kb * (split + 1) / o.splits) - k0;
  const int4v *src[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    // blocks past the operands' ends load their last one, whose products go nowhere
    const int at = min(wave + i * WAVES, ALL - 1), b = at / P;
    src[i] = (b < BN ? o.a + ((int64_t)min(n0 + b, o.na - 1) * o.kb + k0) * P * 64
                     : o.b + ((int64_t)min(m0 + b - BN, o.mb - 1) * o.kb + k0) * P * 64) + (at % P) * 64 + lane;
  }
  const bool fewer = FEWER > 0 && wave >= WAVES - FEWER;
  auto load = [&](int s) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < LOADS - 1 || !fewer) {
        block_to_lds(src[i], &lds[s][wave + i * WAVES][0]);
        src[i] += 64 * P;
      }
  };
  // all but the last `stages` of this wave's stages are in LDS, all but its last block's operands out of it, and every wave
  // has come this far
  auto landed = [&](auto stages) {
    constexpr int n = decltype(stages)::value;
    if constexpr (FEWER > 0 && n > 0) {
      if (fewer) wait_for_blocks<n * (LOADS - 1), READS>();
      else wait_for_blocks<n * LOADS, READS>();
    } else {
      wait_for_blocks<n * LOADS, READS>();
    }
    meet_waves();
  };
  float4v acc[FN][FM][P];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int p = 0; p < P; ++p) acc[j][i][p] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
  struct Operands {
    int4v a[FN][P], b[FM][P];
  };
  auto read = [&](Operands &r, int s) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int p = 0; p < P; ++p) r.b[i][p] = lds[s][(BN + wm * FM + i) * P + p][lane];
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int p = 0; p < P; ++p) r.a[j][p] = lds[s][(wn * FN + j) * P + p][lane];
  };
  auto multiply = [&](const Operands &r) {
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        acc[j][i][0] = product16<H>(r.a[j][0], r.b[i][0], acc[j][i][0]);
        if constexpr (P == 2) {
          acc[j][i][1] = product16<H>(r.a[j][0], r.b[i][1], acc[j][i][1]);
          acc[j][i][1] = product16<H>(r.a[j][1], r.b[i][0], acc[j][i][1]);
        }
      }
  };
  const int ahead = min(S - 1, kb);
  for (int s = 0; s < ahead; ++s) load(s);
  // Step k multiplies block k from registers while block k + 1 comes out of LDS and block k + S - 1 goes there, in the place
  // of block k - 1: every wave has read that one when it passes the barrier of step k.
  Operands even, odd;
  int k = 0;
  if (kb >= S) {
    landed(Ahead<S - 2>{});
    read(even, 0);
    for (; k + S < kb; k += 2) {   // two steps, without a branch: the reads stay in flight over the products
      landed(Ahead<S - 3>{});
      load((k + S - 1) % S);
      read(odd, (k + 1) % S);
      multiply(even);
      landed(Ahead<S - 3>{});
      load((k + S) % S);
      read(even, (k + 2) % S);
      multiply(odd);
    }
    if (k + S == kb) {
      landed(Ahead<S - 3>{});
      load((k + S - 1) % S);
      read(odd, (k + 1) % S);
      multiply(even);
      even = odd;
      ++k;
    }
    static_for<S - 2>([&](auto j) {   // the last steps, with ever fewer loads behind them
      landed(Ahead<S - 3 - decltype(j)::value>{});
      read(odd, (k + 1) % S);
      multiply(even);
      even = odd;
      ++k;
    });
    multiply(even);
  } else {
    landed(Ahead<0>{});
    for (; k < kb; ++k) {
      read(even, k);
      multiply(even);
    }
  }
  wait_for_blocks<0, 0>();
  meet_waves();   // every wave has read its last operands
  constexpr int TURN = 16 * (16 * FN + 4);   // floats: 16 rows whose pieces of 16 bytes fall into distinct banks
  static_assert(WAVES * TURN * 4 <= (int)sizeof(lds), "the tile's turn fits in the stages");
  float4v sum[FN][FM];
#pragma unroll
  for (int j = 0; j < FN; ++j)
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      sum[j][i] = acc[j][i][0];
      if constexpr (P == 2) sum[j][i] += acc[j][i][1] * kLow;
    }
  products.ep[which].template tile<FN, FM>(sum, 16 * (m0 + wm * FM), 16 * (n0 + wn * FN), lane, tn * WN + wn, split,
                           reinterpret_cast<float *>(lds) + wave * TURN);
}

// A wave's 16 rows x 16 FN columns from its lanes (row lane & 15, columns 16 j + 4 (lane >> 4) .. + 3) through its own LDS,
// so that a row's columns leave side by side: f(row, column, 4 values) in pieces of 4.
template <int FN, typename F>
__device__ __forceinline__ void turn_over(const float4v (&v)[FN], float *turn, int lane, F &&f) {
  constexpr int PITCH = 16 * FN + 4, PER = 4 * FN;   // pieces of a row
#pragma unroll
  for (int j = 0; j < FN; ++j)
    *reinterpret_cast<float4v *>(turn + (lane & 15) * PITCH + 16 * j + 4 * (lane >> 4)) = v[j];
  asm volatile("" ::: "memory");   // other lanes read what this one wrote: a wave's LDS accesses keep their order
#pragma unroll
  for (int r = 0; r < FN; ++r) {
    const int at = 64 * r + lane, row = at / PER, c = 4 * (at % PER);
    f(row, c, *reinterpret_cast<const float4v *>(turn + row * PITCH + c));
  }
  asm volatile("" ::: "memory");
}

template <typename H, int P, int WN, int WM, int FN, int FM, int S, typename EP, int COUNT>
void launch_blocks(Products<EP, COUNT> p, hipStream_t st) {
  int64_t all = 0;
  for (Blocks &o : p.of) {
    o.mt = (o.mb + WM * FM - 1) / (WM * FM);
    o.nt = (o.na + WN * FN - 1) / (WN * FN);
    o.tiles = o.mt * o.nt;
    all += (int64_t)o.mt * o.nt * o.splits;
  }
  FLY_REQUIRE(all < ((int64_t)1 << 32) / (64 * WN * WM), "product too large");   // a launch has fewer than 2^32 threads
  hipLaunchKernelGGL((k_blocks<H, P, WN, WM, FN, FM, S, EP, COUNT>), dim3((unsigned)all), dim3(64 * WN * WM), 0, st, p);
  check_launch("product of blocks");
}

}  // namespace fly
