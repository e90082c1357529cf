// A teacher's top logits, and distillation from them.
//
//   top      of each row of z the K largest visible logits in falling order (ties: the lower column first), and
//            tail = log sum exp(z_j / T) over the visible columns that are not listed.
//   distill  S = the listed columns, rest = the other visible ones.  With temperature T,
//              p_i = exp(v_i / T - A), p_t = exp(tail - A), A = log sum of all of them      (teacher)
//              q_i = exp(z_i / T - B), q_t = sum over the rest, B = log sum over all          (student)
//            L = T^2 [ sum_S (p log(p/q) - p + q) + (p_t log(p_t/q_t) - p_t + q_t) ].
//            The -p + q add to nothing over all classes; with them an error e of B changes L by e (sum q - 1) = 0 in
//            first order instead of by e, so float32 keeps a small divergence's digits.
//              dL/dz_j = T (q_j - p_j) on S,  T exp(z_j / T - lse_rest) (q_t - p_t) outside.
//            q_t is summed over the rest itself, never as 1 - sum q.
// Rows, maxima and sums are float32 whatever the logits' type; gradients round once, on their store.
#include "row_rules.hpp"
#include "rows.hpp"

namespace fly {
namespace {

constexpr int kMostListed = 256;             // no chess position has over 218 legal moves
constexpr int64_t kMostColumns = 1 << 20;    // a bit for each column in LDS: 128 KB

// A row's 16-byte pieces, piece tid + j * blockDim for j < NV in a thread's registers (RES), or read again at each pass; a
// last piece that is not whole belongs to thread 0.
template <typename T, int NV, bool RES>
struct Row {
  static constexpr int N = Piece<T>::N;
  const T *z;
  const uint8_t *seen;
  int full, left;   // whole pieces, and elements behind them
  Raw16 kept[RES ? NV : 1], last;

  __device__ __forceinline__ Row(const T *row, const uint8_t *mask, int cols)
      : z(row), seen(mask), full(cols / N), left(threadIdx.x == 0 ? cols % N : 0) {
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        kept[j] = i < full ? load_whole(z, i) : nothing();
      }
      if (seen)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int i = threadIdx.x + j * blockDim.x;
          if (i < full) mask_whole<T>(kept[j], seen, i);
        }
    }
    last = nothing();
    if (left) {
      last = load_last(z, full, left);
      if (seen) mask_last<T>(last, seen, full, left);
    }
  }
  // The next pass takes the pieces apart again: left alone, the compiler keeps every element of 16 bits as a float of its
  // own from pass to pass, twice the registers.
  __device__ __forceinline__ void forget() {
    if constexpr (RES && sizeof(T) == 2)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) asm volatile("" : "+v"(kept[j].v[w]));
  }
  static __device__ __forceinline__ Raw16 nothing() {
    constexpr uint32_t w = sizeof(T) == 4 ? kLowest<T> : kLowest<T> * 0x10001u;
    return Raw16{{w, w, w, w}};
  }
  // f(piece number, piece) for whole waves at once: lanes past the row's end have a piece of -inf
  template <typename F>
  __device__ __forceinline__ void each_wave(F &&f) {
    const int first = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u), lane = threadIdx.x & 63;
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (first + j * (int)blockDim.x < full) f(first + j * (int)blockDim.x + lane, kept[j]);
    } else {
      for (int i0 = first; i0 < full; i0 += blockDim.x) {
        Raw16 p = nothing();
        if (i0 + lane < full) {
          p = load_whole(z, i0 + lane);
          if (seen) mask_whole<T>(p, seen, i0 + lane);
        }
        f(i0 + lane, p);
      }
    }
    if (first == 0 && __builtin_amdgcn_readfirstlane(left)) f(full, last);   // of -inf but in lane 0
  }
  // f(logit, column)
  template <typename F>
  __device__ __forceinline__ void values(F &&f) {
    each([&](int, int i, const Raw16 &p) {
#pragma unroll
      for (int e = 0; e < N; ++e) f(element<T>(p, e), i * N + e);
    });
  }
  template <typename F>
  __device__ __forceinline__ void values_wave(F &&f) {
    each_wave([&](int i, const Raw16 &p) {
#pragma unroll
      for (int e = 0; e < N; ++e) f(element<T>(p, e), i * N + e);
    });
  }
  // f(j, piece number, piece) for this thread's pieces, columns that do not exist at -inf; j = -1 for the last one where it
  // is not whole (a constant after inlining)
  template <typename F>
  __device__ __forceinline__ void each(F &&f) {
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int i = threadIdx.x + j * blockDim.x;
        if (i < full) f(j, i, kept[j]);
      }
    } else {
      for (int i = threadIdx.x; i < full; i += blockDim.x) {
        Raw16 p = load_whole(z, i);
        if (seen) mask_whole<T>(p, seen, i);
        f(0, i, p);
      }
    }
    if (left) f(-1, full, last);
  }
};

// A short row, column tid + j * blockDim for j < E in a thread's registers: every wave holds as many.
template <typename T, int E>
struct Spread {
  float kept[E];
  int cols;
  __device__ __forceinline__ Spread(const T *z, const uint8_t *seen, int n) : cols(n) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
      const int c = threadIdx.x + j * blockDim.x;
      kept[j] = c < cols && (!seen || seen[c]) ? static_cast<float>(z[c]) : -INFINITY;
    }
  }
  template <typename F>
  __device__ __forceinline__ void values(F &&f) {
#pragma unroll
    for (int j = 0; j < E; ++j) f(kept[j], threadIdx.x + j * blockDim.x);
  }
  template <typename F>
  __device__ __forceinline__ void values_wave(F &&f) { values(f); }
  __device__ __forceinline__ void forget() {}
};

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMostFloat = 3.4028234663852886e38f;

__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * kLog2e); }
__device__ __forceinline__ float ln_of(float x) { return log2_of(x) * kLn2; }

// ---- top logits ----------------------------------------------------------------------------------------------------

// A float's place in the order of numbers as an unsigned: NaN above all, the zeros alike, 0 for a column not seen.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == -INFINITY) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);   // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

constexpr int kMostCandidates = 1024;

// What a workgroup of k_top keeps in LDS besides these, 128 entries for each wave (at most 1,024 in the first): the joined
// list, and the waves' own lists, whose place a histogram and the candidates that are not listed (`spare`, by rank) take
// later.
struct TopShared {
  alignas(16) float share[2 * 16];
  uint32_t wave[16];
  uint32_t count, prefix, need;
};
__host__ __device__ inline int top_list(int waves) {
  return waves * kWaveCandidates < kMostCandidates ? waves * kWaveCandidates : kMostCandidates;
}

__device__ __forceinline__ uint64_t candidate(float v, int32_t col) {   // larger is better: the key, then the lower column
  return (uint64_t)order_key(v) << 32 | (uint32_t)~(uint32_t)col;
}

// 64 candidates of a wave in falling order
__device__ __forceinline__ uint64_t sort_wave(uint64_t v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d; d >>= 1) {
      const uint64_t o = __shfl_xor((unsigned long long)v, d);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0 || size == 64);   // this lane keeps the larger one
      v = (o > v) == larger ? o : v;
    }
  return v;
}

// The K largest of the list's `count` candidates in their places, the others to `spare`, each by its rank: the list's own
// order is that of the waves and lanes that met its entries, and nothing may depend on it.  Each 64 are sorted by a
// wave; an entry's rank is its place among them plus, in each of the other 64, the place that a search finds for it.
template <typename T>
__device__ __forceinline__ void rank_candidates(uint64_t *list, float *spare, int count, int k, const T *z, float *values,
                                                int32_t *index) {
  const int lane = threadIdx.x & 63, parts = (count + 63) >> 6;
  for (int p = threadIdx.x >> 6; p < parts; p += blockDim.x >> 6) {
    const uint64_t v = sort_wave(p * 64 + lane < count ? list[p * 64 + lane] : 0);
    list[p * 64 + lane] = v;
  }
  __syncthreads();
  for (int p = threadIdx.x >> 6; p < parts; p += blockDim.x >> 6) {
    const uint64_t mine = list[p * 64 + lane];
    int rank = lane;
    for (int o = 0; o < parts; ++o) {
      if (o == p) continue;
      const uint64_t *other = list + o * 64;
      int before = 0;
#pragma unroll
      for (int step = 32; step; step >>= 1)
        if (other[before + step - 1] > mine) before += step;
      rank += before + (other[before] > mine);   // before <= 63
    }
    if (mine == 0) continue;   // behind the last candidate
    const int32_t col = (int32_t)~(uint32_t)mine;
    const float v = static_cast<float>(z[col]);
    if (rank < k) {
      values[rank] = v;
      index[rank] = col;
    } else {
      spare[rank - k] = v;
    }
  }
  for (int i = count + threadIdx.x; i < k; i += blockDim.x) {
    values[i] = -INFINITY;
    index[i] = -1;
  }
}

__device__ __forceinline__ int lanes_before(uint64_t lanes) {   // of the ballot, below this lane
  return __builtin_amdgcn_mbcnt_hi(lanes >> 32, __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}

// Where a bound leaves too many candidates (ties): the K-th key a byte at a time, its ties by column order, and the rest's
// part of the tail.  The list then holds the row's K.  Reads the row again, a column at a time, for each pass.
// Lanes with the first one's byte count together (rows of one value, 16,384 x 4,168 float16: 456 us, 1,168 with an atomic
// for each lane and one thread searching the bins; 50 us without ties).
template <typename T>
__device__ __forceinline__ PartSum top_by_digits(TopShared &s, uint64_t *list, uint32_t *hist, const T *z, const uint8_t *seen,
                                                 int cols, int k, float scale) {
  const int tid = threadIdx.x, wave = tid >> 6, waves = blockDim.x >> 6;
  auto logit = [&](int c) { return c < cols && (!seen || seen[c]) ? static_cast<float>(z[c]) : -INFINITY; };
  uint32_t prefix = 0, need = k;
#pragma unroll 1
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = tid; i < 256; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    for (int c = tid; c < cols; c += blockDim.x) {
      const uint32_t key = order_key(logit(c));
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) {
        const uint32_t digit = (key >> shift) & 255, first = __builtin_amdgcn_readfirstlane(digit);
        const uint64_t same = __ballot(digit == first);   // of the lanes that are here: most of them where a row ties
        if (digit != first) atomicAdd(&hist[digit], 1u);
        else if (lanes_before(same) == 0) atomicAdd(&hist[first], (uint32_t)__popcll(same));
      }
    }
    __syncthreads();
    if (wave == 0) {   // lane l: bins 255 - 4 l and the three below
      uint32_t n[4], above = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) above += n[j] = hist[255 - 4 * tid - j];
      const uint32_t own = above;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(above, d);
        above += tid >= d ? o : 0;
      }
      // the last lane: fewer than K are seen, and the rest are those that are not, in bin 0
      if (above - own < need && (above >= need || tid == 63)) {
        uint32_t left = need - (above - own);
        int d = 255 - 4 * tid;
#pragma unroll
        for (int j = 0; j < 3; ++j)
          if (d == 255 - 4 * tid - j && n[j] < left) {
            left -= n[j];
            --d;
          }
        s.prefix = prefix | (uint32_t)d << shift;
        s.need = left;
      }
    }
    __syncthreads();
    prefix = s.prefix;
    need = s.need;
  }
  // prefix: the k-th key (0: fewer than k columns are seen); need: how many of its ties are listed, lowest column first
  if (tid == 0) s.count = 0;
  PartSum part{-INFINITY, 0.0f};
  uint32_t before = 0;   // ties in earlier rounds
#pragma unroll 1
  for (int c0 = 0; c0 < cols; c0 += blockDim.x) {
    const float v = logit(c0 + tid);
    const uint32_t key = order_key(v);
    const bool tie = key == prefix && prefix != 0;
    const uint64_t lanes = __ballot(tie);
    __syncthreads();
    if ((tid & 63) == 0) s.wave[wave] = __popcll(lanes);
    __syncthreads();
    uint32_t rank = before + lanes_before(lanes);   // in column order, which is thread order
    for (int w = 0; w < waves; ++w) {
      if (w < wave) rank += s.wave[w];
      before += s.wave[w];
    }
    if (key > prefix || (tie && rank < need)) list[atomicAdd(&s.count, 1u)] = candidate(v, c0 + tid);
    else if (key != 0) join(part, v, scale);
  }
  __syncthreads();
  return part;
}

// One workgroup per row.  A bound from below: with W waves and c = ceil(K / W), the least over the waves of a logit that each
// has c at or above has at least K at or above it.  A wave takes the c-th largest of its lanes' largest (it holds the row
// interleaved, so few more than c logits pass it), or of all its logits (EXACT) where c is most of the lanes; a last wave
// of few lanes does not count (top_shape).  What passes is packed by ballots, without atomics, into the wave's list in LDS,
// and the lists are joined and ranked.  NaN passes every bound.  Lists that would not fit (ties) are left to top_by_digits.
// Bound by the row's bytes where k is small (4,096 x 32,000 bfloat16: k = 8 59 us, k = 64 64 us, 51 us at the rate of a copy),
// by the instructions per candidate where it is not (k = 256 91 us).
template <typename T, typename R, bool EXACT>
__global__ __launch_bounds__(1024, sizeof(R) > 128 && !EXACT ? 8 : 4) void k_top(const T *__restrict__ z, int64_t ldz,
                                              int64_t cols,
                                              const uint8_t *__restrict__ legal, int64_t ldl, int k, int holders,
                                              float inv_t, float *__restrict__ values, int32_t *__restrict__ index,
                                              float *__restrict__ tail) {
  __shared__ TopShared s;
  extern __shared__ uint64_t lists[];
  const int tid = threadIdx.x, waves = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const float scale = inv_t * kLog2e;
  const int64_t r = blockIdx.x;
  const T *zr = z + r * ldz;
  const uint8_t *seen = legal ? legal + r * ldl : nullptr;
  R row(zr, seen, (int)cols);
  const int c = (k + holders - 1) / holders, most = top_list(waves);
  uint64_t *list = lists;
  float2 *found = reinterpret_cast<float2 *>(lists + most);
  float top = -INFINITY;   // NaN where the lane has one
  row.values([&](float v, int) { top = __builtin_elementwise_maximum(top, v); });
  // the c-th largest, rounded down to its key's high 20 bits
  const uint32_t key = order_key(top);
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t next = bound | 1u << bit;
    int passing = 0;
    if constexpr (EXACT) {
      const float x = key_value(next);
      if (next >= 0x00800000u && next <= 0xff800000u)   // a number or +inf
        row.values([&](float v, int) { passing += __popcll(__ballot(!(v < x))); });
    } else {
      passing = __popcll(__ballot(key >= next));
    }
    if (passing >= c) bound = next;
  }
  if ((tid & 63) == 0) s.wave[wave] = bound;
  __syncthreads();
  bound = s.wave[0];
  for (int w = 1; w < holders; ++w) bound = min(bound, s.wave[w]);
  const float floor = bound < 0x00800000u ? -kMostFloat : key_value(bound);   // below it: not seen
  row.forget();
  // The candidates go into the wave's list; the rest adds up for the tail, against the bound, which it stays below.
  PartSum part{-INFINITY, 0.0f};
  const float shift = -floor * scale;
  float sum = 0.0f;
  int mine = 0;
  row.values_wave([&](float v, int col) {
    const bool rest = v < floor;
    const uint64_t lanes = __ballot(!rest);
    if (tail != nullptr) sum += rest ? exp2_of(fmaf(v, scale, shift)) : 0.0f;
    if (lanes) {
      if (!rest) {
        const int slot = mine + lanes_before(lanes);
        if (slot < kWaveCandidates) found[wave * kWaveCandidates + slot] = make_float2(v, __int_as_float(col));
      }
      mine += __popcll(lanes);
    }
  });
  __syncthreads();   // every wave has read the others' bounds
  if ((tid & 63) == 0) s.wave[wave] = mine;
  __syncthreads();
  int count = 0, before = 0;
  bool fits = true;
  for (int w = 0; w < waves; ++w) {
    const int n = s.wave[w];
    fits &= n <= kWaveCandidates;
    before += w < wave ? n : 0;
    count += n;
  }
  if (__builtin_expect(fits && count <= most, 1)) {
    for (int i = tid & 63; i < mine; i += 64) {
      const float2 f = found[wave * kWaveCandidates + i];
      list[before + i] = candidate(f.x, __float_as_int(f.y));
    }
    __syncthreads();
    part = {floor, sum};
    if (top == -INFINITY) {
      part = {-INFINITY, 0.0f};
    } else if (__builtin_expect(tail != nullptr && !(sum > 1e-20f && fabsf(shift) < 1e37f), 0)) {
      // the lane's logits are so far below the bound that their sum would lose digits, or the bound is past what the scale
      // allows: against the lane's own largest
      float low = -INFINITY;
      row.forget();
      row.values([&](float v, int) {
        if (v < floor) low = fmaxf(low, v);
      });
      const float base = base_of(low);
      sum = 0.0f;
      row.forget();
      row.values([&](float v, int) { sum += v < floor ? exp2_of((v - base) * scale) : 0.0f; });
      part = {low, sum};
    }
  } else {
    part = top_by_digits<T>(s, list, reinterpret_cast<uint32_t *>(found), zr, seen, (int)cols, k, scale);
    count = (int)s.count;
  }
  rank_candidates(list, reinterpret_cast<float *>(found), count, k, zr, values + r * k, index + r * k);
  if (tail == nullptr) return;
  __syncthreads();
  for (int i = tid; i < count - k; i += blockDim.x) join(part, reinterpret_cast<float *>(found)[i], scale);
  PartSum all[1] = {part};
  block_part(all, scale, s.share);
  if (tid == 0) tail[r] = all[0].empty() ? -INFINITY : fmaf(base_of(all[0].top), inv_t, log2_of(all[0].sum) * kLn2);
}

// ---- distillation --------------------------------------------------------------------------------------------------

template <typename T>
struct DistillArgs {
  const T *z;
  int64_t ldz, cols;
  const uint8_t *legal;
  int64_t ldl;
  const float *values;
  const int32_t *index;
  const float *tail;
  int k;
  float t, inv_t;
  float *loss;
  T *grad;
  int64_t ldg;
  const float *row_scale;
  float grad_scale;
};

// p log(p/q) - p + q for log p, log q and their exponentials.  Near p = q the logarithms' difference d is small and
// p (d + exp(-d) - 1) keeps its digits: d^2 (1/2! - d/3! + d^2/4! ...), whose terms past d^8 are below 2^-24 of it.
__device__ __forceinline__ float divergence(float logp, float p, float logq, float q) {
  if (p == 0.0f) return q;
  const float d = logp - logq;
  float s = 1.0f / 40320;
  s = fmaf(-d, s, 1.0f / 5040);
  s = fmaf(-d, s, 1.0f / 720);
  s = fmaf(-d, s, 1.0f / 120);
  s = fmaf(-d, s, 1.0f / 24);
  s = fmaf(-d, s, 1.0f / 6);
  s = fmaf(-d, s, 0.5f);
  return fabsf(d) < 0.5f ? p * (d * d * s) : p * d - p + q;
}

// One workgroup per row.  The first waves hold the list and compute the row's scalars; the others wait for the factor of
// their exponentials, so what does not depend on the columns is computed once and not by every wave.  Bound by the row's
// bytes in and out where there are rows to fill the chip (16,384 x 4,168 float16 58 us, 4.7 TB/s of the 5.1 that a copy
// reaches; 2,048 x 50,256 bfloat16 96 us, 4.3 TB/s; x 50,257, whose rows' pieces lie across the lines, 105 us), by a row's
// chain of load, two reductions, list and store where there are few (256 x 4,168 float32 7.2 us).
template <typename T, int NV, bool RES>
__global__ __launch_bounds__(1024, NV == 8 ? 8 : 4) void k_distill(const DistillArgs<T> a) {
  constexpr int N = Piece<T>::N;
  constexpr bool kKeep = RES && NV * N <= 32;  // the exponentials stay in registers for the gradient
  extern __shared__ uint32_t bits[];           // one for each column: listed
  __shared__ __attribute__((aligned(16))) float share[6 * 16], share_loss[2 * (kMostListed / 64)];
  __shared__ float s_factor, s_base, s_loss;
  __shared__ bool s_nothing;
  // the list, an entry in a thread's care throughout: the teacher's logit, then the gradient; the student's; the column
  __shared__ float list_v[kMostListed], list_z[kMostListed];
  __shared__ int32_t list_c[kMostListed];
  const int tid = threadIdx.x, threads = blockDim.x, wave = tid >> 6;
  const int few = (min(a.k, threads) + 63) >> 6;   // waves that hold the list
  const int64_t r = blockIdx.x;
  const T *zr = a.z + r * a.ldz;
  const uint8_t *seen = a.legal ? a.legal + r * a.ldl : nullptr;
  Row<T, NV, RES> row(zr, seen, (int)a.cols);
  for (int w = tid; w < ((int)a.cols + 31) / 32; w += threads) bits[w] = 0;
  __syncthreads();
  bool bad = false;
  for (int i = tid; i < a.k; i += threads) {
    const int32_t c = a.index[r * a.k + i];
    const float v = a.values[r * a.k + i];
    int32_t col = -1;
    float zc = 0.0f;
    if (c >= a.cols) {
      bad = true;
    } else if (c >= 0) {
      zc = static_cast<float>(zr[c]);   // asked for with the mask's byte, not after it
      if (!seen || seen[c]) {
        const uint32_t bit = 1u << (c & 31);
        if (atomicOr(&bits[c >> 5], bit) & bit) bad = true;
        else col = c;
      }
    }
    list_c[i] = col;
    list_v[i] = v;
    list_z[i] = zc;
  }
  __syncthreads();
  // the rest, the teacher's list and the student's listed logits
  const float scale2 = a.inv_t * kLog2e;
  PartSum part[3] = {{-INFINITY, 0.0f}, {-INFINITY, 0.0f}, {-INFINITY, 0.0f}};
  auto erase_listed = [&](int i, Raw16 &p) {
    const uint32_t b = (bits[i * N >> 5] >> (i * N & 31)) & ((1u << N) - 1);
    if (b)
#pragma unroll
      for (int e = 0; e < N; ++e)
        if ((b >> e) & 1) erase<T>(p, e);
  };
  float kept[kKeep ? NV * N : 1];
  float base = 0.0f;   // of this thread's exponentials
  // The maximum comes off before the scale: fma(z, scale, -base * scale) keeps the rounding of its constant, which passes any
  // exponent for logits of 1e10 (fills of hidden moves), and costs as much time.
  if constexpr (RES) {
    float top = -INFINITY, sum = 0.0f;
    row.each([&](int, int i, Raw16 &p) {
      erase_listed(i, p);
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, element<T>(p, e));
    });
    base = base_of(top);
    if (!kKeep) row.forget();
    row.each([&](int j, int, const Raw16 &p) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float x = exp2_of((element<T>(p, e) - base) * scale2);
        if (kKeep && j >= 0) kept[kKeep && j >= 0 ? j * N + e : 0] = x;
        sum += x;
      }
    });
    part[0] = {top, sum};
  } else {
    row.each([&](int, int i, Raw16 &p) {
      erase_listed(i, p);
      float top = part[0].top;
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, element<T>(p, e));
      const float base = base_of(top);
      float sum = part[0].sum * exp2_of((part[0].top - base) * scale2);
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp2_of((element<T>(p, e) - base) * scale2);
      part[0] = {top, sum};
    });
  }
  const float own_top = part[0].top;
  for (int i = tid; i < a.k; i += threads)
    if (list_c[i] >= 0) {
      join(part[1], list_v[i], scale2);
      join(part[2], list_z[i], scale2);
    }
  block_part(part, scale2, share, few);
  const float nan = __builtin_nanf("");
  if (wave < few) {
    // the student's normaliser, against its largest logit: log q = (z - mz) / T - ln_z
    const bool has_rest = !part[0].empty();
    const float mz = base_of(fmaxf(part[0].top, part[2].top)), rest_top = base_of(part[0].top);
    const float ln_z = ln_of(part[0].sum * exp2_of((part[0].top - mz) * scale2) +
                             part[2].sum * exp2_of((part[2].top - mz) * scale2));
    const float logqt = has_rest ? (rest_top - mz) * a.inv_t + ln_of(part[0].sum) - ln_z : -INFINITY;
    // the teacher's, its tail a scaled number already: log p = (v - mv) / T + (x - ma) - ln_a
    const float at = a.tail && has_rest ? a.tail[r] : -INFINITY;   // no rest to put it on: the list alone
    const float mv = base_of(part[1].top);
    const float x = part[1].empty() ? -kMostFloat : fminf(fmaxf(mv * a.inv_t, -kMostFloat), kMostFloat);
    const float ma = fmaxf(x, at);
    const float ln_a = ln_of(part[1].sum * exp_of(x - ma) + exp_of(at - ma)), logpt = at - ma - ln_a;
    const bool some = !(part[1].empty() && at == -INFINITY) && !(part[0].empty() && part[2].empty());
    const float pt = some ? exp_of(logpt) : 0.0f, qt = some ? exp_of(logqt) : 0.0f;
    const float scale = a.grad ? a.t * a.grad_scale * (a.row_scale ? a.row_scale[r] : 1.0f) : 0.0f;
    float l = 0.0f;
    for (int i = tid; i < a.k; i += threads)
      if (list_c[i] >= 0 && some) {
        const float logp = (list_v[i] - mv) * a.inv_t + (x - ma) - ln_a, logq = (list_z[i] - mz) * a.inv_t - ln_z;
        const float p = exp_of(logp), q = exp_of(logq);
        l += divergence(logp, p, logq, q);
        list_v[i] = scale * (q - p);
      }
    l = wave_sum(l);
    bad = __any(bad);
    if (few > 1) {
      if ((tid & 63) == 0) {
        share_loss[2 * wave] = l;
        share_loss[2 * wave + 1] = bad ? 1.0f : 0.0f;
      }
    }
    if (tid == 0) {
      s_base = rest_top;
      s_nothing = !some;
      s_factor = bad ? nan : has_rest ? scale * (qt - pt) / part[0].sum : 0.0f;
      s_loss = some ? divergence(logpt, pt, logqt, qt) : 0.0f;   // the rest's share
      if (few == 1 && a.loss) a.loss[r] = bad ? nan : a.t * (a.t * (l + s_loss));
    }
  }
  __syncthreads();
  float factor = s_factor;
  if (few > 1) {
    float l = share_loss[0], n = share_loss[1];
    for (int w = 1; w < few; ++w) {
      l += share_loss[2 * w];
      n += share_loss[2 * w + 1];
    }
    bad = n != 0.0f;
    if (tid == 0 && a.loss) a.loss[r] = bad ? nan : a.t * (a.t * (l + s_loss));
    if (bad) factor = nan;
  }
  if (!a.grad) return;
  T *gr = a.grad + r * a.ldg;
  // A row past the registers reads its logits again here: its gradients go around the caches, which so still hold them
  // (2,048 x 70,000 bfloat16 140 us against 155).  Rows in registers gain nothing (16,384 x 4,168 float32 106 against 102).
  auto store = [&](int j, int i, const Piece<T> &g) {
    if (j < 0) store_last(gr, i, row.left, g);
    else store_whole<T, !RES>(gr, i, g);
  };
  if (s_nothing && factor == factor) {
    row.each([&](int j, int i, const Raw16 &) {
      Piece<T> g;
#pragma unroll
      for (int e = 0; e < N; ++e) g.v[e] = 0.0f;
      store(j, i, g);
    });
    return;
  }
  if constexpr (RES) {
    if (!kKeep) row.forget();
    // A thread that holds none of the rest has exponentials of 0, and no base of its own to compare with the row's: its
    // gradients are 0, but the row's NaN where the factor is one.
    const float f = factor * (own_top == -INFINITY ? 0.0f : exp2_of((base - s_base) * scale2));
    row.each([&](int j, int i, const Raw16 &p) {
      Piece<T> g;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if (kKeep && j >= 0) g.v[e] = kept[kKeep && j >= 0 ? j * N + e : 0] * f;
        else g.v[e] = exp2_of((element<T>(p, e) - base) * scale2) * f;
      }
      store(j, i, g);
    });
  } else {
    const float base = s_base;
    row.each([&](int j, int i, Raw16 &p) {
      erase_listed(i, p);
      Piece<T> g;
#pragma unroll
      for (int e = 0; e < N; ++e) g.v[e] = exp2_of((element<T>(p, e) - base) * scale2) * factor;
      store(j, i, g);
    });
  }
  __syncthreads();   // the list's own gradients overwrite what the pass left in their columns
  for (int i = tid; i < a.k; i += threads)
    if (list_c[i] >= 0) gr[list_c[i]] = static_cast<T>(bad ? nan : list_v[i]);
}

template <typename F>
void by_type(int32_t type, F &&f) {
  switch (type) {
    case FLY_F32: f(float{}); break;
    case FLY_F16: f(_Float16{}); break;
    case FLY_BF16: f(bhalf{}); break;
    default: FLY_REQUIRE(false, "the logits must be float32, float16 or bfloat16");
  }
}

template <typename F>
void by_shape(const RowShape &s, F &&f) {
  using std::integral_constant;
  switch (s.kept) {
    case 1: f(integral_constant<int, 1>{}, std::true_type{}, s.threads); break;
    case 2: f(integral_constant<int, 2>{}, std::true_type{}, s.threads); break;
    case 4: f(integral_constant<int, 4>{}, std::true_type{}, s.threads); break;
    case 8: f(integral_constant<int, 8>{}, std::true_type{}, s.threads); break;
    default: f(integral_constant<int, 1>{}, std::false_type{}, s.threads);
  }
}

void check_logits(const void *z, int64_t ldz, int64_t rows, int64_t cols, const uint8_t *legal, int64_t ldl, int32_t k,
                  float temperature) {
  FLY_REQUIRE(rows >= 0 && rows < INT32_MAX && cols >= 1 && cols <= kMostColumns, "rows or columns out of range");
  FLY_REQUIRE(k >= 1 && k <= kMostListed, "k must lie in 1..256");
  FLY_REQUIRE(temperature > 0.0f && std::isfinite(temperature) && std::isfinite(1.0f / temperature * kLog2e),
              "the temperature must be positive and finite, and log2(e) / temperature too");
  FLY_REQUIRE(!rows || (z && ldz >= cols), "logits are null or their rows overlap");
  FLY_REQUIRE(!legal || ldl >= cols, "the mask's rows overlap");
}

}  // namespace
}  // namespace fly

using namespace fly;

extern "C" int fly_top_logits(const void *z, int32_t type, int64_t ldz, int64_t rows, int64_t cols,
                              const uint8_t *legal, int64_t ldl, int32_t k, float temperature, float *values,
                              int32_t *index, float *tail, void *stream) {
  return guard([&] {
    check_logits(z, ldz, rows, cols, legal, ldl, k, temperature);
    FLY_REQUIRE(!rows || (values && index), "values and index are required");
    by_type(type, [&](auto t) {
      using T = decltype(t);
      if (!rows) return;
      const TopShape shape = top_shape(rows, cols, sizeof(T), k);
      auto run = [&](auto kernel, int threads) {
        const int waves = threads / 64;
        in_slices(rows, threads, [&](int64_t r, int64_t n) {
          hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads), 8 * (size_t)(top_list(waves) + waves * kWaveCandidates),
                             as_stream(stream), static_cast<const T *>(z) + r * ldz, ldz, cols, legal ? legal + r * ldl : nullptr,
                             ldl, k, shape.holders, 1.0f / temperature, values + r * k, index + r * k,
                             tail ? tail + r : nullptr);
          check_launch("top logits");
        });
      };
      if (shape.spread == 4) run(k_top<T, Spread<T, 4>, true>, 256);
      else if (shape.spread == 16) run(k_top<T, Spread<T, 16>, true>, 256);
      else
        by_shape(shape.row, [&](auto nv, auto res, int threads) {
          run(k_top<T, Row<T, decltype(nv)::value, decltype(res)::value>, false>, threads);
        });
    });
  });
}

extern "C" int fly_distill(const void *z, int32_t type, int64_t ldz, int64_t rows, int64_t cols, const uint8_t *legal,
                           int64_t ldl, const float *values, const int32_t *index, const float *tail, int32_t k,
                           float temperature, float *loss, void *grad, int64_t ldg, const float *row_scale,
                           float grad_scale, void *stream) {
  return guard([&] {
    check_logits(z, ldz, rows, cols, legal, ldl, k, temperature);
    FLY_REQUIRE(!rows || (values && index), "the teacher's values and index are required");
    FLY_REQUIRE(!rows || loss || grad, "neither a loss nor a gradient is asked for");
    FLY_REQUIRE(!grad || ldg >= cols, "the gradient's rows overlap");
    by_type(type, [&](auto t) {
      using T = decltype(t);
      if (!rows) return;
      const size_t lds = (size_t)round_up(cols, 32) / 8;
      by_shape(row_shape(rows, cols, sizeof(T), 64, 4), [&](auto nv, auto res, int threads) {
        constexpr auto kernel = &k_distill<T, decltype(nv)::value, decltype(res)::value>;
        if (lds > 60 * 1024) allow_lds(kernel, kMostColumns / 8);
        in_slices(rows, threads, [&](int64_t r, int64_t n) {
          const DistillArgs<T> a{static_cast<const T *>(z) + r * ldz, ldz, cols, legal ? legal + r * ldl : nullptr, ldl,
                                 values + r * k, index + r * k, tail ? tail + r : nullptr, k, temperature, 1.0f / temperature,
                                 loss ? loss + r : nullptr, grad ? static_cast<T *>(grad) + r * ldg : nullptr, ldg,
                                 row_scale ? row_scale + r : nullptr, grad_scale};
          hipLaunchKernelGGL(kernel, dim3((unsigned)n), dim3(threads), lds, as_stream(stream), a);
          check_launch("distillation");
        });
      });
    });
  });
}
