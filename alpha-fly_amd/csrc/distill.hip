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
#include "rows.hpp"

namespace fly {
namespace {

constexpr int kMostListed = 256;             // no chess position has over 218 legal moves
constexpr int64_t kMostColumns = 1 << 20;    // a bit for each column in LDS: 128 KB

// A row's 16-byte pieces, piece tid + j * blockDim for j < NV in a thread's registers (RES), or read again at each pass.
template <typename T, int NV, bool RES>
struct Row {
  static constexpr int N = Piece<T>::N;
  const T *z;
  const uint8_t *seen;
  int64_t cols, pieces;
  Raw16 kept[RES ? NV : 1];

  __device__ __forceinline__ Row(const T *row, const uint8_t *mask, int64_t n) : z(row), seen(mask), cols(n), pieces((n + N - 1) / N) {
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int64_t i = threadIdx.x + j * (int64_t)blockDim.x;
        if (i < pieces) kept[j] = load_raw(z, i, cols);
      }
      if (seen)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int64_t i = threadIdx.x + j * (int64_t)blockDim.x;
          if (i < pieces) mask_raw<T>(kept[j], seen, i, cols);
        }
    }
  }
  // f(piece number, piece) for this thread's pieces, columns that do not exist at -inf
  template <typename F>
  __device__ __forceinline__ void each(F &&f) {
    if constexpr (RES) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int64_t i = threadIdx.x + j * (int64_t)blockDim.x;
        if (i < pieces) f(i, kept[j]);
      }
    } else {
      for (int64_t i = threadIdx.x; i < pieces; i += blockDim.x) {
        Raw16 p = load_raw(z, i, cols);
        if (seen) mask_raw<T>(p, seen, i, cols);
        f(i, p);
      }
    }
  }
};

// How many pieces a thread keeps and how many threads a row gets: {1, 2, 4, 8} pieces, the fewest that 512 threads cover a
// row with, or 8 on up to 1,024 threads; longer rows are read at every pass (kept = 0) by 1,024 threads.
struct RowShape {
  int kept, threads;
};
RowShape row_shape(int64_t cols, size_t elem, int least) {
  const int64_t pieces = (cols * (int64_t)elem + 15) / 16;
  for (int kept : {1, 2, 4, 8}) {
    const int64_t threads = std::max<int64_t>(round_up((pieces + kept - 1) / kept, 64), least);
    if (threads <= (kept == 8 ? 1024 : 512)) return {kept, (int)threads};
  }
  return {0, 1024};
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f, kMostFloat = 3.4028234663852886e38f;

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

struct TopShared {
  union {
    uint64_t list[kMostCandidates];
    uint32_t hist[256];
  };
  float share[2 * 16];
  uint32_t wave[16];
  uint32_t count, prefix, need;
  int32_t cut;
};

__device__ __forceinline__ uint64_t candidate(float v, int64_t col) {   // larger is better: the key, then the lower column
  return (uint64_t)order_key(v) << 32 | (uint32_t)~(uint32_t)col;
}

// The K largest of `count` candidates in their places, the others to rest(value); any number of threads.
template <typename T, typename F>
__device__ __forceinline__ void rank_candidates(const TopShared &s, int count, int k, const T *z, float *values,
                                                int32_t *index, F &&rest) {
  for (int i = threadIdx.x; i < count; i += blockDim.x) {
    const uint64_t mine = s.list[i];
    int rank = 0;
    for (int j = 0; j < count; ++j) rank += s.list[j] > mine;
    const int32_t col = (int32_t)~(uint32_t)mine;
    const float v = static_cast<float>(z[col]);
    if (rank < k) {
      values[rank] = v;
      index[rank] = col;
    } else {
      rest(v);
    }
  }
  for (int i = count + threadIdx.x; i < k; i += blockDim.x) {
    values[i] = -INFINITY;
    index[i] = -1;
  }
}

// Where a bound leaves too many candidates (ties): the K-th key a byte at a time, its ties by column order, and the rest's
// part of the tail.  The list then holds the row's K.  Reads the row again for each pass.
template <typename T>
__device__ __forceinline__ PartSum top_by_digits(TopShared &s, const T *z, const uint8_t *seen, int64_t cols, int k, float scale) {
  Row<T, 1, false> row(z, seen, cols);
  constexpr int N = Piece<T>::N;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  uint32_t prefix = 0, need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = tid; i < 256; i += blockDim.x) s.hist[i] = 0;
    __syncthreads();
    row.each([&](int64_t, const Raw16 &p) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t key = order_key(element<T>(p, e));
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&s.hist[(key >> shift) & 255], 1u);
      }
    });
    __syncthreads();
    if (tid == 0) {
      uint32_t left = need;
      int d = 255;
      for (; d > 0 && s.hist[d] < left; --d) left -= s.hist[d];
      s.prefix = prefix | (uint32_t)d << shift;
      s.need = left;
    }
    __syncthreads();
    prefix = s.prefix;
    need = s.need;
  }
  // prefix: the k-th key (0: fewer than k columns are seen); need: how many of its ties are listed, lowest column first
  if (tid == 0) {
    s.count = 0;
    s.cut = -1;
  }
  __syncthreads();
  uint32_t before = 0;   // ties in earlier rounds
  for (int64_t i0 = 0; i0 < row.pieces; i0 += blockDim.x) {
    uint32_t key[N] = {}, eq = 0;
    if (i0 + tid < row.pieces) {
      Raw16 p = load_raw(row.z, i0 + tid, row.cols);
      if (row.seen) mask_raw<T>(p, row.seen, i0 + tid, row.cols);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        key[e] = order_key(element<T>(p, e));
        eq += key[e] == prefix && prefix != 0;
      }
    }
    uint32_t at = eq;   // inclusive prefix sum of the ties in thread order, which is column order
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t o = __shfl_up(at, d);
      if (lane >= d) at += o;
    }
    if (lane == 63) s.wave[wave] = at;
    __syncthreads();
    uint32_t rank = before + at - eq;
    for (int w = 0; w < waves; ++w) {
      if (w < wave) rank += s.wave[w];
      before += s.wave[w];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      bool take = key[e] > prefix;
      const int32_t col = (int32_t)((i0 + tid) * N + e);
      if (key[e] == prefix && prefix != 0) {
        take = rank < need;
        if (rank == need - 1) s.cut = col;
        ++rank;
      }
      if (take) s.list[atomicAdd(&s.count, 1u)] = (uint64_t)key[e] << 32 | (uint32_t)~(uint32_t)col;
    }
    __syncthreads();
  }
  const int32_t cut = s.cut;
  PartSum part{-INFINITY, 0.0f};
  row.each([&](int64_t i, const Raw16 &p) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float v = element<T>(p, e);
      const uint32_t key = order_key(v);
      if (key != 0 && (key < prefix || (key == prefix && (int32_t)(i * N + e) > cut))) join(part, v, scale);
    }
  });
  return part;
}

// One workgroup per row.  A bound from below: with W waves and c = ceil(K / W), each wave has c lanes whose largest logit
// is at least the wave's c-th largest of those, so the least of these over the waves has at least K logits at or above
// it.  Few more than K are (a wave's lanes hold the row interleaved): they go to a list in LDS, where each counts those
// before it.  NaN passes every bound.  A list that would not fit is left to top_by_digits.
template <typename T, int NV, bool RES>
__global__ __launch_bounds__(1024) void k_top(const T *__restrict__ z, int64_t ldz, int64_t cols,
                                              const uint8_t *__restrict__ legal, int64_t ldl, int k, float inv_t,
                                              float *__restrict__ values, int32_t *__restrict__ index,
                                              float *__restrict__ tail) {
  constexpr int N = Piece<T>::N;
  __shared__ TopShared s;
  const int tid = threadIdx.x, waves = blockDim.x >> 6;
  const float scale = inv_t * kLog2e;
  const int64_t r = blockIdx.x;
  const T *zr = z + r * ldz;
  Row<T, NV, RES> row(zr, legal ? legal + r * ldl : nullptr, cols);
  if (tid == 0) s.count = 0;
  float top = -INFINITY;
  row.each([&](int64_t, const Raw16 &p) {
#pragma unroll
    for (int e = 0; e < N; ++e) top = fmaxf(top, element<T>(p, e));
  });
  // the c-th largest of the wave's lanes, rounded down to its high 20 bits
  const int c = (k + waves - 1) / waves;
  const uint32_t key = order_key(top);
  uint32_t bound = 0;
#pragma unroll
  for (int bit = 31; bit >= 12; --bit) {
    const uint32_t next = bound | 1u << bit;
    if (__popcll(__ballot(key >= next)) >= c) bound = next;
  }
  if ((tid & 63) == 0) s.wave[tid >> 6] = bound;
  __syncthreads();
  for (int w = 0; w < waves; ++w) bound = min(bound, s.wave[w]);
  const float floor = bound < 0x00800000u ? -kMostFloat : key_value(bound);   // below it: not seen
  PartSum part{-INFINITY, 0.0f};
  float low = -INFINITY;   // the largest logit below the bound
  row.each([&](int64_t i, const Raw16 &p) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float v = element<T>(p, e);
      if (v < floor) {
        low = fmaxf(low, v);
      } else {
        const uint32_t slot = atomicAdd(&s.count, 1u);
        if (slot < kMostCandidates) s.list[slot] = candidate(v, i * N + e);
      }
    }
  });
  __syncthreads();
  int count = (int)s.count;
  if (count > kMostCandidates) {
    part = top_by_digits<T>(s, zr, row.seen, cols, k, scale);
    count = (int)s.count;
  } else if (tail != nullptr) {
    const float base = base_of(low);
    float sum = 0.0f;
    row.each([&](int64_t, const Raw16 &p) {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float v = element<T>(p, e);
        sum += v < floor ? exp2f((v - base) * scale) : 0.0f;
      }
    });
    part = {low, sum};
  }
  rank_candidates(s, count, k, zr, values + r * k, index + r * k, [&](float v) { join(part, v, scale); });
  if (tail == nullptr) return;
  PartSum all[1] = {part};
  block_part(all, scale, s.share);
  if (tid == 0) tail[r] = all[0].empty() ? -INFINITY : fmaf(base_of(all[0].top), inv_t, log2f(all[0].sum) * kLn2);
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

// p log(p/q) - p + q for log p, log q and their exponentials; near p = q the logarithms' difference d is small and
// p (d + exp(-d) - 1) keeps its digits.
__device__ __forceinline__ float divergence(float logp, float p, float logq, float q) {
  if (p == 0.0f) return q;
  const float d = logp - logq;
  return fabsf(d) < 0.5f ? p * (d + expm1f(-d)) : p * d - p + q;
}

// One workgroup per row.
template <typename T, int NV, bool RES>
__global__ __launch_bounds__(1024) void k_distill(const DistillArgs<T> a) {
  constexpr int N = Piece<T>::N;
  constexpr int kEntries = kMostListed / 64;   // of the list, at most, for a thread
  extern __shared__ uint32_t bits[];           // one for each column: listed
  __shared__ float share[6 * 16], share_loss[16];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int64_t r = blockIdx.x;
  const T *zr = a.z + r * a.ldz;
  const uint8_t *seen = a.legal ? a.legal + r * a.ldl : nullptr;
  Row<T, NV, RES> row(zr, seen, a.cols);
  for (int64_t w = tid; w < (a.cols + 31) / 32; w += threads) bits[w] = 0;
  __syncthreads();
  float av[kEntries], zs[kEntries];
  int32_t col[kEntries];
  bool bad = false;
#pragma unroll
  for (int j = 0; j < kEntries; ++j) {
    av[j] = zs[j] = -INFINITY;
    col[j] = -1;
    const int i = tid + j * threads;
    if (i < a.k) {
      const int32_t c = a.index[r * a.k + i];
      if (c >= a.cols) {
        bad = true;
      } else if (c >= 0 && (!seen || seen[c])) {
        const uint32_t bit = 1u << (c & 31);
        if (atomicOr(&bits[c >> 5], bit) & bit) {
          bad = true;
        } else {
          col[j] = c;
          av[j] = a.values[r * a.k + i];
          zs[j] = static_cast<float>(zr[c]);
        }
      }
    }
  }
  bad = __syncthreads_or(bad);
  // the rest, the teacher's list and the student's listed logits
  const float scale2 = a.inv_t * kLog2e;
  PartSum part[3] = {{-INFINITY, 0.0f}, {-INFINITY, 0.0f}, {-INFINITY, 0.0f}};
  auto erase_listed = [&](int64_t i, Raw16 &p) {
    const uint32_t b = (bits[i * N >> 5] >> (i * N & 31)) & ((1u << N) - 1);
    if (b)
#pragma unroll
      for (int e = 0; e < N; ++e)
        if ((b >> e) & 1) erase<T>(p, e);
  };
  if constexpr (RES) {
    float top = -INFINITY, sum = 0.0f;
    row.each([&](int64_t i, Raw16 &p) {
      erase_listed(i, p);
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, element<T>(p, e));
    });
    const float base = base_of(top);
    row.each([&](int64_t, const Raw16 &p) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp2f((element<T>(p, e) - base) * scale2);
    });
    part[0] = {top, sum};
  } else {
    row.each([&](int64_t i, Raw16 &p) {
      erase_listed(i, p);
      float top = part[0].top;
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, element<T>(p, e));
      const float base = base_of(top);
      float sum = part[0].sum * exp2f((part[0].top - base) * scale2);
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp2f((element<T>(p, e) - base) * scale2);
      part[0] = {top, sum};
    });
  }
#pragma unroll
  for (int j = 0; j < kEntries; ++j)
    if (col[j] >= 0) {
      join(part[1], av[j], scale2);
      join(part[2], zs[j], scale2);
    }
  block_part(part, scale2, share);
  // the student's normaliser, against its largest logit: log q = (z - mz) / T - ln_z
  const bool has_rest = !part[0].empty();
  const float mz = base_of(fmaxf(part[0].top, part[2].top)), rest_top = base_of(part[0].top);
  const float ln_z = logf(part[0].sum * exp2f((part[0].top - mz) * scale2) + part[2].sum * exp2f((part[2].top - mz) * scale2));
  const float logqt = has_rest ? (rest_top - mz) * a.inv_t + logf(part[0].sum) - ln_z : -INFINITY;
  // the teacher's, its tail a scaled number already: log p = (v - mv) / T + (x - ma) - ln_a
  const float at = a.tail && has_rest ? a.tail[r] : -INFINITY;   // no rest to put it on: the list alone
  const float mv = base_of(part[1].top), x = part[1].empty() ? -kMostFloat : fmaxf(mv * a.inv_t, -kMostFloat);
  const float ma = fmaxf(x, at);
  const float ln_a = logf(part[1].sum * expf(x - ma) + expf(at - ma)), logpt = at - ma - ln_a;
  const bool some = !(part[1].empty() && at == -INFINITY) && !(part[0].empty() && part[2].empty());
  const float nan = __builtin_nanf("");
  const float pt = some ? expf(logpt) : 0.0f, qt = some ? expf(logqt) : 0.0f;
  float p[kEntries], q[kEntries], l = 0.0f;
#pragma unroll
  for (int j = 0; j < kEntries; ++j) {
    p[j] = q[j] = 0.0f;
    if (col[j] >= 0 && some) {
      const float logp = (av[j] - mv) * a.inv_t + (x - ma) - ln_a, logq = (zs[j] - mz) * a.inv_t - ln_z;
      p[j] = expf(logp);
      q[j] = expf(logq);
      l += divergence(logp, p[j], logq, q[j]);
    }
  }
  if (a.loss) {
    l = block_sum(l, share_loss);
    if (tid == 0)
      a.loss[r] = bad ? nan : some ? a.t * a.t * (l + divergence(logpt, pt, logqt, qt)) : 0.0f;
  }
  if (!a.grad) return;
  const float scale = a.t * a.grad_scale * (a.row_scale ? a.row_scale[r] : 1.0f);
  const float coef = bad ? nan : some && has_rest ? scale * (qt - pt) / part[0].sum : 0.0f;
  const bool nothing = !some && !bad;
  T *gr = a.grad + r * a.ldg;
  row.each([&](int64_t i, Raw16 &v) {
    if constexpr (!RES) erase_listed(i, v);
    Piece<T> g;
#pragma unroll
    for (int e = 0; e < N; ++e) g.v[e] = nothing ? 0.0f : exp2f((element<T>(v, e) - rest_top) * scale2) * coef;
    store_piece(gr, i, a.cols, g);
  });
  __syncthreads();   // the list's own gradients overwrite what the pass left in their columns
#pragma unroll
  for (int j = 0; j < kEntries; ++j)
    if (col[j] >= 0 && some && !bad) gr[col[j]] = static_cast<T>(scale * (q[j] - p[j]));
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
  FLY_REQUIRE(temperature > 0.0f && std::isfinite(temperature) && std::isfinite(1.0f / temperature),
              "the temperature must be positive and finite");
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
      by_shape(row_shape(cols, sizeof(T), (int)round_up(k, 64)), [&](auto nv, auto res, int threads) {
        hipLaunchKernelGGL((k_top<T, decltype(nv)::value, decltype(res)::value>), dim3((unsigned)rows), dim3(threads), 0,
                           as_stream(stream), static_cast<const T *>(z), ldz, cols, legal, ldl, k, 1.0f / temperature,
                           values, index, tail);
      });
      check_launch("top logits");
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
      const DistillArgs<T> a{static_cast<const T *>(z), ldz, cols, legal, ldl, values, index, tail, k, temperature,
                             1.0f / temperature, loss, static_cast<T *>(grad), ldg, row_scale, grad_scale};
      const size_t lds = (size_t)round_up(cols, 32) / 8;
      by_shape(row_shape(cols, sizeof(T), 64), [&](auto nv, auto res, int threads) {
        constexpr auto kernel = &k_distill<T, decltype(nv)::value, decltype(res)::value>;
        if (lds > 60 * 1024)
          FLY_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)lds));
        hipLaunchKernelGGL(kernel, dim3((unsigned)rows), dim3(threads), lds, as_stream(stream), a);
      });
      check_launch("distillation");
    });
  });
}
