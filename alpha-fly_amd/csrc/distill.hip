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

// ---- top logits ----------------------------------------------------------------------------------------------------

// A float's place in the order of numbers as an unsigned: NaN above all, the zeros alike, 0 for a column not seen.
__device__ __forceinline__ uint32_t order_key(float v) {
  if (v != v) return 0xffffffffu;
  if (v == -INFINITY) return 0;
  const uint32_t b = __float_as_uint(v + 0.0f);   // -0 + 0 = +0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

template <typename T>
__global__ __launch_bounds__(256) void k_top(const T *__restrict__ z, int64_t ldz, int64_t cols,
                                             const uint8_t *__restrict__ legal, int64_t ldl, int k, float inv_t,
                                             float *__restrict__ values, int32_t *__restrict__ index,
                                             float *__restrict__ tail) {
  constexpr int N = Piece<T>::N;
  __shared__ uint32_t hist[256];
  __shared__ uint32_t s_prefix, s_need, s_count;
  __shared__ float share[16];
  __shared__ uint32_t list_key[kMostListed];
  __shared__ int32_t list_col[kMostListed];
  __shared__ int32_t s_cut;
  __shared__ int wave_eq[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x;
  const T *zr = z + row * ldz;
  const uint8_t *seen = legal ? legal + row * ldl : nullptr;
  const int64_t pieces = (cols + N - 1) / N;
  auto piece = [&](int64_t i) {
    Piece<T> p = load_piece(zr, i, cols, -INFINITY);
    if (seen) mask_piece(p, seen, i, cols);
    return p;
  };
  // the k-th largest key, a byte at a time
  uint32_t prefix = 0, need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    hist[tid] = 0;
    __syncthreads();
    for (int64_t i = tid; i < pieces; i += 256) {
      const Piece<T> p = piece(i);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t key = order_key(p.v[e]);
        if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1u);
      }
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = need;
      int d = 255;
      for (; d > 0 && hist[d] < left; --d) left -= hist[d];
      s_prefix = prefix | (uint32_t)d << shift;
      s_need = left;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
  }
  // prefix: the k-th key (0: fewer than k columns are seen); need: how many of its ties are listed, lowest column first
  if (tid == 0) {
    s_count = 0;
    s_cut = -1;
  }
  if (tid < k) list_key[tid] = 0;
  __syncthreads();
  int before = 0;   // ties in earlier rounds
  for (int64_t i0 = 0; i0 < pieces; i0 += 256) {
    Piece<T> p;
    uint32_t key[N];
    int eq = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) key[e] = 0;
    if (i0 + tid < pieces) {
      p = piece(i0 + tid);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        key[e] = order_key(p.v[e]);
        eq += key[e] == prefix && prefix != 0;
      }
    }
    int at = eq;   // inclusive prefix sum of the ties in thread order, which is column order
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(at, d);
      if (lane >= d) at += o;
    }
    if (lane == 63) wave_eq[wave] = at;
    __syncthreads();
    int base = before;
    for (int w = 0; w < 4; ++w) {
      if (w < wave) base += wave_eq[w];
      before += wave_eq[w];
    }
    int rank = base + at - eq;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      bool take = key[e] > prefix;
      if (key[e] == prefix && prefix != 0) {
        take = rank < (int)need;
        if (rank == (int)need - 1) s_cut = (int32_t)((i0 + tid) * N + e);
        ++rank;
      }
      if (take) {
        const uint32_t slot = atomicAdd(&s_count, 1u);
        list_key[slot] = key[e];
        list_col[slot] = (int32_t)((i0 + tid) * N + e);
      }
    }
    __syncthreads();
  }
  const int count = (int)s_count;
  const int32_t cut = s_cut;
  if (tid < k) {
    int64_t at = tid;
    float v = -INFINITY;
    int32_t c = -1;
    if (tid < count) {
      const uint32_t key = list_key[tid];
      c = list_col[tid];
      at = 0;
      for (int j = 0; j < count; ++j) at += list_key[j] > key || (list_key[j] == key && list_col[j] < c);
      v = static_cast<float>(zr[c]);
    }
    values[row * k + at] = v;
    index[row * k + at] = c;
  }
  if (tail == nullptr) return;
  float m[1] = {-INFINITY};
  auto rest = [&](auto &&f) {
    for (int64_t i = tid; i < pieces; i += 256) {
      const Piece<T> p = piece(i);
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const uint32_t key = order_key(p.v[e]);
        const bool out = key < prefix || (key == prefix && (int32_t)(i * N + e) > cut);
        if (out && key) f(p.v[e] * inv_t);
      }
    }
  };
  rest([&](float v) { m[0] = v > m[0] || v != v ? v : m[0]; });
  block_max(m, share);
  float s[1] = {0.0f};
  if (m[0] != -INFINITY) rest([&](float v) { s[0] += expf(v - m[0]); });
  block_sum(s, share);
  if (tid == 0) tail[row] = m[0] == -INFINITY ? -INFINITY : m[0] + logf(s[0]);
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

template <typename T>
__global__ __launch_bounds__(256) void k_distill(const DistillArgs<T> a) {
  constexpr int N = Piece<T>::N;
  extern __shared__ uint32_t bits[];   // one for each column: listed
  __shared__ float share[3 * 4];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const T *zr = a.z + row * a.ldz;
  const uint8_t *seen = a.legal ? a.legal + row * a.ldl : nullptr;
  const int64_t pieces = (a.cols + N - 1) / N;
  for (int64_t w = tid; w < (a.cols + 31) / 32; w += 256) bits[w] = 0;
  __syncthreads();
  // this thread's entry of the list
  float av = -INFINITY, zs = -INFINITY;
  int32_t col = -1;
  bool bad = false;
  if (tid < a.k) {
    const int32_t c = a.index[row * a.k + tid];
    if (c >= a.cols) {
      bad = true;
    } else if (c >= 0 && (!seen || seen[c])) {
      const uint32_t bit = 1u << (c & 31);
      if (atomicOr(&bits[c >> 5], bit) & bit) {
        bad = true;
      } else {
        col = c;
        av = a.values[row * a.k + tid] * a.inv_t;
        zs = static_cast<float>(zr[c]) * a.inv_t;
      }
    }
  }
  bad = __syncthreads_or(bad);
  auto rest_piece = [&](int64_t i) {
    Piece<T> p = load_piece(zr, i, a.cols, -INFINITY);
    if (seen) mask_piece(p, seen, i, a.cols);
    const uint32_t b = bits[i * N >> 5] >> (i * N & 31);
#pragma unroll
    for (int e = 0; e < N; ++e) p.v[e] = (b >> e) & 1 ? -INFINITY : p.v[e] * a.inv_t;
    return p;
  };
  float m[3] = {-INFINITY, av, zs};   // the rest, the teacher's list, the student's listed logits
  for (int64_t i = tid; i < pieces; i += 256) {
    const Piece<T> p = rest_piece(i);
#pragma unroll
    for (int e = 0; e < N; ++e) m[0] = p.v[e] > m[0] || p.v[e] != p.v[e] ? p.v[e] : m[0];
  }
  block_max(m, share);
  const bool has_rest = m[0] != -INFINITY;
  const float at = a.tail && has_rest ? a.tail[row] : -INFINITY;   // no rest to put it on: the list alone
  const float ma = at > m[1] || at != at ? at : m[1];
  const float mz = m[0] > m[2] || m[0] != m[0] ? m[0] : m[2];
  const bool some = ma != -INFINITY && mz != -INFINITY;
  float s[3] = {0.0f, some ? expf(av - ma) : 0.0f, some ? expf(zs - mz) : 0.0f};
  if (has_rest)
    for (int64_t i = tid; i < pieces; i += 256) {
      const Piece<T> p = rest_piece(i);
#pragma unroll
      for (int e = 0; e < N; ++e) s[0] += expf(p.v[e] - m[0]);
    }
  block_sum(s, share);
  const float nan = __builtin_nanf("");
  const float rest = has_rest ? m[0] + logf(s[0]) : -INFINITY;
  const float lse = mz + logf(s[2] + (has_rest ? expf(rest - mz) : 0.0f));
  const float total = ma + logf(s[1] + (at != -INFINITY ? expf(at - ma) : 0.0f));
  const float logp = av - total, logq = zs - lse, p = expf(logp), q = expf(logq);
  const float pt = expf(at - total), qt = expf(rest - lse);
  float l[1] = {col >= 0 ? divergence(logp, p, logq, q) : 0.0f};
  block_sum(l, share);
  if (tid == 0 && a.loss)
    a.loss[row] = bad ? nan : some ? a.t * a.t * (l[0] + divergence(at - total, pt, rest - lse, qt)) : 0.0f;
  if (!a.grad) return;
  const float scale = a.t * a.grad_scale * (a.row_scale ? a.row_scale[row] : 1.0f);
  const float coef = bad ? nan : some ? scale * (qt - pt) : 0.0f;
  const float shift = has_rest ? rest : 0.0f;
  T *gr = a.grad + row * a.ldg;
  for (int64_t i = tid; i < pieces; i += 256) {
    Piece<T> g = rest_piece(i);
#pragma unroll
    for (int e = 0; e < N; ++e) g.v[e] = some || bad ? expf(g.v[e] - shift) * coef : 0.0f;
    store_piece(gr, i, a.cols, g);
  }
  __syncthreads();   // the list's own gradients overwrite what the pass left in their columns
  if (col >= 0 && some && !bad) gr[col] = static_cast<T>(scale * (q - p));
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
      hipLaunchKernelGGL(k_top<T>, dim3((unsigned)rows), dim3(256), 0, as_stream(stream), static_cast<const T *>(z),
                         ldz, cols, legal, ldl, k, 1.0f / temperature, values, index, tail);
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
      if (lds > 60 * 1024)
        FLY_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(&k_distill<T>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
      hipLaunchKernelGGL(k_distill<T>, dim3((unsigned)rows), dim3(256), lds, as_stream(stream), a);
      check_launch("distillation");
    });
  });
}
