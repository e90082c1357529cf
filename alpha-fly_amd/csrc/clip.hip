// The norm of many tensors together, and their scaling by it.
//
//   norm = sqrt(sum g^2)  or  max |g|,    c = min(1, limit / (norm + 1e-6)),    g <- c g
//
// Two passes, each one launch for up to 128 tensors: their addresses and sizes travel in the launch's own arguments, and a
// workgroup finds the tensor of its next chunk there, so the tensors' number costs no launches and no copy.  Squares are added
// in float64: exact products of float32, whose sums neither overflow nor lose small tensors beside large ones; the conversions
// and sums take less than the memory's time.  Each workgroup leaves one partial sum, in an order that depends on the sizes
// alone, and every workgroup of the second pass adds them all up: 2,048 at most, from the L2.
//
// Bound by memory: 38 million float32 gradients below their limit 33 us a call (153 MB read once, 4.7 TB/s), 454 million bfloat16 ones
// above it 524 us (read twice and written: 5.2 TB/s, as a copy) and below it 160 us.
#include "rows.hpp"

#include <cmath>

namespace fly {
namespace {

constexpr int kTensors = 128;           // of a launch: 2.7 KB of its 4 KB of arguments
constexpr int kThreads = 256, kPieces = 8;
constexpr int kChunk = kThreads * kPieces * 16;   // bytes of a chunk
constexpr int kGroups = 2048;           // workgroups of a pass, and partial sums, at most

struct Table {
  void *p[kTensors];
  int64_t n[kTensors];              // elements
  uint32_t first[kTensors + 1];     // the tensor's first chunk
  uint8_t type[kTensors];
  int32_t tensors;
};

template <bool MAX>
__device__ __forceinline__ double merge(double a, double b) {
  if constexpr (MAX) return b > a || b != b ? b : a;
  else return a + b;
}

// over the workgroup, in every thread; `share` holds kThreads / 64 doubles
template <bool MAX>
__device__ __forceinline__ double block_merge(double v, double *share) {
  for (int d = 1; d < 64; d <<= 1) v = merge<MAX>(v, __shfl_xor(v, d));
  if ((threadIdx.x & 63) == 0) share[threadIdx.x >> 6] = v;
  __syncthreads();
  v = share[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) v = merge<MAX>(v, share[w]);
  return v;
}

// f(tensor, byte offset of the chunk) for this workgroup's chunks; BACK: the last ones first.
template <bool BACK, typename F>
__device__ __forceinline__ void each_chunk(const Table &t, F &&f) {
  const uint32_t chunks = t.first[t.tensors];
  int i = BACK ? t.tensors - 1 : 0;
  for (uint32_t k = blockIdx.x; k < chunks; k += gridDim.x) {
    const uint32_t c = BACK ? chunks - 1 - k : k;
    if constexpr (BACK) while (c < t.first[i]) --i;
    else while (c >= t.first[i + 1]) ++i;
    f(i, (int64_t)(c - t.first[i]) * kChunk);
  }
}

template <typename T, typename F>
__device__ __forceinline__ void each_value(const T *p, int64_t left, F &&f) {
  constexpr int N = Piece<T>::N;
  if (left >= kChunk / (int)sizeof(T)) {
    Raw16 raw[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) raw[j] = load_whole(p, threadIdx.x + kThreads * j);
#pragma unroll
    for (int j = 0; j < kPieces; ++j)
#pragma unroll
      for (int e = 0; e < N; ++e) f(element<T>(raw[j], e));
  } else {
    for (int64_t i = threadIdx.x; i * N < left; i += kThreads) {
      const Piece<T> v = load_piece(p, i, left, 0.0f);   // zeros past the end change neither sum nor maximum
#pragma unroll
      for (int e = 0; e < N; ++e) f(v.v[e]);
    }
  }
}

template <typename T, typename F>
__device__ __forceinline__ void change_values(T *p, int64_t left, F &&f) {
  constexpr int N = Piece<T>::N;
  if (left >= kChunk / (int)sizeof(T)) {
    Raw16 raw[kPieces];
#pragma unroll
    for (int j = 0; j < kPieces; ++j) raw[j] = load_whole(p, threadIdx.x + kThreads * j);
#pragma unroll
    for (int j = 0; j < kPieces; ++j) {
      Piece<T> v;
#pragma unroll
      for (int e = 0; e < N; ++e) v.v[e] = f(element<T>(raw[j], e));
      store_whole<T, false>(p, threadIdx.x + kThreads * j, v);
    }
  } else {
    for (int64_t i = threadIdx.x; i < left; i += kThreads) p[i] = static_cast<T>(f(static_cast<float>(p[i])));
  }
}

template <typename F>
__device__ __forceinline__ void typed(uint8_t type, void *p, int64_t bytes, int64_t n, F &&f) {
  if (type == FLY_F32) f(reinterpret_cast<float *>(static_cast<char *>(p) + bytes), n - bytes / 4);
  else if (type == FLY_F16) f(reinterpret_cast<_Float16 *>(static_cast<char *>(p) + bytes), n - bytes / 2);
  else f(reinterpret_cast<bhalf *>(static_cast<char *>(p) + bytes), n - bytes / 2);
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void k_norm(const Table t, double *__restrict__ parts) {
  __shared__ double share[kThreads / 64];
  double sum = 0.0;
  each_chunk<false>(t, [&](int i, int64_t at) {
    typed(t.type[i], t.p[i], at, t.n[i], [&](auto *p, int64_t left) {
      using T = std::remove_pointer_t<decltype(p)>;
      each_value<T>(p, left, [&](float v) {
        if constexpr (MAX) sum = merge<true>(sum, (double)fabsf(v));
        else sum = fma((double)v, (double)v, sum);
      });
    });
  });
  sum = block_merge<MAX>(sum, share);
  if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

template <bool MAX>
__device__ __forceinline__ double join(const double *__restrict__ parts, int count, double *share) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) sum = merge<MAX>(sum, parts[i]);
  return block_merge<MAX>(sum, share);
}

template <bool MAX>
__global__ __launch_bounds__(kThreads) void k_norm_join(const double *__restrict__ parts, int count, double *__restrict__ one,
                                                        float *__restrict__ norm) {
  __shared__ double share[kThreads / 64];
  const double sum = join<MAX>(parts, count, share);
  if (threadIdx.x == 0) {
    if (one) *one = sum;
    if (norm) *norm = static_cast<float>(MAX ? sum : sqrt(sum));
  }
}

// The chunks that the first pass read last come first: up to 256 MB of them are still in the Infinity Cache.
template <bool MAX>
__global__ __launch_bounds__(kThreads) void k_clip(const Table t, const double *__restrict__ parts, int count, float limit,
                                                   float *__restrict__ norm) {
  __shared__ double share[kThreads / 64];
  const double sum = join<MAX>(parts, count, share);
  const float n = static_cast<float>(MAX ? sum : sqrt(sum)), c = limit / (n + 1e-6f);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  if (c >= 1.0f) return;   // every value would be written as it is; a NaN goes on
  each_chunk<true>(t, [&](int i, int64_t at) {
    typed(t.type[i], t.p[i], at, t.n[i], [&](auto *p, int64_t left) {
      using T = std::remove_pointer_t<decltype(p)>;
      change_values<T>(p, left, [&](float v) { return v * c; });
    });
  });
}

int64_t elem_bytes(int32_t type) { return type == FLY_F32 ? 4 : 2; }
int64_t chunks_of(int64_t n, int32_t type) { return (n * elem_bytes(type) + kChunk - 1) / kChunk; }

// f(table, workgroups) for each launch's tensors.
template <typename F>
void each_table(void *const *grads, const int64_t *sizes, const int32_t *types, int64_t n, F &&f) {
  for (int64_t i = 0; i < n;) {
    Table t;
    int64_t chunks = 0;
    t.tensors = 0;
    for (; i < n && t.tensors < kTensors; ++i) {
      if (!sizes[i]) continue;
      const int64_t c = chunks_of(sizes[i], types[i]);
      if (chunks && chunks + c >= INT32_MAX) break;
      t.p[t.tensors] = grads ? grads[i] : nullptr;
      t.n[t.tensors] = sizes[i];
      t.type[t.tensors] = (uint8_t)types[i];
      t.first[t.tensors++] = (uint32_t)chunks;
      chunks += c;
    }
    t.first[t.tensors] = (uint32_t)chunks;
    if (t.tensors) f(t, (int)std::min<int64_t>(chunks, kGroups));
  }
}

void require_sizes(const int64_t *sizes, const int32_t *types, int64_t n) {
  FLY_REQUIRE(n >= 0 && n < (1 << 24), "bad number of tensors");
  FLY_REQUIRE(!n || (sizes && types), "null pointer");
  for (int64_t i = 0; i < n; ++i) {
    FLY_REQUIRE(sizes[i] >= 0 && sizes[i] < ((int64_t)1 << 40), "bad size");
    FLY_REQUIRE(types[i] >= FLY_F32 && types[i] <= FLY_BF16, "gradients must be float32, float16 or bfloat16");
  }
}

size_t clip_ws(const int64_t *sizes, const int32_t *types, int64_t n) {
  int64_t parts = 0;
  each_table(nullptr, sizes, types, n, [&](const Table &, int groups) { parts += groups; });
  return (size_t)(parts + 1) * sizeof(double);
}

template <bool MAX>
void clip(void *const *grads, const int64_t *sizes, const int32_t *types, int64_t n, float limit, float *norm, double *parts,
          hipStream_t st) {
  int count = 0;
  each_table(grads, sizes, types, n, [&](const Table &t, int groups) {
    hipLaunchKernelGGL(k_norm<MAX>, dim3(groups), dim3(kThreads), 0, st, t, parts + count);
    check_launch("gradient norm");
    count += groups;
  });
  const bool scale = limit >= 0.0f;
  // without a second pass, or with more sums than each of its workgroups should add up, one workgroup does
  if (!scale || count > kGroups || !count) {
    hipLaunchKernelGGL(k_norm_join<MAX>, dim3(1), dim3(kThreads), 0, st, parts, count, parts + count, norm);
    check_launch("gradient norm");
    if (!scale) return;
    parts += count;
    count = 1;
    norm = nullptr;
  }
  each_table(grads, sizes, types, n, [&](const Table &t, int groups) {
    hipLaunchKernelGGL(k_clip<MAX>, dim3(groups), dim3(kThreads), 0, st, t, parts, count, limit, norm);
    check_launch("gradient clipping");
  });
}

}  // namespace
}  // namespace fly

using namespace fly;

extern "C" size_t fly_clip_workspace(const int64_t *sizes, const int32_t *types, int64_t n) {
  size_t bytes = 0;
  guard([&] {
    require_sizes(sizes, types, n);
    bytes = clip_ws(sizes, types, n);
  });
  return bytes;
}

extern "C" int fly_clip_gradients(void *const *grads, const int64_t *sizes, const int32_t *types, int64_t n, int32_t norm_kind,
                                  float limit, float *norm, void *ws, size_t ws_bytes, void *stream) {
  return guard([&] {
    require_sizes(sizes, types, n);
    FLY_REQUIRE(norm_kind == FLY_NORM_2 || norm_kind == FLY_NORM_MAX, "the norm must be FLY_NORM_2 or FLY_NORM_MAX");
    FLY_REQUIRE(limit == limit, "the limit must not be NaN");
    FLY_REQUIRE(norm != nullptr && (!n || grads), "null pointer");
    FLY_REQUIRE(ws && ws_bytes >= clip_ws(sizes, types, n) && aligned(ws, 8), "workspace too small or misaligned");
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (int64_t i = 0; i < n; ++i) {
      if (!sizes[i]) continue;
      FLY_REQUIRE(grads[i] && aligned(grads[i], (size_t)elem_bytes(types[i])), "a gradient is null or misaligned");
      const uintptr_t p = reinterpret_cast<uintptr_t>(grads[i]);
      spans.emplace_back(p, p + (uintptr_t)(sizes[i] * elem_bytes(types[i])));
    }
    if (limit >= 0.0f) {   // scaled twice, in no order, where they overlap
      std::sort(spans.begin(), spans.end());
      for (size_t i = 1; i < spans.size(); ++i) FLY_REQUIRE(spans[i].first >= spans[i - 1].second, "gradients overlap");
    }
    double *parts = static_cast<double *>(ws);
    if (norm_kind == FLY_NORM_2) clip<false>(grads, sizes, types, n, limit, norm, parts, as_stream(stream));
    else clip<true>(grads, sizes, types, n, limit, norm, parts, as_stream(stream));
  });
}
