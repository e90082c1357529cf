// Which workgroup a row of logits takes: host rules, free of GPU calls.  Times are of one MI355X.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace fly {

// How many pieces a thread keeps and how many threads a row gets.  Few rows: the fewest of {1, 2, 4, 8} pieces that 512
// threads cover a row with.  From 1,024 rows on (4 for each CU) at least `many`, since what a wave does once per row weighs
// more than the waves that are left idle: 8 for the top logits (1,500 x 4,168 float32 12.1 us with 8, 14.7 with 4), 4 for
// the distillation, whose 8 cost it registers (with gradient: 16,384 x 4,168 float16 57 us with 4, 64 with 8, 77 with 2;
// float32 100, 112 with 8; 16,384 x 1,000 float32 26.6, 30.6 with 8).  Past 512 threads 1,024 of them, as two workgroups of
// 16 waves fill a CU evenly (8 pieces: 2,048 x 50,256 95 us, with the 832 threads that it needs 111).  For many rows that is
// where `many` pieces need them (distillation, 4 pieces on 1,024 threads against 8 on 512: 4,096 x 32,000 bfloat16 102 us
// against 110 with gradient, but 58 against 47 without; 4,096 x 12,000 float32 76 against 82), for few only where 8 do (256 x
// 12,000 float32 with 4 13.0 us, with 8 11.4).  Longer rows are read at every pass (kept = 0).  Loss and gradient take the
// same shape, so the loss has the same bits with the gradient and alone.
struct RowShape {
  int kept, threads;
};
inline RowShape row_shape(int64_t rows, int64_t cols, size_t elem, int least, int many) {
  const int64_t pieces = (cols * (int64_t)elem + 15) / 16;   // whole ones at most
  for (int kept : {1, 2, 4, 8}) {
    const int64_t threads = std::max<int64_t>(round_up((pieces + kept - 1) / kept, 64), least);
    const bool enough = kept >= many;
    if (threads <= 512 && (enough || rows < 1024)) return {kept, (int)threads};
    if (threads <= 1024 && (kept == 8 || (enough && rows >= 1024))) return {kept, 1024};
  }
  return {0, 1024};
}

constexpr int kWaveCandidates = 128;   // what a wave may find above the bound of the top logits

// How many logits of a wave are expected to reach the bound of k largest that `holders` waves give, each lane holding `per`
// logits in any order.  A wave has c = ceil(k / holders) lanes whose largest is at or above its bound; the last one may hold
// few lanes of the row's `full` whole pieces, and bounds it lowest: a share c / lanes of all lanes passes there, and of
// their logits 1 - (1 - share)^(1 / per).
inline double expected_candidates(int full, double per, int holders, int k) {
  const int lanes = std::min(64, full - 64 * (holders - 1)), c = (k + holders - 1) / holders;
  const double share = c < lanes ? 1.0 - std::pow(1.0 - (double)c / lanes, 1.0 / per) : 1.0;
  return std::min(64, full) * per * share;
}

// The top logits' workgroup: twice as many lanes as k (16,384 x 4,168 float16, k = 200: 204 us against 214 with as many; 4,000
// x 20,000 74 against 181), and `holders`, the waves that bound the row: all that hold whole pieces, or all but the last
// where that one's few lanes would give a low bound or none (1,000 x 2,060 float16, k = 32: 10.4 us, 24.6 with it).  Where more
// than 80 logits of a wave are expected to pass even so, its list of 128 may overflow, and the row would go to the search
// that ties need.  It is spread over 4 waves column by column then (spread: columns a thread) and bounded by all its logits
// (1,000 x 560 float32, k = 64 10.0 us against 13.6; 20,000 x 700 float16, k = 64 93 against 121).  Not past 4,096 columns,
// nor for a small k of many short rows, where the search costs less (20,000 x 200 float16, k = 64 72 us against 97, k = 128
// 108 against 97).
struct TopShape {
  RowShape row;
  int holders, spread;
};
inline TopShape top_shape(int64_t rows, int64_t cols, size_t elem, int k) {
  const RowShape row = row_shape(rows, cols, elem, (int)round_up(2 * k, 64), 8);
  const int full = (int)(cols * (int64_t)elem / 16);
  int holders = std::max(1, std::min(row.threads, full + 63) / 64);
  const double per = 16.0 / (double)elem * std::max(1.0, (double)full / row.threads);
  double most = expected_candidates(full, per, holders, k);
  if (holders > 1) {
    const double without = expected_candidates(full, per, holders - 1, k);
    if (without < most) {
      most = without;
      --holders;
    }
  }
  const bool search = cols > 4096 || (rows >= 1024 && cols <= 400 && k <= 64);
  const int spread = cols <= kWaveCandidates || most <= 80 || search ? 0 : cols <= 1024 ? 4 : 16;
  if (spread) holders = (int)std::min<int64_t>(4, (cols + 63) / 64);
  return {row, holders, spread};
}

}  // namespace fly
