// Which kernels a read-out loss takes and how its products are cut: host rules, free of GPU calls.  Times are of one MI355X.
#pragma once

#include <algorithm>
#include <cstdint>

#include "common.hpp"

namespace fly {

struct Call {
  int32_t type;
  int64_t rows, d, v, k;
  bool gx, gw, gb;
  bool grads() const { return gx || gw || gb; }
};

// The workgroup's tile (m x n): one plane 64 x 64 (4 waves), 128 x 128 (8) or 256 x 256 (16), two planes 64 x 64 (4), 128 x 128 (16) or
// 192 x 128 (8).  64 x 64, and 128 x 128 of one plane, run two workgroups per CU, the others one.
enum Shape { kSmall, kMedium, kLarge };
struct Tile {
  int m, n, places;   // and how many of them run at once
};
inline Tile tile_of(int planes, Shape s) {
  if (s == kSmall) return {64, 64, 512};
  if (s == kMedium) return {128, 128, planes == 2 ? 256 : 512};
  return planes == 2 ? Tile{192, 128, 256} : Tile{256, 256, 256};
}
inline int64_t tiles_of(const Tile &t, int64_t m, int64_t n) { return ((m + t.m - 1) / t.m) * ((n + t.n - 1) / t.n); }

// The logits' tile: the one whose rounds of workgroups cost least.  A round's cost, from one that fills it, in those of 128 x 128: one
// plane 0.5 (64 x 64) and 1.85 (256 x 256), two planes 0.72 and 1.6 (192 x 128).  Measured, us of the loss, 64 x 64 / 128 x 128 /
// large: bfloat16 2,333 into 4,168 256 rows 35 / 39 / 69, 1,120 rows 60 / 49 / 72, 4,096 rows 139 / 108 / 135, 10,000 rows 303 / 223 /
// 216; 1,024 into 32,000 1,120 rows 158 / 116 / 130, 4,096 rows 445 / 320 / 306; float32 2,333 into 4,168 256 rows 52 / 59 / 79, 543
// rows 76 / 62 / 81, 1,120 rows 105 / 105 / 88, 4,096 rows 301 / 259 / 239; 1,024 into 32,000 256 rows 116 / 101 / 119, 543 rows 191 /
// 170 / 152.
inline Shape logits_shape(int planes, int64_t m, int64_t n) {
  const double cost[3] = {planes == 2 ? 0.72 : 0.5, 1.0, planes == 2 ? 1.6 : 1.85};
  Shape best = kSmall;
  double least = 0.0;
  for (Shape s : {kSmall, kMedium, kLarge}) {
    const Tile t = tile_of(planes, s);
    const double c = cost[s] * (double)((tiles_of(t, m, n) + t.places - 1) / t.places);
    if (s == kSmall || c < least) best = s, least = c;
  }
  return best;
}
// Columns of the logits that a wave of a shape holds, 2 to the this, and how many such parts a row of `cols` columns has.
inline int part_shift(int planes, Shape s) { return s == kSmall || (planes == 2 && s == kMedium) ? 5 : 6; }
inline int parts_of(int planes, Shape s, int64_t cols) {
  const Tile t = tile_of(planes, s);
  return (int)((cols + t.n - 1) / t.n * (t.n >> part_shift(planes, s)));
}
// The tile of the gradients' products, whose tiles are counted together; parts of k even their rounds out.  One plane: up to 200 rows,
// whose product with the rows is soon over, 64 x 64 (bfloat16, 100 rows of 1,024 into 32,000 118 us against 126 and 129), else 256 x 256
// from 500 tiles on (1,120 rows 339 against 372; 2,333 into 4,168 4,096 rows, 330 tiles, 321 against 296), 128 x 128 from 600 on (1,120
// rows 125 against 130), else 64 x 64.  Two planes: 128 x 128 from 400 tiles on (4,096 rows 724 us, with 192 x 128 787, with 64 x 64 893;
// 256 rows 113, 124 and 117), else 64 x 64 (4,096 rows of 512 into 2,000 139 against 145).
inline Shape grad_shape(int planes, const Call &c, int64_t rows) {
  const int64_t m = (c.gx ? rows : 0) + (c.gw ? c.v : 0);
  if (planes == 2) return tiles_of(tile_of(2, kMedium), m, c.d) >= 400 ? kMedium : kSmall;
  if (rows <= 200) return kSmall;
  if (tiles_of(tile_of(1, kLarge), m, c.d) >= 500) return kLarge;
  return tiles_of(tile_of(1, kMedium), m, c.d) >= 600 ? kMedium : kSmall;
}

// In how many parts the k of the gradients' products run, side by side in one launch.  Jobs are counted in blocks of k of one tile; one
// that is longer than what each of the CUs' places gets keeps the others waiting.  A part costs its sums' way to memory and back, so
// none is shorter than 16 blocks, and all parts' sums fit kShareBytes.
constexpr int64_t kShareBytes = (int64_t)64 << 20;
struct Splits {
  int x = 1, w = 1;
};
inline Splits splits_of(int planes, const Call &c, int64_t rows) {
  const Tile t = tile_of(planes, grad_shape(planes, c, rows));
  const int64_t kx = (c.v + 31) / 32, kw = (rows + 31) / 32;
  const int64_t all = (c.gx ? tiles_of(t, rows, c.d) * kx : 0) + (c.gw ? tiles_of(t, c.v, c.d) * kw : 0);
  const double most = std::max(16.0, (double)all / (double)t.places);
  auto parts = [&](int64_t m, int64_t k) {
    const int64_t fit = kShareBytes / 2 / (m * round_up(c.d, 32) * 4);
    return (int)std::max<int64_t>(1, std::min((int64_t)((double)k / most + 0.99), fit));
  };
  Splits p;
  if (c.gx) p.x = parts(rows, kx);
  if (c.gw) p.w = parts(c.v, kw);
  return p;
}

// Up to 32 rows: at 32 of 2,333 into 4,168 the loss takes 27 us (float32) and 20 (bfloat16) against 43 and 34 with the operands laid
// out, with gradients 63 and 56 against 95 and 72.  At 48 the loss takes 49 against 43; float32 with gradients 92 against 98, and at
// 64 100 against 102 (1,024 into 32,000 219 against 250).  A small product's launches cost more than its work: 64 rows of 256 into
// 2,000 33 us against 40, 96 rows 37 against 40.
inline bool few_rows(const Call &c) {
  if (c.d < (c.type == FLY_F32 ? 4 : 8)) return false;   // rows have a whole piece
  const int64_t most = c.type == FLY_F32 && c.grads() ? 64 : 32;
  return c.rows <= most || (c.rows <= 96 && c.rows * c.d * c.v <= (int64_t)1 << 26);
}

// What a row's gradient is made of: p = exp2((z - top) log2 e - log_sum), u = share p - a / whole; 0 where the
// factor is 0 (share and whole 0).
struct RowInfo {
  float top, log_sum, share, whole;
};

// The largest of the weights' units and of the rows' factors times theirs, by which products over columns and over rows are scaled.  A
// factor times a unit may pass float32's range where the gradient does not: it is a double, and as floats power times fraction.
struct Maxima {
  double row;
  float weight, power, fraction;
};

// Rows run in pieces whose logits, u and x laid out take this much at most, and of as many rows: tiles of rows are counted in 16 bits.
constexpr int64_t kPieceBytes = (int64_t)1 << 32;
constexpr int64_t kPieceRows = (int64_t)1 << 19;

// Where everything lies in the workspace.
struct Space {
  int64_t piece;      // rows at a time
  int64_t db, vb, rb; // blocks of 32
  int parts;
  bool several;
  size_t x, xt, w, wt, z, g, gt, unit_x, unit_w, bias, stat, info, factor, turned, sums, maxima, acc_w, acc_b, column, weight,
      logit, list_sums, share_x, share_w, bytes;
  Space(const Call &c, int planes) {
    db = (c.d + 31) / 32;
    vb = (c.v + 31) / 32;
    parts = parts_of(planes, kSmall, vb * 32);   // the most that a shape has, but for a tile's rounding
    parts = (int)round_up(parts, 4);
    const int64_t kept = c.grads() ? planes * 2 : 0;   // bytes of a logit
    const int64_t each = vb * 32 * (kept + 2 * planes * ((c.gx ? 1 : 0) + (c.gw ? 1 : 0))) + db * 64 * planes * (c.gw ? 2 : 1) +
                         12 * c.k + 8 * parts_of(planes, kSmall, vb * 32);
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
    z = kept ? take(piece * vb * 32 * kept) : 0;
    g = c.gx ? take(rb * vb * block) : 0;
    gt = c.gw ? take(rb * vb * block) : 0;
    unit_x = take(rb * 32 * 4);
    unit_w = take(vb * 32 * 4);
    bias = take(vb * 32 * 4);
    stat = take(piece * parts * 8);
    info = take(piece * sizeof(RowInfo));
    factor = take(piece * 4);
    turned = take(piece * 8);
    sums = c.gb ? take(piece / 64 * vb * 32 * 4) : 0;
    maxima = take(sizeof(Maxima));
    acc_w = several && c.gw ? take(c.v * db * 32 * 4) : 0;
    acc_b = several && c.gb ? take(vb * 32 * 4) : 0;
    column = take(piece * c.k * 4);
    weight = take(piece * c.k * 4);
    logit = take(piece * c.k * 4);
    list_sums = take(piece * 8);
    const Splits p = splits_of(planes, c, piece < c.rows ? piece : c.rows);
    share_x = several && c.gx ? take(kShareBytes / 2) : p.x > 1 ? take(p.x * c.rows * db * 128) : 0;
    share_w = several && c.gw ? take(kShareBytes / 2) : p.w > 1 ? take(p.w * c.v * db * 128) : 0;
    bytes = at;
  }
};

}  // namespace fly
