// How a call of the 8-bit integer product is cut into tiles and how many
// stages a CTA's ring has (host code, shared by the launch and its test).
#pragma once

#include <algorithm>
#include <cstdint>

namespace ms {

constexpr int kI8Rows = 128;      // channels of a tile
constexpr int kI8Step = 128;      // bytes of K of a stage
constexpr int kI8MaxStages = 10;
constexpr int kI8Cols = 256;      // columns of an accumulator
constexpr int kI8Ring = 208 * 1024;

// Tiles of a call: tokens (bn) and channels (rows) of one, and whether two SMs
// share it, by the clocks that the busiest SM needs.
struct I8Tiling {
  int bn, rows;
  bool pair;
};

inline I8Tiling i8_tiling(int64_t M, int64_t N, int64_t K, int out_size, int sms) {
  I8Tiling best{};
  double least = 0;
  const double steps = (double)((K + kI8Step - 1) / kI8Step);
  for (int pair = 0; pair < 2; ++pair) {
    const int ctas = pair + 1, grain = 16 * ctas;
    const int64_t workers = sms / ctas, parts0 = (M + kI8Cols - 1) / kI8Cols;
    int seen = 0;
    for (int64_t parts = parts0; parts < parts0 + 12; ++parts) {
      // equal token tiles, rounded up to what an N of the product, and half of it for a pair, allow
      const int bn = (int)(((M + parts - 1) / parts + grain - 1) / grain * grain);
      if (bn == seen) continue;
      seen = bn;
      const int64_t tok_tiles = (M + bn - 1) / bn;
      // 128 channels, or the same rounds of tiles with the channels spread evenly over them
      for (int spread = 0; spread < 2 - pair; ++spread) {
        int64_t rows = kI8Rows;
        int64_t tiles = (N + rows * ctas - 1) / (rows * ctas) * tok_tiles;
        const int64_t rounds = (tiles + workers - 1) / workers;
        if (spread) {
          const int64_t most = rounds * workers / tok_tiles;
          if (most < 1) continue;
          rows = (N + most - 1) / most;
          if (rows > kI8Rows) continue;
        }
        // a step of 128 bytes of K: the products (512 clocks for 256 tokens), the SM's reads (64 bytes a clock,
        // 24 of them from HBM where no other tile uses the weights); the stores run under the next tile's
        // steps, whole lines at 24 bytes a clock, others slower (512 x 896 x 151936: 102 us, 117 us with odd
        // tiles); what is hidden still takes a part of the SM's way to L2
        const double reads = (rows + bn / ctas) * 128 / 60.0, hbm = tok_tiles == 1 ? rows * 128 / 24.0 : 0;
        const double step = std::max(2.0 * bn, std::max(reads, hbm));
        const double store = (double)rows * std::min<int64_t>(bn, M) * out_size / (rows % 32 ? 16 : 24);
        const double cost = rounds * (std::max(steps * step, store) + 0.3 * std::min(steps * step, store)) + store;
        if (!best.bn || cost < least) best = {bn, (int)rows, pair != 0}, least = cost;
      }
    }
  }
  return best;
}

// A stage: 128 channels and a CTA's tokens of one step of K.
inline int i8_stage_bytes(int bn, bool pair) { return (kI8Rows + bn / (pair ? 2 : 1)) * kI8Step; }

inline int i8_stages(int64_t M, int64_t K, int bn, bool pair) {
  const int fit = kI8Ring / i8_stage_bytes(bn, pair);
  // One narrow tile of tokens and rows that are not long: all SMs only stream weights, and fewer bytes in flight on
  // each do better, six stages against ten: 1 x 896 x 151936 27.8 against 28.3 us, 16 x 896 x 156250 26.7 against
  // 28.7, 16 x 4096 x 34179 26.3 against 26.4.  Not past 16 tokens (24 x 896 x 156250 33.5 against 29.1, 30 x 4096 x
  // 60000 54.4 against 46.6), nor with longer rows (16 x 8192 x 8192 19.3 against 17.6).
  if (M <= 16 && K <= 4096 && fit > 6) return 6;
  return fit < kI8MaxStages ? fit : kI8MaxStages;
}

}  // namespace ms
