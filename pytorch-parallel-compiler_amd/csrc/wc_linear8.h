// Which kernel makes an 8-bit product: rules on its tiles of 16 rows, 16 outputs and 64 columns, of all models.
#pragma once

#include <cstdint>

namespace wc {

constexpr int kFusedPieces = 1024;         // pieces of 16 columns that a workgroup finds the codes of for itself
constexpr int kLargeTiles = 16;            // tiles along each side of the largest

enum class Linear8Form { fused, few, ring6, ring3, large, tiles };

inline Linear8Form linear8_form(int64_t n, int64_t m, int64_t mtiles, int64_t otiles, int64_t ktiles) {
  auto over = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  if (m <= 16 && m * ktiles * 4 <= kFusedPieces) return Linear8Form::fused;
  // A workgroup for each 16 rows and outputs while all of them are at work at once, eight a compute unit: W comes from L2 for all
  // rows but the first 16, which costs less than long walks on few units do (129 rows [7280 -> 416], two models, codes
  // included: 51 us by tiles of 64 x 128, 30 so; 128 rows [4096 -> 4096], 2048 of them: 36.6 and 32.4; 293 rows [6832 -> 1004], 2394
  // of them: 50 and 64).
  if (mtiles == 1 || n * mtiles * otiles <= 2048) return Linear8Form::few;
  // Where tiles are fewer than compute units, one has a unit's LDS to itself and more stages on their way (293 rows [6832 -> 1004], two
  // models: by tiles of 128 x 128 in two stages 62 us, so 50).
  if (n * over(mtiles, 4) * over(otiles, 8) <= 256) return Linear8Form::ring6;
  if (mtiles <= 4) return Linear8Form::ring3;
  // The largest tiles where few units are left without one (2 models' 1280 rows [2048 -> 4096], 160 of them: 45.9 us, by tiles of 128 x 128
  // 55.7; 2048 rows [4096 -> 4096], 128 of them: 67.8 and 61.5)
  if (n * over(mtiles, kLargeTiles) * over(otiles, kLargeTiles) >= 150) return Linear8Form::large;
  return Linear8Form::tiles;
}

}  // namespace wc
