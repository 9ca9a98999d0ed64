// quant_grid.hpp -- which workgroup of a product with 4-bit weights takes what.  A
// workgroup takes a set of tiles of outputs and a block of tokens.
#pragma once

namespace glacier {

struct QuantPlace {
  int set, block;
};
// Sets are taken eight abreast, all blocks of tokens of the eight in a row: workgroups go
// round the eight XCDs, so a set's blocks are on one, whose L2 has its weights then.  The
// last ones, fewer than eight, go round with as many as they are: every workgroup has
// work.  [2048] 896 -> 896, 128, 128: 576 workgroups, 17.3 us; rounded up to eight abreast
// 1024, whose surplus worked for nothing, 22.6.
constexpr int kQuantAbreast = 8;
constexpr QuantPlace quant_place(int number, int sets, int blocks) {
  if (blocks == 1) return {number, 0};
  const int round = number / (kQuantAbreast * blocks), first = round * kQuantAbreast;
  const int width = sets - first < kQuantAbreast ? sets - first : kQuantAbreast;
  const int rest = number - first * blocks;
  return {first + rest % width, rest / width};
}
// Workgroups of a call: numbers below this are places, each one once.
constexpr int quant_grid(int sets, int blocks) { return sets * blocks; }

}  // namespace glacier
