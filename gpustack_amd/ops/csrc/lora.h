// What the adapters' launches and their binding share.
#pragma once

#include "common.h"

// mt, nt: a tile of the first launch in 16 rows and columns; held: of its workgroups a CU
// holds; up: rows of the second in 16.
struct LoraPlan { int mt, nt, held, up; };

// Tiles of `each` rows that T rows of S slots can need: at most T slots have rows.
static inline int lora_tiles(long T, long S, long each) {
  const long used = S < T ? S : T, most = (T + used * (each - 1)) / each;
  return (int)(most < T ? most : T);
}
