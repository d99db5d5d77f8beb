// Host build of csrc/decode_plan.h for tests/test_decode_plan*.py.
#include "decode_plan.h"

extern "C" {

// args: batch, tokens, query heads of a key head, key heads, keys that a sequence may have, window, head_dim;
// out: wide, rows of a row tile, row tiles of a key head, items, CTAs of a cluster, CTAs, tiles that an item may have
void plan(const long long* args, long long* out) {
  const fa::DecodePlan d = fa::decode_plan(static_cast<int>(args[0]), static_cast<int>(args[1]), static_cast<int>(args[2]),
                                           static_cast<int>(args[3]), args[4], static_cast<int>(args[5]), args[6] == 128 ? 64 : 128);
  const long long all[] = {d.wide, d.part_rows, d.row_tiles, d.items, d.cluster, d.ctas, d.tiles};
  for (int i = 0; i < 7; ++i) out[i] = all[i];
}
}
