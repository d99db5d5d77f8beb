// How flash_decode runs a call: which kernel, in tiles of how many rows, by CTAs of their own or along one line. Host code.
#pragma once

namespace fa {

// CTAs of a call on a B200's 148 SMs: two a SM for up to 16 rows, else one (their rings of tiles keep 192 KB a SM in flight
// either way). On a device with fewer SMs they run one after the other.
inline int decode_ctas(long long rows) { return rows <= 16 ? 296 : 148; }
// Rows (query heads of a key head times new tokens) of a row tile, of which a tile of keys is read once: 64 at most in
// decode_kernel, 128 in decode_wide_kernel.
inline int decode_part_rows(long long rows, bool wide) {
  return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 || !wide ? 64 : 128;
}
// Whether decode_wide_kernel takes a call: it starts and ends an item later by 5 us together, and takes half as long over a tile.
// `work`: tiles of keys a CTA, if all sequences were as long as they may be. us, decode_kernel -> decode_wide_kernel, 16 sequences of
// one length on 8 key heads (in brackets the tiles a CTA). d128: 32 rows (27) 37.0 -> 38.9, (48) 53.8 -> 53.8, (83) 82.8 -> 78.6,
// (166) 167 -> 140; 64 rows (6) 31.1 -> 32.2, (13) 41.9 -> 37.2, (27) 60.8 -> 48.8; 128 rows (3) 22.6 -> 31.0, (6) 32.9 -> 34.0, (10)
// 51.7 -> 36.9, (20) 81.4 -> 50.3. d64, where the borders are not the best ones: 32 rows (6) 18.0 -> 19.5, (13) 24.2 -> 24.1, (27)
// 37.5 -> 36.2, (41) 49.7 -> 45.6, (55) 61.9 -> 55.8; 64 rows (3) 19.2 -> 23.4, (6) 27.5 -> 27.0, (13) 37.9 -> 32.6; 128 rows (3) 21.6
// -> 28.7, (5) 28.1 -> 31.9, (6) 34.1 -> 34.1, (10) 53.2 -> 38.8. 2048 tokens of 32 heads on 8 over 8192 keys 1271 -> 404.
inline bool decode_wide(long long rows, long long work) { return rows > 16 && work >= (rows > 64 ? 5 : rows > 32 ? 10 : 48); }
// CTAs of a cluster that takes an item (a sequence, key head and tile of rows) of up to `tiles` tiles of keys as a whole, 1 for
// a CTA alone, or 0 where the items are cut by the line and joined by a second launch (which takes as long as four tiles or
// five). An item of two tiles has a CTA; short items of a large batch fill the SMs by their number; fewer items have clusters of
// up to eight CTAs, where a CTA's tiles are not many more than if the line had cut them, and uneven lengths cannot cost much.
// us, cut -> not cut (sequences x longest, key heads, head_dim): 1 x 512, 4, 64 8.6 -> 6.5; 1 x 512, 8, 128 8.2 -> 6.8;
// 1 x 2048, 8, 128 9.5 -> 9.1; 4 x 2048, 8, 128 11.7 -> 10.2; 128 x 400, 8, 128 48.5 -> 34.5; but 1 x 4096, 4, 64 8.8 -> 9.7.
inline int decode_cluster(long long tiles, long long items, int ctas) {
  if (tiles <= 2 || (tiles <= 8 && items >= ctas)) return 1;
  if (8 * items > ctas || tiles > 64 || tiles * (ctas - 8 * items) > 26ll * ctas) return 0;
  return tiles <= 4 ? 4 : 8;
}

struct DecodePlan {
  bool wide;            // decode_wide_kernel
  int ctas, part_rows;  // rows of a row tile
  long long row_tiles;  // of a key head
  long long items, tiles;  // (sequence, key head, row tile)s, and the tiles of keys that one may have
  int cluster;             // CTAs that take an item as a whole, or 0
};

// `room`: keys that a sequence may have; group: query heads of a key head.
inline DecodePlan decode_plan(int batch, int tokens, int group, int kv_heads, long long room, int window_left, int tile_keys) {
  const long long rows = static_cast<long long>(group) * tokens;
  long long longest = room;  // keys that an item may have
  if (window_left >= 0 && longest > static_cast<long long>(window_left) + tokens)
    longest = static_cast<long long>(window_left) + tokens;
  const auto row_tiles = [&](int of) { return (rows + of - 1) / of; };
  const long long heads = static_cast<long long>(batch) * kv_heads;
  DecodePlan d;
  d.ctas = decode_ctas(rows);
  d.tiles = (longest + tile_keys - 1) / tile_keys + (window_left >= 0);
  d.wide = decode_wide(rows, heads * row_tiles(128) * d.tiles / d.ctas);
  d.part_rows = decode_part_rows(rows, d.wide);
  d.row_tiles = row_tiles(d.part_rows);
  d.items = heads * d.row_tiles;
  d.cluster = decode_cluster(d.tiles, d.items, d.ctas);
  if (d.wide && d.cluster > 1) d.cluster = 0;
  return d;
}

}  // namespace fa
