// How the keys of a (sample, head) are shared out where its rows are few: arithmetic alone, the same on the host and the device.
#pragma once

// Share y of `shares` over `count` keys in tiles of `tile` keys: the tiles [t0, t1), even to one tile, and the end of their keys.
// `end` is what a share's buffer descriptors cover: never more than `count`, so that the hardware's bounds check holds for every
// request, and a share without tiles (t0 == t1) makes none.
struct KeyShare { int t0, t1, end; };
constexpr KeyShare key_share(int count, int tile, int shares, int y) {
  const unsigned tiles = ((unsigned)count + tile - 1) / tile;   // at most 2^19 tiles and 64 shares: the products fit
  const int t0 = (int)(tiles * y / shares), t1 = (int)(tiles * (y + 1) / shares);
  return {t0, t1, t1 * tile < count ? t1 * tile : count};
}
