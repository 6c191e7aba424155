// What the kernel that widens a cache kept in 8 bits into dense bfloat16 tiles and the attention that reads the tiles share:
// the marks of a tile (AT_MARK words a (sequence, tile, kv head)).
#pragma once
#define AT_MARK 8                // words: flags, then a bit a key that is missing (up to 128)
#define AT_MARK_NAN 1u           // a key of the tile is NaN (a value that is makes its key so)
#define AT_MARK_MISSING 2u       // a key of the tile lies in a page that is not held
