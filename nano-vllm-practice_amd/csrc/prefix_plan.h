// Pieces of a shared prefix, by the call's shape (host code, no HIP).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace femto {

constexpr int kPrefixTile = 64;  // keys of a key tile

// The one statement of how a prefix is cut: the tile kernel takes piece i as
// the keys [i * piece_keys, (i + 1) * piece_keys) and the merge expects the
// states of ceil(keys / piece_keys) pieces from a sequence that sees `keys` of
// the prefix.
struct PrefixPieces {
    int pieces, piece_keys;
    bool longest;  // the tiles outlast the tails
};

// n_heads / group and rows_per_tile: the tile kernel's head groups and the
// query tokens (here sequences) of its tiles; tail: keys of the longest tail.
//
// More pieces shorten the tiles' chains (1.2 us per tile of 64 keys where a CU
// has one), but each writes and merges 520 bytes per query row.  With T key
// tiles and R query rows the best of 2 .. 64 pieces was near
// 2 sqrt(T) / (1 + R / 24 / 128) over 160 shapes (3-256 sequences, prefixes of
// 256-16384 keys, five head shapes): 16384 keys, 16 sequences on 16/8 heads
// 28 us with 32, 31 with 16, 45 with 8; 256 on 64/8 heads 195 us with 4, 231
// with 16; 4096 keys, 8 on 16/8 heads 15.2 with 16, 16.6 with 12, 18.9 with 8.
// Beyond one workgroup per CU beside the workers (a row tile is one workgroup
// per piece) they only queue (4096 keys, 256 sequences on 16/8 heads with tails
// of up to 512: 65 us with 4, 71 with 8, 79 with 16).
inline PrefixPieces prefix_pieces(int num_seqs, int n_heads, int n_kv_heads, int group, int rows_per_tile,
                                  int prefix_keys, int tail, int cus) {
    PrefixPieces p{0, 0, false};
    if (prefix_keys <= 0) return p;
    const int tiles = (prefix_keys + kPrefixTile - 1) / kPrefixTile;
    const double units = (double)(n_heads / group) * ((num_seqs + rows_per_tile - 1) / rows_per_tile);
    const double rows = (double)num_seqs * n_heads;
    const double best = std::min(2.0 * std::sqrt((double)tiles) / (1.0 + rows / (24.0 * 128)), std::max(4.0, cus / units));
    const int at_least = std::max({1, (tiles + 63) / 64, (int)(tiles / best + 0.5)});
    p.pieces = (tiles + at_least - 1) / at_least;
    const int per = (tiles + p.pieces - 1) / p.pieces;  // as even as that many pieces can be
    p.piece_keys = per * kPrefixTile;
    // Where the tiles outlast the tails their waves issue before the workers' on
    // the same SIMD: from one tile of 64 keys for 11 pages of the tails on (it takes
    // ~1.2 us of a CU, a page of a KV head, 8 KB, 1.4 ns of HBM time; the host knows
    // the longest tail only, which is about twice the mean), and where a workgroup's
    // chain is 5 tiles or more (of 1-4 it cost 2.5-6 % on average).
    // Measured with and without over 2,051 shapes (4-256 sequences, prefixes of
    // 256-16384 keys, longest tails of 1/64 to 1/2 of them, six head shapes): where it
    // is taken 1.9 % faster on average, and over all shapes 0.3 % behind the better of
    // the two, 8 % at worst (never ahead 1.0 and 15, always 2.7 and 17).  16384 keys,
    // 256 sequences, longest tails of 1638, 1365 and 1024 keys, us: 32/8 heads 175 and
    // 181, 164 and 158, 153 and 141; 16/8 heads (half the tiles), 1024, 819 and 512:
    // 113 and 120, 97 and 105, 84 and 82; 64/8 heads, 4096, 2048: 399 and 405, 294 and 267.
    const double tail_pages = (double)num_seqs * n_kv_heads * (tail / 16.0);
    p.longest = per >= 5 && 11 * units * tiles >= tail_pages;
    return p;
}

}  // namespace femto
