// The units of time in which drafted trees' blocks are dealt out (see attn_deal.h, whose arithmetic this is: the device and a test on the host run the same).
#pragma once
#include <stdint.h>

namespace pimdl {
namespace attn {

constexpr uint32_t DEAL_BATCH = 512;  // rows of the batch that fit
// Units are a 14th of the time that a tile takes with 256 rows.  Measured, 40 sequences with blocks of 2 to 8 groups of 32 rows each, us a tile: of 64 keys 1.86, 2.13, 2.19, 2.57, 2.81,
// 3.32, 3.54 (bf16, 128 dims), 1.11, 1.46, 1.53, 1.83, 1.91, 2.40, 2.47 (fp16, 64), 2.35, 3.08, 3.31, 4.00, 4.33, 5.44, 5.72 (fp32, 64); of 32 keys, which waves do not share, 2.25, 2.41, 2.54,
// 3.30, 3.58, 3.72, 3.95 (fp32, 80), 3.18, 3.35, 3.59 (fp32, 128).
template <int TILE>
constexpr uint32_t tile_units(uint32_t groups)
{
    if (TILE == 64) return groups + (groups > 6 ? 6 : 5);
    return groups <= 4 ? 8 + groups / 3 : 10 + groups / 2;
}
constexpr uint32_t TILE_MOST = 8;     // units of a tile for each of a block's groups, at most
constexpr uint32_t DEAL_BLOCK = 36;   // units of a block without its tiles: its queries, the first keys' way and the results (10 to 12, 5.5 to 7.4, 8 to 10, 7 to 9 and 6 to 9 us)
constexpr uint32_t DEAL_SHORT = 64;   // units of tiles up to which a block is not worth cutting
constexpr uint32_t DEAL_LEAST = 48;   // units of a share, at least

// Units of `rows` query rows in `batch` sequences over up to `keys` keys each, at most
constexpr uint64_t deal_most_units(uint64_t rows, uint32_t batch, uint32_t kv_heads, uint64_t keys, uint32_t tile)
{
    const uint64_t groups = rows / 32 + batch;  // (of 32 rows)
    return groups * kv_heads * (TILE_MOST * (keys / tile + 1) + DEAL_BLOCK);
}

// Sums of units end at 2^31 - 1, which the host makes sure that rows with tokens of their own do not reach: starts that fall again, so that rows share tokens, could, and
// the last rows get nothing then.
constexpr uint32_t add_units(uint32_t x, uint32_t y)
{
    const uint32_t sum = x + y;
    return sum < 0x7fffffffu ? sum : 0x7fffffffu;
}

constexpr uint32_t share_of(uint32_t total, uint32_t shares)
{
    const uint32_t s = (total + shares - 1) / shares;
    return s > DEAL_LEAST ? s : DEAL_LEAST;
}

// A row of the batch: blocks of its rows, equal ones as near as groups of 32 allow, and tiles of keys (a block without keys has one, so that somebody writes its zeros)
struct DealRow {
    uint32_t blocks, rows, tiles;  // rows: of a block but the last
    uint32_t whole, last;          // units of a tile of a block, and of the last one
    constexpr uint32_t block_units(uint32_t each) const { return DEAL_BLOCK + each * tiles; }
    constexpr uint32_t units() const { return blocks ? (blocks - 1) * block_units(whole) + block_units(last) : 0; }  // of a key head
};
// of `rows` query rows (not none) to a key head, in blocks of up to `most`
template <int TILE>
constexpr DealRow deal_row_of(uint32_t rows, uint32_t most, int32_t tiles)
{
    DealRow d = {(rows + most - 1) / most, 0, tiles > 0 ? (uint32_t)tiles : 1u, 0, 0};
    const uint32_t groups = (rows + 31) / 32, each = (groups + d.blocks - 1) / d.blocks;
    d.blocks = (groups + each - 1) / each;  // (the last ones may have come out empty)
    d.rows = 32 * each;
    d.whole = tile_units<TILE>(each);
    d.last = tile_units<TILE>(groups - (d.blocks - 1) * each);
    return d;
}

// What a share that has come to `unit` and ends at `stop` has of the block that `unit` lies in, of a row whose first unit is of_row.
struct DealPiece {
    uint32_t kh, block;
    uint32_t each, first, end;  // units of a tile; first unit of the tiles; the block's end
    int32_t from, to;           // the share's tiles
};
constexpr DealPiece deal_piece(const DealRow& d, uint32_t of_row, uint32_t unit, uint32_t stop)
{
    DealPiece p = {0, 0, 0, 0, 0, 0, 0};
    const uint32_t head_units = d.units(), at = unit - of_row, kh = at / head_units, in_head = at - kh * head_units;
    const uint32_t guess = in_head / d.block_units(d.whole), block = guess < d.blocks - 1 ? guess : d.blocks - 1;
    const uint32_t each = block == d.blocks - 1 ? d.last : d.whole, begin = of_row + kh * head_units + block * d.block_units(d.whole), end = begin + d.block_units(each);
    // a tile is the share's that its first unit lies in, a short block's are all with the first one
    const uint32_t first = begin + DEAL_BLOCK, step = each * d.tiles <= DEAL_SHORT ? each * d.tiles : each;
    const uint32_t from = unit > first ? (unit - first + step - 1) / step : 0, to = stop > first ? (stop - first + step - 1) / step : 0;
    const uint32_t tiles = step == each ? d.tiles : 1;
    const int32_t most = (int32_t)d.tiles;
    p.kh = kh, p.block = block, p.each = each, p.first = first, p.end = end;
    p.from = from < tiles ? (int32_t)from : most, p.to = to < tiles ? (int32_t)to : most;
    return p;
}
// Shares that have some of a block that begins in `share` and goes on (none is behind the last one: see add_units)
constexpr uint32_t deal_shares(const DealPiece& p, uint32_t tiles, uint32_t per, uint32_t share, uint32_t shares)
{
    const uint32_t last = (p.first + p.each * (tiles - 1)) / per;
    return (last < shares ? last : shares - 1) - share + 1;
}

}  // namespace attn
}  // namespace pimdl
