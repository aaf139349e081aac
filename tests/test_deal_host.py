"""The deal of drafted trees' blocks over shares, without a GPU: the arithmetic that the kernel runs (csrc/attn_deal_units.h), compiled for the host and walked through as the kernel's
workgroups do.  Of batches whose rows have tokens of their own every tile has one owner, and the shares that a join is told are those that left something.  Of starts that fall again, so that
rows share tokens and the units of all reach the end of their sums, every key head, block, tile, slot and share stays in range."""
import subprocess

import pytest

from __graft_entry__ import load_package

pimdl = load_package()

SOURCE = r"""
#include <stdio.h>
#include <stdlib.h>
#include <map>
#include <random>
#include <tuple>
#include <vector>
#include "attn_deal_units.h"
using namespace pimdl::attn;

#define NEED(x) do { if (!(x)) { printf("line %d: %s (case %d, share %u)\n", __LINE__, #x, number, share); exit(1); } } while (0)

struct Batch { std::vector<uint32_t> rows, keys; };  // of each row of the batch: query rows to a key head, keys there are

// ordinary: rows have tokens of their own
template <int TILE>
void walk(int number, const Batch& in, uint32_t kv_heads, uint32_t most_rows, uint32_t shares, bool ordinary, uint64_t* pieces, uint32_t* top)
{
    const uint32_t batch = (uint32_t)in.rows.size();
    std::vector<DealRow> row(batch);
    std::vector<uint32_t> unit(batch + 1);
    uint32_t share = 0, sum = 0;
    for (uint32_t b = 0; b < batch; ++b) {
        const uint32_t tiles = (in.keys[b] + TILE - 1) / TILE;
        row[b] = in.rows[b] ? deal_row_of<TILE>(in.rows[b], most_rows, (int32_t)tiles) : DealRow{0, most_rows, 1, 1, 1};
        if (in.rows[b]) {  // blocks cover the rows, none is empty, none too large
            NEED(row[b].blocks >= 1 && row[b].rows <= most_rows && row[b].rows % 32 == 0);
            NEED((uint64_t)(row[b].blocks - 1) * row[b].rows < in.rows[b] && (uint64_t)row[b].blocks * row[b].rows >= in.rows[b]);
            NEED(row[b].whole <= TILE_MOST * (row[b].rows / 32) && row[b].last <= row[b].whole);
        }
        const uint64_t mine = (uint64_t)row[b].units() * kv_heads;
        NEED(mine < 1ull << 31);
        unit[b] = sum;
        sum = add_units(sum, (uint32_t)mine);
    }
    unit[batch] = sum;
    *top = sum;
    const uint32_t per = share_of(sum, shares);
    NEED((uint64_t)per * shares >= sum);
    std::map<std::tuple<uint32_t, uint32_t, uint32_t>, int32_t> done;       // (row, key head, block) -> tiles so far
    std::map<std::tuple<uint32_t, uint32_t, uint32_t>, uint32_t> told, had; // ... -> shares that its first one told, that had some
    for (share = 0; share < shares; ++share) {
        if ((uint64_t)share * per > 0xffffffffu) { NEED(false); }
        uint32_t at = share * per;
        const uint32_t stop = at + per < sum ? at + per : sum;
        if (at >= stop) continue;
        uint32_t b = 0, begun = 0, ended = 0;
        for (uint32_t up = batch; up - b > 1;) {
            const uint32_t mid = (b + up) / 2;
            if (unit[mid] <= at) b = mid;
            else up = mid;
        }
        while (at < stop) {
            while (unit[b + 1] <= at) { ++b; NEED(b < batch); }
            NEED(unit[b] <= at && row[b].blocks);
            const DealPiece p = deal_piece(row[b], unit[b], at, stop);
            ++*pieces;
            NEED(p.kh < kv_heads && p.block < row[b].blocks);
            NEED(p.from >= 0 && p.from <= (int32_t)row[b].tiles && p.to >= 0 && p.to <= (int32_t)row[b].tiles);
            NEED(p.end > at);  // it goes on
            at = p.end < stop ? p.end : stop;
            if (p.from >= p.to) continue;
            const auto key = std::make_tuple(b, p.kh, p.block);
            const bool whole = p.from == 0 && p.to == (int32_t)row[b].tiles;
            if (ordinary) NEED(done[key] == p.from);
            done[key] = p.to;
            ++had[key];
            if (!whole && p.from == 0) {  // slot 2 share + 1, and the join's list
                NEED(++begun == 1);
                const uint32_t count = deal_shares(p, row[b].tiles, per, share, shares);
                NEED(count >= 1 && count <= shares && share + count <= shares);
                if (ordinary) NEED(count >= 2);
                told[key] = count;
            } else if (!whole) {  // slot 2 share
                NEED(++ended == 1);
            }
        }
    }
    share = 0;
    if (!ordinary) return;
    for (uint32_t b = 0; b < batch; ++b)
        for (uint32_t kh = 0; kh < kv_heads; ++kh)
            for (uint32_t block = 0; block < row[b].blocks; ++block) {
                const auto key = std::make_tuple(b, kh, block);
                NEED(done.count(key) && done[key] == (int32_t)row[b].tiles);
                NEED((told.count(key) ? told[key] : 1) == had[key]);
            }
}

int main()
{
    std::mt19937_64 rng(7);
    auto below = [&](uint64_t n) { return (uint32_t)(rng() % n); };
    auto spread = [&](uint32_t n) { return below(1ull << below(n + 1)); };  // even over the logarithm
    uint64_t pieces = 0;
    uint32_t top = 0, share = 0;
    int number = 0;
    for (; number < 1500; ++number) {
        const uint32_t batch = 1 + (number % 10 ? spread(5) : below(DEAL_BATCH)), kv = 1 + spread(3), shares = number % 7 ? 256 : 1 + below(304), most = number % 2 ? 256 : 128;
        Batch in;
        uint64_t rows = 0, keys = 0;
        for (uint32_t b = 0; b < batch; ++b) {
            in.rows.push_back(below(9) ? spread(11) : 0);
            in.keys.push_back(below(9) ? spread(17) : 0);
            rows += in.rows.back();
            keys = std::max<uint64_t>(keys, in.keys.back());
        }
        if (deal_most_units(rows, batch, kv, keys, 32) >= 1ull << 31) continue;
        walk<64>(number, in, kv, most, shares, true, &pieces, &top);
        NEED(top <= deal_most_units(rows, batch, kv, keys, 64));
        walk<32>(number, in, kv, most, shares, true, &pieces, &top);
        NEED(top <= deal_most_units(rows, batch, kv, keys, 32));
    }
    // starts that fall again: every second row has all tokens (those between have none), or all that are left from some start
    uint32_t reached = 0;
    for (; number < 2100; ++number) {
        const uint32_t batch = 2 + below(DEAL_BATCH - 1), kv = 1 + spread(3), shares = number % 7 ? 256 : 1 + below(304), most = number % 2 ? 256 : 128;
        const uint32_t all = 32 + spread(16);
        uint32_t keys = 1 + spread(10);  // ... and as many as there can be, so that a few rows' units are all that there are
        while (keys < 1u << 30 && deal_most_units(all, batch, kv, 2 * keys, 32) < 1ull << 31) keys *= 2;
        if (deal_most_units(all, batch, kv, keys, 32) >= 1ull << 31) continue;
        Batch in;
        for (uint32_t b = 0; b < batch; ++b) {
            in.rows.push_back(number % 3 ? (b % 2 ? 0 : all) : below(all + 1));
            in.keys.push_back(number % 5 ? keys : below(keys + 1));
        }
        walk<64>(number, in, kv, most, shares, false, &pieces, &top);
        reached += top == 0x7fffffffu;
        walk<32>(number, in, kv, most, shares, false, &pieces, &top);
        reached += top == 0x7fffffffu;
    }
    NEED(reached > 50 && pieces > 100000);
    NEED(add_units(0x7fffffffu, 0x7fffffffu) == 0x7fffffffu && add_units(1, 2) == 3);
    printf("fine: %llu pieces, %u ended at the most\n", (unsigned long long)pieces, reached);
    return 0;
}
"""


@pytest.fixture(scope="module")
def walker(tmp_path_factory):
    d = tmp_path_factory.mktemp("deal")
    (d / "walk.cpp").write_text(SOURCE)

    def run(include):
        subprocess.check_call(["g++", "-std=c++17", "-O2", "-Wall", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", str(include), "-o", str(d / "walk"), str(d / "walk.cpp")])
        return subprocess.run([str(d / "walk")], capture_output=True, text=True, timeout=120)

    return run


def test_the_deal_gives_every_tile_one_owner_and_stays_in_range(walker):
    r = walker(pimdl.CSRC)
    assert r.returncode == 0 and r.stdout.startswith("fine"), r.stdout + r.stderr


@pytest.mark.parametrize("guard,without", [("return sum < 0x7fffffffu ? sum : 0x7fffffffu;", "return sum;"), ("(last < shares ? last : shares - 1)", "last")])
def test_the_walk_misses_each_guard(walker, tmp_path, guard, without):
    """What the walk would say of a deal without one of them (on the host)."""
    with open(f"{pimdl.CSRC}/attn_deal_units.h") as f:
        text = f.read()
    assert text.count(guard) == 1
    (tmp_path / "attn_deal_units.h").write_text(text.replace(guard, without))
    assert walker(tmp_path).returncode != 0
