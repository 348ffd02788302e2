// Which work each workgroup of the differential-attention kernels takes.  Plain arithmetic that includes nothing, so that a host program
// can include it too (with its own MEP_DEV) and check that everything is taken once.
#pragma once

namespace mep {

// The (batch row, key head) pair and the block of rows or keys of workgroup x of bgs * blocks.
// Workgroups go round the 8 XCDs by their index; where the pairs divide evenly over them, a pair's blocks
// stay on one XCD (or on a few, in turn), so that its keys are read into one L2.
// Causal calls: the blocks differ by up to their number in length, and all pairs' longest come first.  Where two workgroups share a
// compute unit (`shared`) and both halves of the first 512 are there from the start, the second half goes the other way, so that
// the longest shares its unit with the shortest (B 2, T 4096, 8 heads, 64 / 128, bf16: forward 199 us, 207 without that turn, 230 pair by
// pair).
enum Order { IN_TURN, FIRST_LONGEST, LAST_LONGEST };
struct Place { int bg, block; };
MEP_DEV Place place_of(int x, int bgs, int blocks, Order order, bool shared) {
    Place p;
    // position s of n on one XCD of 8, or in all; the 32 / 256 units' second ones the other way
    auto turn = [&](int s, int n, int units) {
        const int last = (n < 2 * units ? n : 2 * units) - 1;
        return shared && s >= units && s <= last ? units + last - s : s;
    };
    if (bgs % 8 == 0) {
        const int q = bgs / 8;
        p.bg = x & 7;
        if (order == IN_TURN) {
            const int s = x >> 3, pair = s / blocks;
            p.bg += pair * 8;
            p.block = s - pair * blocks;
        } else {
            const int s = turn(x >> 3, blocks * q, 32);
            p.block = s / q;
            p.bg += (s - p.block * q) * 8;
        }
    } else if (8 % bgs == 0 && blocks % (8 / bgs) == 0) {
        const int per = 8 / bgs, s = order == IN_TURN ? x >> 3 : turn(x >> 3, blocks / per, 32);
        p.bg = (x & 7) / per;
        p.block = s * per + (x & 7) % per;
    } else if (order == IN_TURN) {
        p.bg = x / blocks;
        p.block = x - p.bg * blocks;
    } else {
        const int s = turn(x, blocks * bgs, 256);
        p.block = s / bgs;
        p.bg = s - p.block * bgs;
    }
    if (order == LAST_LONGEST) p.block = blocks - 1 - p.block;
    return p;
}

// k_diff_split: the tiles of keys of all (batch row, key head, 32 rows) stand in one row, and each of `groups` workgroups takes an equal
// share of it.  A batch row with keys has its tiles, and DA_SPLIT_START more to begin with, `per` times (once a (key head, 32 rows), an item).
constexpr int DA_SPLIT_START = 3;
struct Shares { long tiles, share; };      // in all; a workgroup's
MEP_DEV Shares shares_of(long before_end, int per, int groups) {
    Shares s;
    s.tiles = before_end * per;
    s.share = (s.tiles + groups - 1) / groups;
    s.share = s.share < 4 ? 4 : s.share;      // 4 tiles at least: a part costs as much as one
    return s;
}
// what a workgroup that stands at tile `in` of a batch row's n per, with `left` tiles of its share to go, takes next: keys of the
// tiles tile0 .. tile1 - 1 of an item (none where tile0 >= tile1), `taken` of the share
struct Piece { int item, tile0, tile1, taken; };
MEP_DEV Piece piece_at(long in, long left, int n) {
    Piece p;
    p.item = (int)(in / n);
    const int from = (int)(in - (long)p.item * n), to = (int)(from + left < n ? from + left : n);
    p.tile0 = from > DA_SPLIT_START ? from - DA_SPLIT_START : 0;
    p.tile1 = to - DA_SPLIT_START;
    p.taken = to - from;
    return p;
}
// A part is left by each of a workgroup's two waves for every item it comes to: workgroup w's of batch row b's item stand at twice this.
// (The workgroups' shares follow each other, and so do the items: two neighbours meet in one item at most.)
MEP_DEV long part_at(long w, int b, int per, int item) { return w + (long)b * per + item; }
// the workgroups that come to an item whose n tiles begin at `tile` of all: first .. first + count - 1
struct Meet { long first; int count; };
MEP_DEV Meet meet_of(long tile, int n, long share) {
    Meet m;
    m.first = (tile + DA_SPLIT_START) / share;      // (before the first key a workgroup leaves nothing)
    m.count = n ? (int)((tile + n - 1) / share - m.first + 1) : 0;
    return m;
}

// k_diff_bwd_kv: the tiles of rows from all0 (a tile's first) to all1 over the splits
struct Range { int begin, end; };
MEP_DEV Range split_rows(int all0, int all1, int tile, int split, int splits) {
    const int share = ((all1 - all0 + tile - 1) / tile + splits - 1) / splits * tile;
    Range r;
    r.begin = all0 + split * share;
    r.end = all1 < r.begin + share ? all1 : r.begin + share;
    return r;
}

}  // namespace mep
