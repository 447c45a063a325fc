// How a launch whose work is `tiles` live tiles of `rt` units each goes to at most `grid` workgroups, in equal shares of a fixed
// order: the end of one tile, whole ones, the start of another.  Plain C++ (constexpr functions run on both sides): the
// kernel that works on the shares, the one that joins them and the host agree by calling the same functions.
#pragma once

struct Share {                 // one piece of a workgroup's share: units [t0, t1) of tile `tile`
    long long tile;
    int t0, t1;
};

struct Shares {
    long long units;           // in all
    int rt, nb;                // units a tile, workgroups that share them
    // workgroup i's units are [begin(i), begin(i + 1))
    constexpr long long begin(int i) const { return units * i / nb; }
    // the workgroup that holds unit x
    constexpr int owner(long long x) const { return (int)(((x + 1) * nb + units - 1) / units) - 1; }
    // the piece that starts at unit u of a share that ends at u1
    constexpr Share piece(long long u, long long u1) const {
        const long long tile = u / rt;
        const int t0 = (int)(u - tile * rt);
        return Share{tile, t0, (int)(t0 + (u1 - u) < rt ? t0 + (u1 - u) : rt)};
    }
    // a share may leave two partial tiles, its first piece and its last: where piece `part` (0, 1, ..) of workgroup i's goes
    constexpr static long long slot(int i, int part) { return 2ll * i + (part > 0); }
    // which piece of its first workgroup, i = owner(x0), the tile from unit x0 on is; it is the first piece of every later one
    constexpr int part_of(int i, long long x0) const { return begin(i) < x0 ? 1 : 0; }
};

// With three or more workgroups a tile the shares end at tile borders.  A tile never has more workgroups than units: the launch
// may be sized for far more tiles than are live, and a share without a unit would leave a slot that the join adds unwritten.
constexpr Shares shares_of(long long tiles, int grid, int rt) {
    const long long per = tiles > 0 ? grid / tiles : 0;      // workgroups a tile
    return Shares{tiles * rt, rt, per >= 3 ? (int)((per < rt ? per : rt) * tiles) : grid};
}
