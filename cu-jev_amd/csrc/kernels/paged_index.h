/* Where the paged operators read and write: how a sequence's lengths are cut,
 * which pages a tile of rows visits, how the visits are shared out. No HIP in
 * here: the kernels and the launchers use these functions, and a host program
 * can check every index against the buffers. */
#ifndef CUJEV_PAGED_INDEX_H
#define CUJEV_PAGED_INDEX_H

#include <stddef.h>

constexpr int PG = 64;   /* tokens a page, keys a tile */
constexpr int VTOK = 16; /* positions of a V group of the prep */

constexpr int pg_min(int a, int b) { return a < b ? a : b; }
constexpr int pg_max(int a, int b) { return a > b ? a : b; }
constexpr int pg_div_up(int a, int b) { return a / b + (a % b != 0); } /* a >= 0, b > 0 */

/* Sequence b as one call sees it: rows q0 .. q0 + ql - 1, the first at position
 * p0 (negative where it has fewer keys than rows: those rows have no slot), keys
 * 0 .. kv - 1, where rows past max_q bring none. Lengths outside the call's N rows,
 * max_q and max_kv are cut, so no value in q_start or kv_len leads out of a buffer.
 * N and B are at most PG_MOST, max_kv PG_MOST_KEYS: sums and differences of two
 * fit an int, and the key tiles of fewer than 512 units 32 bits. */
constexpr int PG_MOST = 1 << 30, PG_MOST_KEYS = 1 << 28;
struct pg_seq {
    int q0, ql, kv, p0;
};
constexpr pg_seq pg_clean_seq(int q0, int q1, int kv, int N, int max_q, int max_kv) {
    pg_seq s{};
    s.q0 = pg_min(pg_max(q0, 0), N);
    const int ql = pg_min(pg_max(q1, s.q0), N) - s.q0;
    s.p0 = pg_max(kv, 0) - ql;
    s.ql = pg_min(ql, max_q);
    s.kv = pg_min(pg_max(s.p0 + s.ql, 0), max_kv);
    return s;
}

/* The positions [lo, hi) of the new tokens that have a slot */
constexpr int pg_new_lo(const pg_seq &s) { return pg_max(s.p0, 0); }
constexpr int pg_new_hi(const pg_seq &s) { return pg_min(s.p0 + s.ql, s.kv); }
/* Pages that the new tokens touch; a call has at most min(N, N / PG + 2 B) of them. */
constexpr int pg_v_pages(const pg_seq &s) {
    const int lo = pg_new_lo(s), hi = pg_new_hi(s);
    return hi > lo ? (hi - 1) / PG - lo / PG + 1 : 0;
}

/* Key tiles that the new tokens i0 .. i1 of a sequence visit, in order: the
 * sinks' first (nsk of them, tiles 0 .. nsk - 1), then from tile t0 on. */
struct pg_tiles {
    int nsk, t0, ntl;
};
constexpr pg_tiles pg_tile_list(const pg_seq &s, int i0, int i1, int window, int sinks) {
    pg_tiles t{};
    const int hi = pg_min(s.p0 + i1, s.kv - 1); /* last key of the last row */
    if (hi < 0)
        return t;
    const int lo = window > 0 ? pg_max(s.p0 + i0 - window + 1, 0) : 0; /* first of the first */
    t.t0 = pg_min(lo, hi) / PG;
    t.nsk = pg_min(pg_div_up(pg_min(sinks, hi + 1), PG), t.t0);
    t.ntl = t.nsk + hi / PG - t.t0 + 1;
    return t;
}
/* the page-table column of entry i of the list */
constexpr int pg_tile_page(const pg_tiles &t, int i) { return i < t.nsk ? i : i - t.nsk + t.t0; }

/* Most entries a list of a tile of `tok` tokens can have */
constexpr int pg_max_tiles(int tok, int max_kv, int window, int sinks) {
    const int all = pg_div_up(max_kv, PG);
    if (window <= 0 || window > max_kv || tok > max_kv)
        return all;
    return pg_min(all, (window + tok) / PG + 2 + pg_div_up(pg_min(sinks, max_kv), PG));
}

/* ---- how the attention's work is shared out ----------------------------------
 * A unit is a tile of rt packed rows (token, q-head of the group) of a sequence and
 * kv-head. rt is PG_FEW where no sequence of the call has more rows than that (one
 * unit each; 16 are the columns of its MFMA), PG_MANY otherwise: 64 sequences' 16 rows
 * on 2560 e4m3 keys take 78 us as the former, 103 as the latter. It is one for the
 * call: single tokens beside a prompt are tiles of PG_MANY, too (64 on up to 4096 e4m3
 * keys and a prompt of 512 127 us; 68 and 25 in two calls, one for each kind).
 *
 * PG_FEW: the units' key tiles, one after the other, are a line that pieces of equal
 * size cut, a wave's work each; what lies in one piece of one unit is a part.
 * PG_MANY: a unit's key tiles are cut into as many even shares as the plan asks
 * for, a workgroup each. Parts of a unit of several leave theirs in slots. */
constexpr int PG_FEW = 16, PG_MANY = 128;

struct pg_plan {
    int rt;
    int units;  /* units of a kv-head, at most */
    int shares; /* pieces (PG_FEW) or parts of a kv-head's units, at most (0: no
                 * work, -1: too many) */
    int slots;  /* of parts with something to merge, at most (0: no merge) */
    int goal;   /* waves (PG_FEW) or workgroups of a kv-head that the chip runs at
                 * once; 0 (PG_MANY): whole units fill it */
};

constexpr int pg_units(const pg_seq &s, int G, int rt) {
    return (int)(((long long)s.ql * G + rt - 1) / rt);
}
/* Key tiles of a sequence's longest unit, 1 at least: the last one's (with a window
 * a full one before it may have a tile or two more) */
constexpr int pg_longest(const pg_seq &s, int G, int rt, int window, int sinks) {
    if (s.ql <= 0)
        return 0;
    const int units = pg_units(s, G, rt);
    const pg_tiles t =
        pg_tile_list(s, (int)((long long)(units - 1) * rt / G), s.ql - 1, window, sinks);
    return pg_max(t.ntl, 1);
}
/* PG_FEW: tiles a piece of a line of U units with T tiles. Pieces of one tile instead
 * of two gain nothing where there are many, since a wave's first loads take longer
 * than a tile (16 sequences of 1024 e4m3 keys 17.4 us with one, 15.4 with two); but
 * a short line has waves enough for its tiles (530 bf16 keys 9.9 and 12.2), and
 * units of a tile each stay apart (256 of 64 keys 16 and 21). */
constexpr int PG_FEW_SHORT = 16;
constexpr int pg_few_share(const pg_plan &p, int U, unsigned T) {
    const unsigned n = (unsigned)p.goal;
    return pg_max((int)(T / n + (T % n != 0)), T > PG_FEW_SHORT && T / 2 >= (unsigned)U ? 2 : 1);
}
/* PG_FEW: the slot of part j of a unit that begins in piece p0 and goes on after it.
 * A piece has at most two such parts: of a unit that came in from the piece before,
 * and of one that begins here and goes on. */
constexpr int pg_few_slot(int p0, int j) { return 2 * (p0 + j) + (j == 0); }

/* PG_MANY: key tiles a share has at most, of U units with T tiles in all and
 * `longest` the most that one has: about the least for which the parts do not
 * outnumber the workgroups that run at once. Try pg_share_first, then pg_share_next
 * of it until they fit; `sure` fits without trying. Where a share is then not
 * shorter by what a merge takes, some 6 tiles (10 us), all stay whole: 8 sequences'
 * 200 tokens on up to 1500 keys take 57 us so, 67 in 71 parts for 64 workgroups, and
 * 32 x 8 on 1000 35 in shares of 8 tiles, 39 whole (16).
 * Shares have 8 tiles at least: 2 x 64 tokens on 2048 keys take 27 us, 37 with 16;
 * with 4 it is 25, and no less where there is more to do. */
constexpr int PG_MANY_LEAST = 8, PG_MANY_MERGE = 6;
constexpr bool pg_splits(const pg_plan &p, int U) { return p.goal > 0 && U < p.goal; }
constexpr int pg_share_first(const pg_plan &p, int U, unsigned T, bool sure) {
    /* a unit's last share is half full on average */
    const unsigned n = (unsigned)(p.goal - (sure ? U : U / 2));
    return pg_max((int)(T / n + (T % n != 0)), PG_MANY_LEAST);
}
constexpr int pg_share_next(int share) { return share + pg_max(share / 16, 1); }
constexpr int pg_share_last(int share, int longest) {
    return share + PG_MANY_MERGE >= longest ? PG_MOST : share;
}
constexpr int pg_nshare(int tiles, int share) { return pg_max(pg_div_up(tiles, share), 1); }
/* PG_MANY: a sequence's first units, those with no more tiles than a share, stay whole;
 * the others are pg_nshare(longest, share) parts each: a new sequence's first rows
 * have few, and leave workgroups to its last ones (1500 e4m3 keys 57 -> 50 us). */
constexpr int pg_short_units(const pg_seq &s, int G, int window, int longest, int share) {
    const int units = pg_units(s, G, PG_MANY);
    if (longest <= share)
        return units;
    if (window > 0 || share >= PG_MOST / PG)
        return 0;
    const int rows = pg_min(PG * share - s.p0, s.ql); /* that see no more */
    return rows <= 0 ? 0 : (int)pg_min((int)((long long)rows * G / PG_MANY), units);
}
constexpr int pg_parts(const pg_seq &s, int G, int window, int longest, int share) {
    const int units = pg_units(s, G, PG_MANY);
    const int whole = pg_short_units(s, G, window, longest, share);
    return whole + (units - whole) * pg_nshare(longest, share);
}
/* about the tiles that its units have in all */
constexpr unsigned pg_all_tiles(const pg_seq &s, int G, int window, int longest) {
    const int units = pg_units(s, G, PG_MANY);
    /* last key of the first unit */
    const int last = pg_min(pg_min(s.p0, s.kv) + (PG_MANY - 1) / G, s.kv - 1);
    const int first = window > 0 ? longest : pg_min(pg_max(last, 0) / PG + 1, longest);
    return (unsigned)units * (unsigned)(first + longest + 1) / 2;
}
/* First list entry of share i of n even ones */
constexpr int pg_share_begin(int ntl, int i, int n) { return (int)((long long)ntl * i / n); }

/* PG_FEW: waves of a kv-head. A wave a SIMD: 64 sequences of 1024 bf16 keys take 53 us
 * so, 61 with two a SIMD, and half as many as SIMDs leave 24 of 5000 at 58 instead of
 * 52. Few units: no more parts each than a merge takes in one go, 64 (one of 65536
 * keys 42 us; 43 with 128 parts, 60 with 32). */
constexpr int pg_few_goal(long long units, int Hkv) {
    const int chip = pg_max(1024 / Hkv, 1);
    return 64 * units < chip ? (int)(64 * units) : chip;
}
/* and pieces, at most, of a line of `units` units of up to `most` tiles: pieces of two
 * tiles, or of one if there are no more than this of them */
constexpr int pg_few_pieces(long long units, long long most, int goal) {
    const long long line = units * most, two = (line + 1) / 2;
    const long long one = units > PG_FEW_SHORT / 2 ? 2 * units : PG_FEW_SHORT;
    const long long n = two > one ? two : line < one ? line : one;
    return n < goal ? (int)n : goal;
}
constexpr int pg_many_goal(int Hkv) { return pg_max(256 / Hkv, 1); }
/* Lists this long may be split among workgroups */
constexpr bool pg_many_long(long long most) { return most > PG_MANY_LEAST + PG_MANY_MERGE; }
/* Work-items that a launch may have, and units (and shares) times kv-heads of a call */
constexpr long long PG_MOST_ITEMS = 0xffffffffll;
constexpr int PG_MOST_UNITS = 1 << 22;
/* The merge: a workgroup a row of few rows after many keys, or a wave; 16 of many rows.
 * Workgroups of a unit (few rows) or slot and kv-head. */
constexpr bool pg_merge_by_row(const pg_plan &p, int rows, int Hkv) {
    return p.rt == PG_FEW && (long long)p.units * rows * Hkv <= 512;
}
constexpr int pg_merge_groups(const pg_plan &p, int rows, int Hkv) {
    if (p.rt != PG_FEW)
        return PG_MANY / 16;
    return pg_merge_by_row(p, rows, Hkv) ? rows : pg_div_up(rows, 4);
}
constexpr long long pg_merge_items(const pg_plan &p, int rows, int Hkv) {
    return 256ll * (p.rt == PG_FEW ? p.units : p.slots) * Hkv * pg_merge_groups(p, rows, Hkv);
}

constexpr pg_plan pg_make_plan(int N, int B, int max_q, int max_kv, int G, int Hkv, int window,
                               int sinks) {
    pg_plan p{};
    const long long mq = pg_min(max_q, N);
    p.rt = mq * G <= PG_FEW ? PG_FEW : PG_MANY;
    if (mq <= 0 || B <= 0)
        return p;
    if (window >= max_kv)
        window = sinks = 0;
    const int tok = p.rt == PG_FEW ? (int)mq : PG_MANY / G + 2;
    const long long most = pg_max(pg_max_tiles(tok, max_kv, window, sinks), 1);
    long long units = B, shares = 0, slots = 0;
    if (p.rt == PG_FEW) {
        p.goal = pg_few_goal(units, Hkv);
        shares = units * most > 0x7fffffff ? PG_MOST : pg_few_pieces(units, most, p.goal);
        slots = most > 1 ? 2 * shares : 0;
    } else {
        const long long by_rows = (long long)N * G / PG_MANY + B;
        const long long by_len = B * ((mq * G + PG_MANY - 1) / PG_MANY);
        units = by_rows < by_len ? by_rows : by_len;
        /* the rows that the caller brings fill the chip: whole units */
        p.goal = pg_many_goal(Hkv);
        if ((long long)N * G / PG_MANY >= p.goal)
            p.goal = 0;
        const bool split = p.goal > 0 && pg_many_long(most);
        if (!split)
            p.goal = 0;
        shares = units > p.goal ? units : p.goal;
        slots = split ? p.goal : 0;
    }
    if (units * Hkv > PG_MOST_UNITS || shares * Hkv > PG_MOST_UNITS) {
        p.shares = -1;
        return p;
    }
    p.units = (int)units;
    p.shares = (int)shares;
    p.slots = (int)slots;
    if (slots > 0 && pg_merge_items(p, (int)mq * G, Hkv) > PG_MOST_ITEMS)
        p.shares = -1;
    return p;
}

/* ---- workspace -------------------------------------------------------------------
 * o (256), l and mu of the slots' rows as floats, then info: {int, int} a unit, or 4
 * ints a slot. */
constexpr size_t pg_slot_bytes(int slots, int rt, int Hkv, int infos, int info_bytes) {
    return slots <= 0 ? 0
                      : (size_t)slots * Hkv * rt * (256 + 2) * 4 + (size_t)infos * info_bytes;
}
constexpr size_t pg_ws_bytes(const pg_plan &p, int Hkv) {
    return p.rt == PG_FEW ? pg_slot_bytes(p.slots, p.rt, Hkv, p.units, 8)
                          : pg_slot_bytes(p.slots, p.rt, Hkv, p.slots, 16);
}
/* The most that a call of these heads can need whose N, B, max_q and max_kv are these or
 * less, whatever its window: a prompt's rows fill the chip and leave nothing to merge,
 * and the steps after it, smaller calls, do. Slots rise with B and max_kv up to what
 * the chip runs at once, so that it is about 34 MB at the very most. */
constexpr size_t pg_ws_most(int N, int B, int max_q, int max_kv, int G, int Hkv) {
    const long long mq = pg_min(max_q, N);
    if (mq <= 0 || B <= 0)
        return 0;
    const int most = pg_div_up(pg_max(max_kv, 0), PG);
    const int units = pg_min(B, PG_MOST_UNITS / Hkv);
    const int pieces = pg_few_pieces(units, most, pg_few_goal(units, Hkv));
    const size_t few = pg_slot_bytes(most > 1 ? 2 * pieces : 0, PG_FEW, Hkv, units, 8);
    const int goal = mq * G > PG_FEW && pg_many_long(most) ? pg_many_goal(Hkv) : 0;
    const size_t many = pg_slot_bytes(goal, PG_MANY, Hkv, goal, 16);
    return few > many ? few : many;
}

/* The row at position p sees the keys j <= min(p, kv - 1) with j > pg_low or j <
 * sinks; a key is some row's from pmin on where it is before kv and past
 * pg_low(pmin) or a sink. -1 where the window reaches key 0, so that no position
 * from -PG_MOST on and no window leaves an int. */
constexpr int pg_low(int p, int window) {
    return window > 0 ? pg_max(pg_max(p, -1) - window, -1) : -1;
}
/* Whether every row at positions pmin .. pmax sees all PG keys from k0 on */
constexpr bool pg_tile_whole(int k0, int pmin, int pmax, int kv, int window, int sinks) {
    return k0 + PG - 1 <= pg_min(pmin, kv - 1) &&
           (k0 > pg_low(pmax, window) || k0 + PG <= sinks);
}
/* Whether keys of the tile are no key of the call (behind the last one, or
 * before every window and no sink): whatever is there may not reach a product. */
constexpr bool pg_tile_foreign(int k0, int pmin, int kv, int window, int sinks) {
    return k0 + PG > kv || (k0 <= pg_low(pmin, window) && k0 + PG > sinks);
}

#endif
