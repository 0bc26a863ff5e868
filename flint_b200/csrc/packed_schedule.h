// How a ragged batch's attention is shared out over CTAs (the arithmetic is plain C++: tests/test_packed_schedule.py
// checks it on the CPU).
//
// A tile is 2^log_tokens tokens of one sequence with all query heads of one K/V head; it works on key
// tiles of 128 positions from 0 up to its last token's own. The tiles of all sequences, in the order
// (sequence, K/V head, tile), lie one behind the other on a line, each as long as its key tiles
// and two more for what starting and ending it costs. The line is cut into as many equal parts as
// there are CTAs, so that however long and short the sequences are, CTAs work equally long; a cut
// that falls close to a tile's end moves there. A tile that a cut splits is put together from parts afterwards.
//
// Batches of up to 128 sequences without a tile that is much longer than a CTA's part keep their tiles whole (dealt_rank).
#pragma once

namespace fb {

#if defined(__CUDACC__)
#define FB_SCHEDULE __device__ __forceinline__
#else
#define FB_SCHEDULE inline
#endif

constexpr int kKeyTile = 128;
constexpr int kTileEnds = 2;

// a / b for b > 0, by the short division where it does (the long one takes hundreds of instructions).
FB_SCHEDULE long long quotient(long long a, long long b) {
    if (((a | b) >> 31) == 0) {
        return static_cast<unsigned>(a) / static_cast<unsigned>(b);
    }
    return a / b;
}

// Sum of w >> shift over w = 0 .. z.
FB_SCHEDULE long long floor_sum(long long z, int shift) {
    const long long q = z >> shift;
    const long long rest = z - (q << shift);
    return ((q * (q - 1) / 2) << shift) + q * (rest + 1);
}

// Key tiles of tile i: its last token sees before + (tokens up to it) positions, where `before` is the
// position of the sequence's first new token (negative where tokens have no position). At
// least one, in which such tokens find nothing.
FB_SCHEDULE int key_tiles(int before, int tokens, int log_tokens, int i) {
    const long long end = (static_cast<long long>(i) + 1) << log_tokens;
    const long long visible = before + (end < tokens ? end : tokens);
    return visible <= kKeyTile ? 1 : static_cast<int>((visible + kKeyTile - 1) >> 7);
}

// Length on the line of the tiles 0 .. i - 1 of one head, all of them full: without a loop, since
// 2^log_tokens divides a key tile, so that ceil((b + x 2^t) / 128) = (u + x) >> (7 - t).
FB_SCHEDULE long long tiles_before(int before, int log_tokens, int i) {
    long long none = before < 0 ? (-static_cast<long long>(before)) >> log_tokens : 0;   // see nothing
    none = none < i ? none : i;
    const long long from = before + (none << log_tokens);
    const long long rest = i - none;
    if (rest == 0) {
        return (1 + kTileEnds) * none;
    }
    const long long u = (from + kKeyTile - 1) >> log_tokens;
    const int shift = 7 - log_tokens;
    return (1 + kTileEnds) * none + kTileEnds * rest + floor_sum(u + rest, shift) - floor_sum(u, shift);
}

FB_SCHEDULE int tile_count(int tokens, int log_tokens) {
    return static_cast<int>((static_cast<long long>(tokens) + (1LL << log_tokens) - 1) >> log_tokens);
}

// How many tiles of one head have `least` key tiles or more: they are its last ones.
FB_SCHEDULE int tiles_of_at_least(int before, int tokens, int log_tokens, int least) {
    const int count = tile_count(tokens, log_tokens);
    const int beyond = (least - 1) * kKeyTile - before;      // so many tokens see less
    return least <= 1 || beyond <= 0 ? count : tokens <= beyond ? 0 : count - (beyond >> log_tokens);
}

// Length on the line of one head of a sequence.
FB_SCHEDULE long long head_length(int before, int tokens, int log_tokens) {
    if (tokens == 0) {
        return 0;
    }
    const int last = tile_count(tokens, log_tokens) - 1;
    return tiles_before(before, log_tokens, last) + key_tiles(before, tokens, log_tokens, last) + kTileEnds;
}

// A place on the line. `tile` may be one past a head's last, `offset` is then 0.
struct Cut {
    long long at;
    int sequence, head, tile, offset;
};

// The place `at`, which lies `into` behind the beginning of `sequence`, moved to an end of its tile
// where that is at most `tolerance` away.
FB_SCHEDULE Cut cut_at(long long at, long long into, int sequence, int before, int tokens, int log_tokens,
                       long long length, long long tolerance) {
    Cut c;
    c.sequence = sequence;
    c.head = static_cast<int>(quotient(into, length));
    const long long x = into - c.head * length;
    int low = 0, high = tile_count(tokens, log_tokens) - 1;   // the last tile that begins at or before x
    while (low < high) {
        const int middle = low + (high - low + 1) / 2;
        if (tiles_before(before, log_tokens, middle) <= x) {
            low = middle;
        } else {
            high = middle - 1;
        }
    }
    const long long offset = x - tiles_before(before, log_tokens, low);
    const long long rest = key_tiles(before, tokens, log_tokens, low) + kTileEnds - offset;
    c.at = at;
    c.tile = low;
    c.offset = static_cast<int>(offset);
    if (offset <= rest ? offset <= tolerance : rest <= tolerance) {
        c.at += offset <= rest ? -offset : rest;
        c.tile += offset <= rest ? 0 : 1;
        c.offset = 0;
    }
    return c;
}

// Parts that the line is cut into (up to `most`, none shorter than `least`), the place of cut k, and how
// far a cut may move.
FB_SCHEDULE int part_count(long long total, int most, int least) {
    const long long parts = quotient(total + least - 1, least);
    return parts < most ? static_cast<int>(parts) : most;
}
FB_SCHEDULE long long cut_place(long long total, int parts, int k) {
    const long long each = quotient(total, parts), over = total - each * parts;
    return each * k + quotient(over * k, parts);
}
// About what a split costs (a second start and end, and the join's share), but never so far that two cuts could meet.
FB_SCHEDULE long long cut_tolerance(long long total, int parts) {
    const long long each = quotient(total, parts);
    const long long wanted = each < 24 ? 2 : 3;
    return wanted < (each - 1) / 2 ? wanted : (each - 1) / 2;
}

// Where no tile is much longer than a CTA's part, the tiles stay whole: sorted by their key tiles, longest first, and dealt
// out to the CTAs forwards and backwards in turn. The rank of CTA k's tile in a round.
FB_SCHEDULE long long dealt_rank(int round, int cta, int ctas) {
    return static_cast<long long>(round) * ctas + (round % 2 == 0 ? cta : ctas - 1 - cta);
}

// A sequence's place in the rows (its new tokens) and how many keys it has, those among them.
struct Sequence {
    int first, count, keys;
    FB_SCHEDULE int before() const { return keys - count; }
};

// A stretch of key tiles [from, to) of one tile.
struct Piece {
    Sequence sequence;
    int index;          // of the sequence
    int head;           // K/V head
    int first_token;    // of the tile, in the sequence
    int tokens;         // in the tile
    int from, to, tiles;
    FB_SCHEDULE int position() const { return sequence.before() + first_token; }   // of the first token
};

// The pieces between two cuts, in order; get(s) is sequence s. Every role of a CTA walks on its own.
struct Walk {
    long long at, end;
    int s, head, tile, offset;
    Sequence sequence;

    template <typename Get>
    FB_SCHEDULE void begin(const Get& get, const Cut& first, long long stop) {
        at = first.at;
        end = stop;
        s = first.sequence;
        head = first.head;
        tile = first.tile;
        offset = first.offset;
        if (at < end) {
            sequence = get(s);
        }
    }
    template <typename Get>
    FB_SCHEDULE bool next(const Get& get, int sequences, int kv_heads, int log_tokens, Piece& out) {
        while (at < end) {
            if (tile == tile_count(sequence.count, log_tokens)) {
                tile = 0;
                if (sequence.count == 0 || ++head == kv_heads) {
                    head = 0;
                    if (++s >= sequences) {
                        return false;
                    }
                    sequence = get(s);
                }
                continue;
            }
            const int tiles = key_tiles(sequence.before(), sequence.count, log_tokens, tile);
            const long long rest = tiles + kTileEnds - offset;
            const long long taken = rest < end - at ? rest : end - at;
            const int stop = offset + static_cast<int>(taken);
            out.sequence = sequence;
            out.index = s;
            out.head = head;
            out.first_token = tile << log_tokens;
            const int left = sequence.count - out.first_token;
            out.tokens = left < (1 << log_tokens) ? left : 1 << log_tokens;
            out.from = offset;
            out.to = stop < tiles ? stop : tiles;
            out.tiles = tiles;
            at += taken;
            offset = 0;
            ++tile;
            if (out.from < out.to) {
                return true;
            }
        }
        return false;
    }
};

// What the CTA between two cuts leaves for the join of split tiles.
struct Record {
    int head_part;    // its first tile began earlier: 0 no, 1 it ends here, 2 it goes on
    int tail_part;    // its last tile begins here and goes on
    int first_row;    // of that tile: the row of its first token,
    int tokens;       // how many,
    int kv_head;
    int position;     // of the first one
    int pad[2];
};

template <typename Get>
FB_SCHEDULE Record make_record(const Get& get, int log_tokens, const Cut& lo, const Cut& hi) {
    Record r = {};
    if (lo.at >= hi.at) {
        return r;
    }
    if (lo.offset > 0) {
        const Sequence q = get(lo.sequence);
        const int left = key_tiles(q.before(), q.count, log_tokens, lo.tile) - lo.offset;
        r.head_part = left <= 0 ? 0 : hi.at - lo.at < left ? 2 : 1;
    }
    if (hi.offset > 0 && hi.at - hi.offset >= lo.at) {
        const Sequence q = get(hi.sequence);
        r.tail_part = hi.offset < key_tiles(q.before(), q.count, log_tokens, hi.tile) ? 1 : 0;
        const int first = hi.tile << log_tokens;
        const int left = q.count - first;
        r.first_row = q.first + first;
        r.tokens = left < (1 << log_tokens) ? left : 1 << log_tokens;
        r.kv_head = hi.head;
        r.position = q.before() + first;
    }
    return r;
}

}  // namespace fb
