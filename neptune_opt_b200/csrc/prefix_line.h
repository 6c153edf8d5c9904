// The line of work that the stream kernel of attention behind a shared prefix deals out to its workers: plain arithmetic,
// for kernels and host compilers alike.
//
// A unit is a tile of query rows and the keys they share: units of the prefix (a key/value head each, as few query rows as
// one tile holds; none when the prefix runs on the tensor cores), then units of the caches (sequence, key/value head, row
// tile). All units' steps of 16
// keys stand in one line, each unit's behind kEntry places for its own start and end, and every worker takes an equal piece
// of the line, whatever the sequences' lengths are. A piece covers the end of one unit, whole units, the beginning of
// another: worker w's result for unit u goes to slot w + u, which no other pair has, and span[u] says which workers had a
// share in u: the first is the one with the unit's first step, the last the one with its last.
#pragma once

#include <stdint.h>

#include "plain.h"

namespace nb200 {
namespace prefix {

constexpr int kStepKeys = 16;  // keys of a worker's step
constexpr int kEntry = 2;      // what a unit costs beside its steps, in steps

NB200_PLAIN int steps_of(int keys) { return (keys + kStepKeys - 1) / kStepKeys; }
// Places of a unit in the line.
NB200_PLAIN int places_of(int keys) { return keys > 0 ? kEntry + steps_of(keys) : 0; }

struct Line {
    const int* lens;  // tokens of each sequence (null: all of the cache)
    int batch, kv_heads, cache;
    int prefix;     // keys of the prefix's units (0: there are none)
    int own_tiles;  // row tiles of a sequence's query rows

    NB200_PLAIN int tokens(int b) const {
        const int n = lens ? lens[b] : cache;
        return n < 0 ? 0 : n < cache ? n : cache;
    }
    NB200_PLAIN int64_t shared_places() const { return (int64_t)kv_heads * places_of(prefix); }
    NB200_PLAIN int shared_units() const { return prefix ? kv_heads : 0; }
    NB200_PLAIN int64_t units_of_a_sequence() const { return (int64_t)kv_heads * own_tiles; }
};

// A position in the line: a step of a unit, and how many places of the worker's piece are left from there on.
struct Cursor {
    int batch;  // -1: a unit of the prefix
    int head, tile, step, steps, keys;
    int left;   // <= 0: at the end

    NB200_PLAIN void sequence(const Line& a, int b) {
        batch = b, head = 0, tile = 0, keys = a.tokens(b), steps = steps_of(keys);
    }
    // The first place of a piece: place `at` of the prefix's units (b = -1) or of sequence b's.
    NB200_PLAIN void start(const Line& a, int b, int64_t at) {
        if (b < 0) batch = -1, keys = a.prefix, steps = steps_of(keys);
        else sequence(a, b);
        const int tiles = b < 0 ? 1 : a.own_tiles;
        const int places = kEntry + steps, unit = (int)(at / places), place = (int)(at - (int64_t)unit * places) - kEntry;
        head = unit / tiles, tile = unit % tiles;
        step = place > 0 ? place : 0;
        left -= place < 0 ? -place : 0;
    }
    // The first step of the next unit; only while places are left.
    NB200_PLAIN void next_unit(const Line& a) {
        step = 0;
        left -= kEntry;
        if (batch >= 0 && ++tile < a.own_tiles) return;
        tile = 0;
        if (++head < a.kv_heads) return;
        int b = batch;
        do sequence(a, ++b);
        while (steps == 0 && b + 1 < a.batch);
    }
    NB200_PLAIN void next(const Line& a) {
        --left;
        if (++step == steps && left > 0) next_unit(a);
    }
    // Whether the piece holds the unit's last step, and on to the next unit of the piece, if there is one.
    NB200_PLAIN bool ends_unit() const { return left >= steps - step; }
    NB200_PLAIN bool skip_unit(const Line& a) {
        left -= steps - step;
        if (left > 0) next_unit(a);
        return left > 0;
    }
    NB200_PLAIN int unit(const Line& a) const {
        return batch < 0 ? head : a.shared_units() + (batch * a.kv_heads + head) * a.own_tiles + tile;
    }
};

// Whether `first` to `last` can be the workers that had a share in a unit. They name slots, and nothing but what the stream
// kernel left in memory says that they are right.
NB200_PLAIN bool are_workers(int first, int last, int workers) { return 0 <= first && first <= last && last < workers; }

}  // namespace prefix
}  // namespace nb200
