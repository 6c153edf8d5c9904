"""How attention behind a shared prefix deals its work out, on the host: every step of every unit is taken exactly once, a
unit's span names the workers that took them, and that stays so when a worker gives up anywhere in its piece."""
from __future__ import annotations

import ctypes
import random

import pytest

from host_code import compiled

SOURCE = r"""
#include "prefix_line.h"
#include <map>
#include <utility>
#include <vector>
using namespace nb200::prefix;

struct Span { int x = -7, y = -7; };

// The workers of a call, one behind the other; worker w gives up before its stop[w]th step (< 0: never). 0: all is right.
extern "C" int deal(const int* lens, int batch, int kv_heads, int prefix, int cache, int own_tiles, int workers,
                    const int* stop) {
    Line a;
    a.lens = lens, a.batch = batch, a.kv_heads = kv_heads, a.prefix = prefix, a.cache = cache;
    a.own_tiles = own_tiles;
    const int64_t shared = a.shared_places(), each = a.units_of_a_sequence();
    int64_t all = shared;
    for (int b = 0; b < batch; ++b) all += each * places_of(a.tokens(b));
    const int64_t share = (all + workers - 1) / workers;
    const int units = a.shared_units() + kv_heads * batch * own_tiles;
    std::vector<Span> span(units);
    std::map<std::pair<int, int>, int> slot;             // (worker, unit): steps taken, -1 where it gave up
    std::vector<std::vector<int>> taken(units);
    for (int w = 0; w < workers; ++w) {
        int64_t at = w * share;
        Cursor c;
        c.left = 0;
        if (at >= all) continue;
        c.left = (int)(share < all - at ? share : all - at);
        int b = -1;
        if (at >= shared) {
            at -= shared;
            for (b = 0; at >= each * places_of(a.tokens(b)); ++b) at -= each * places_of(a.tokens(b));
        }
        c.start(a, b, at);
        if (c.left <= 0) continue;
        if (c.step == 0) span[c.unit(a)].x = w;
        int steps = 0;
        for (int run = 0;;) {
            const int u = c.unit(a);
            if (u < 0 || u >= units || c.step >= c.steps) return 1;
            if (steps == stop[w]) {
                for (;;) {
                    const int v = c.unit(a);
                    if (v < 0 || v >= units) return 2;
                    slot[{w, v}] = -1;
                    if (c.ends_unit()) span[v].y = w;
                    if (!c.skip_unit(a)) break;
                    span[c.unit(a)].x = w;
                }
                break;
            }
            ++steps, ++run;
            taken[u].push_back(c.step);
            const bool ends = c.step + 1 == c.steps;
            if (c.left > 1 && !ends) {
                ++c.step, --c.left;
                continue;
            }
            slot[{w, u}] = run;
            run = 0;
            if (ends) span[u].y = w;
            c.next(a);
            if (c.left <= 0) break;
            span[c.unit(a)].x = w;
        }
    }
    for (int u = 0; u < units; ++u) {
        const int keys = u < a.shared_units() ? prefix : a.tokens((u - a.shared_units()) / (int)each);
        if (!keys) {
            if (span[u].x != -7 || span[u].y != -7) return 3;
            continue;
        }
        if (!are_workers(span[u].x, span[u].y, workers)) return 4;
        int steps = 0;
        bool whole = true;
        for (int w = span[u].x; w <= span[u].y; ++w) {
            if (!slot.count({w, u})) return 5;  // a slot that is read was never written
            if (slot[{w, u}] < 0) whole = false;
            else steps += slot[{w, u}];
        }
        if (whole && (steps != steps_of(keys) || (int)taken[u].size() != steps)) return 6;
        for (size_t i = 1; whole && i < taken[u].size(); ++i)
            if (taken[u][i] != taken[u][i - 1] + 1) return 7;
    }
    for (auto& s : slot)
        if (s.first.first < span[s.first.second].x || s.first.first > span[s.first.second].y) return 8;
    return 0;
}
extern "C" int are(int x, int y, int workers) { return are_workers(x, y, workers); }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    return compiled(tmp_path_factory.mktemp("line"), SOURCE)


def _deal(lib, rng, gives_up):
    batch, kv_heads, own_tiles = rng.randint(1, 70), rng.choice([1, 2, 3, 8]), rng.choice([1, 1, 2, 5])
    cache, prefix = rng.choice([0, 1, 16, 17, 300, 2000]), rng.choice([0, 0, 0, 1, 15, 16, 333, 5000])
    lens = [rng.choice([0, 0, 1, cache, cache + 9, -4, rng.randint(0, cache)]) for _ in range(batch)]
    workers = 4 * rng.choice([1, 2, 7, 148, 296, 592])
    stop = [rng.choice([0, 1, 2, 5, 20]) if rng.random() < gives_up else -1 for _ in range(workers)]
    as_ints = lambda v: (ctypes.c_int * len(v))(*v)  # noqa: E731
    with_lens = as_ints(lens) if rng.random() < 0.8 else None
    return lib.deal(with_lens, batch, kv_heads, prefix, cache, own_tiles, workers, as_ints(stop))


@pytest.mark.parametrize("gives_up", [0.0, 0.05, 0.6, 1.0])
def test_every_step_is_taken_once_and_spans_name_the_takers(lib, gives_up):
    rng = random.Random(int(100 * gives_up))
    for i in range(600):
        assert _deal(lib, rng, gives_up) == 0, i


def test_spans_that_name_no_workers(lib):
    assert lib.are(0, 0, 1) and lib.are(3, 9, 10) and lib.are(4, 4, 5)
    low, high = -2 ** 31, 2 ** 31 - 1
    for x, y in ((-1, 0), (0, 10), (5, 4), (10, 10), (low, 3), (3, high), (high, low), (low, high), (0, low)):
        assert not lib.are(x, y, 10), (x, y)
