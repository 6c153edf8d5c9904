"""How the logits' kernels cut rows into vectors, on the host: no block of 16 bytes that they load reaches past the row, and
every token is moved exactly once."""
from __future__ import annotations

import ctypes

import pytest

from host_code import compiled

SOURCE = r"""
#include "logits_rows.h"
#include <string.h>
using nb200::RowCut;

// 0: the row is right. Marks the tokens that vectors and single moves write, and holds every block that a vector loads
// against the row's tokens 0 .. vocab.
template <int SIZE>
static int64_t look(uintptr_t x, uintptr_t out, int64_t vocab, int size, unsigned char* moved) {
    const RowCut<SIZE> r(x, out, vocab);
    constexpr int V = RowCut<SIZE>::V;
    memset(moved, 0, vocab);
    const int64_t tiles = (vocab + size - 1) / size;  // as the launch counts them
    for (int64_t t = 0; t < tiles; ++t) {
        const int64_t lo = r.begin(t, size, vocab), hi = r.end(t, size, vocab), body = r.body(t, size, vocab);
        const int n = r.vectors(body, hi, vocab);
        if (lo > body || (hi > body ? hi : body) < lo || hi - lo > size + 2 * V) return 1;
        for (int i = 0; i < n; ++i) {
            const int64_t v = body + (int64_t)i * V;
            if ((out + v * SIZE) % 16 || v + V > hi) return 2;
            if ((x + (v - r.shift) * SIZE) % 16) return 3;
            if (v - r.shift < 0 || v - r.shift + (int64_t)r.blocks() * V > vocab) return 4;  // past the row's memory
            if (r.shift + V > r.blocks() * V) return 5;                                      // too few blocks
            for (int j = 0; j < V; ++j) moved[v + j]++;
        }
        for (int64_t v = lo; v < body && v < hi; ++v) moved[v]++;
        for (int64_t v = body + (int64_t)n * V; v < hi; ++v) moved[v]++;
    }
    for (int64_t v = 0; v < vocab; ++v)
        if (moved[v] != 1) return 6;
    return 0;
}
extern "C" int64_t look2(uintptr_t x, uintptr_t out, int64_t vocab, int size, unsigned char* moved) {
    return look<2>(x, out, vocab, size, moved);
}
extern "C" int64_t look4(uintptr_t x, uintptr_t out, int64_t vocab, int size, unsigned char* moved) {
    return look<4>(x, out, vocab, size, moved);
}
"""


@pytest.fixture(scope="module")
def look(tmp_path_factory):
    lib = compiled(tmp_path_factory.mktemp("rows"), SOURCE)
    room = ctypes.create_string_buffer(1 << 18)
    calls = {}
    for size, f in ((2, lib.look2), (4, lib.look4)):
        f.restype = ctypes.c_int64
        f.argtypes = [ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int64, ctypes.c_int, ctypes.c_char_p]
        calls[size] = lambda x, out, vocab, tile, f=f: f(x, out, vocab, tile, room)
    return calls


@pytest.mark.parametrize("size", [2, 4])
def test_every_place_behind_a_boundary(look, size):
    """Any row of any tensor: input and output behind a 16-byte boundary by any number of elements."""
    base = 1 << 30
    for vocab in [*range(1, 70), 127, 128, 129, 255, 256, 257, 1003, 4095, 4096, 4097, 4111, 8200]:
        for x in range(0, 16, size):
            for out in range(0, 16, size):
                for tile in (64, 4096):
                    assert look[size](base + x, 2 * base + out, vocab, tile) == 0, (vocab, x, out, tile)


@pytest.mark.parametrize("size,rows,wide,at,vocab", [
    (2, 1024, 131072, 1, 131071), (4, 512, 131072, 1, 131071), (2, 9, 32001, 0, 32000), (2, 16, 131072, 0, 131071),
    (2, 9, 1024, 5, 1003), (4, 9, 50009, 3, 50001)])
def test_views_of_wider_buffers(look, size, rows, wide, at, vocab):
    """The rows of base[:, at:at + vocab] of a [rows, wide] buffer; the last ones end where its memory does."""
    for r in range(max(0, rows - 16), rows):
        x, out = (1 << 30) + (r * wide + at) * size, (1 << 31) + r * vocab * size
        assert look[size](x, out, vocab, 8192 if size == 2 else 4096) == 0, r
