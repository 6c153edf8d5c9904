// How a row of logits is cut into tiles and 16-byte vectors: plain arithmetic, for kernels and host compilers alike.
#pragma once

#include <stdint.h>

#include "plain.h"

namespace nb200 {

// A row of elements of SIZE bytes. Vectors of V tokens start on the output's 16-byte boundaries; the input of each lies
// `shift` tokens behind one, in one block of 16 bytes (shift 0) or two neighbouring ones, all of which lie in the row.
template <int SIZE>
struct RowCut {
    static constexpr int V = 16 / SIZE;
    int head;   // tokens before the first whole vector of the output; tile 0 holds those, too
    int shift;
    NB200_PLAIN RowCut(uintptr_t x, uintptr_t out, int64_t vocab) {
        const int first = (V - (int)((uint32_t)out & 15u) / SIZE) % V;
        shift = ((int)((uint32_t)x & 15u) / SIZE + first) % V;
        const int before = first < shift ? first + V : first;
        head = before < vocab ? before : (int)vocab;
    }
    // Where tile t of `size` tokens begins (tile 0: with the row) and ends, and where its vectors begin.
    NB200_PLAIN int64_t begin(int64_t t, int size, int64_t vocab) const { return t ? end(t - 1, size, vocab) : 0; }
    NB200_PLAIN int64_t end(int64_t t, int size, int64_t vocab) const {
        const int64_t e = head + (t + 1) * size;
        return e < vocab ? e : vocab;
    }
    NB200_PLAIN int64_t body(int64_t t, int size, int64_t vocab) const { return t ? end(t - 1, size, vocab) : head; }
    // 16-byte blocks of a vector's input, the first one from token v - shift on.
    NB200_PLAIN int blocks() const { return shift ? 2 : 1; }
    // Whole vectors from token `from` to `to` whose blocks end in the row.
    NB200_PLAIN int vectors(int64_t from, int64_t to, int64_t vocab) const {
        const int64_t last = shift ? vocab - (V - shift) : vocab;
        if (to > last) to = last;
        return to > from ? (int)((to - from) / V) : 0;
    }
};

}  // namespace nb200
