// What the kernels of attention over a cache in 8 bits take.
#pragma once

#include "cache8.h"

// The C entry points' arguments (ops/cache8.py fills it; the same fields in the same order).
struct PulseAttn8 {
    const void* q;               // [tokens, >= nq * d], rows q_stride elements apart
    int64_t q_stride;
    void* out;                   // [tokens, >= nq * d]
    int64_t o_stride;
    const uint8_t *keys, *values;
    const float* scales;
    const int *positions, *token_entry, *table;
    const void* gate;            // logits of an output gate, [tokens, nq] or [tokens, nq * gate_width]; null: none
    int64_t gate_stride;
    const float* sink;           // [nq]: exp(sink) is one more term of the head's denominator; null: none
    const int* items;            // the matrix-core kernels' work: (first row, rows, entry, 0) a piece, and how it is cut (attn8_cut)
    const int* cut;
    float *part_o, *part_ml;
    int dtype, tokens, entries, table_width, nq, nkv, d, page_size, num_pages, window, chunk, gate_width, n_items, max_work, join_here, unused;
    float scale, softcap;
};

namespace cache8 {

constexpr int TILE = 64;         // keys of a step of the matrix-core kernels

// The lowest key that a token at `pos` sees.
__device__ __forceinline__ int low_key(int window, int chunk, int pos) {
    if (chunk > 0) return pos > 0 ? pos / chunk * chunk : 0;
    return window > 0 ? max(0, pos - window + 1) : 0;
}
__device__ __forceinline__ float sigmoid_of(float x) { return 1.f / (1.f + __expf(-x)); }

// What a cut is: for every workgroup a piece (no rows: nothing to do), for every item its first piece and how many it has, then
// the counters of arrived pieces where the last one joins them.
struct Piece {
    int row0, rows, entry, item;              // the item
    int tile, tile_end, first, pieces;        // its stretch of tiles; the item's first piece and how many there are
    int hi, pos0, unused[2];                  // the positions of the item's last and first row
};
constexpr int PIECE_INTS = sizeof(Piece) / 4;

}  // namespace cache8
