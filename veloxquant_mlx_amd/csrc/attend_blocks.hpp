// A call of attention over chosen blocks of a packed store (attend_blocks.hip) and how it is cut: the store, parts and scratch of
// attention over spans (attend_span.hpp; one map, no prefix, no window), and the lists of blocks.
#pragma once
#include "attend_span.hpp"

namespace vq {

struct BlockCall {
    SpanCall s;
    const int32_t *blocks;   // [B][Hkv][tiles][count]
    int64_t tiles, count, block_tokens, query_block;
    int few;                 // 1: by the matrix-unit kernel for few rows (attend_span_few.hpp), with
    BlockLists lists;
    // 0: by blocks_any_kernel, with
    int rows16, row_tiles;   // 16s of rows of a tile, tiles of rows of a tile of queries
    int64_t sub;             // slots of an entry (at most the store's)
    int64_t list_slots, units;   // of a list, units of 32 of them and of the tail's
};

int launch_blocks_few2(const SpanCall &c, const BlockLists &l);
int launch_blocks_few4(const SpanCall &c, const BlockLists &l);

}  // namespace vq
