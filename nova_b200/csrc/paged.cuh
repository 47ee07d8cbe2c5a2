// Layout shared by the paged-cache kernels: plan records and cache addressing.
#pragma once

#include "common.cuh"

namespace nova {
namespace paged {

constexpr int D = 128;          // head_dim
constexpr int PT = 64;          // tokens per page
constexpr int HALF_ROW = PT * D;   // elements of K (or V) of one page and head

// Plan records (int32, see nova_paged_plan).
struct Seq {                    // one request
    int q_start, q_len, kv_len, page_off, tail_in, tail_out, pad0, pad1;
};
struct RowsItem {               // few query rows x a range of 64-token blocks
    int row0, nrows, blk0, blk1, part0, split, n_splits;
    int q_start, start, kv_len, page_off, tail;   // the request's: first token row, position of its first new token, ...
    int page[4];                // of blocks blk0 .. blk0 + 3: each warp's first, so that its loads need no other record
};
struct TileSeg {                // many query rows (up to 256) x a range of blocks; part < 0: the whole tile
    int head, row0, nrows, blk0, blk1, part, q_start;
    int start, kv_len, page_off, tail;   // the request's: position of its first new token, ...
    int page[4];                // of blocks blk0 .. blk0 + 3, so that the first loads need no other record
    int next;                   // the CTA's next segment, -1: none (segment c is CTA c's first)
};
struct TileJoin {               // a tile whose segments left partials
    int seq, head, row0, nrows, part0, n_parts, pad0, pad1;
};
struct OpenToken {              // one new token whose page stays open
    int row, pos, tail, pad;
};
struct Block {                  // one 64-token block of a request (write list: those that the step completes; read list)
    int blk, first, kv_len, row;         // row: token row of position `first`, the first new (written) or copied (read) one
    int tail_in, tail_out, page, pad;    // page: -1 while the block is open
};

constexpr int ROWS_MAX = 16;    // query rows of one KV head that the few-rows kernel takes per tile
constexpr int PART = 132;       // floats per row of a few-rows partial: m, l, 2 unused, acc[128]

constexpr int64_t WS_HEAD = 256;   // bytes of the workspace before the arrival counters: the error word

// Element offset of K (j = 0) or V (j = 1) of a page or tail buffer.
__host__ __device__ __forceinline__ int64_t half_off(int64_t index, int kv_heads, int head, int j) {
    return ((index * kv_heads + head) * 2 + j) * HALF_ROW;
}

}  // namespace paged
}  // namespace nova
