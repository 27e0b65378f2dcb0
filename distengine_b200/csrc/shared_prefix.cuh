// Work items of the attention whose requests share a prefix (shared_prefix.cu and the tensor-core
// kernels beside it); the host makes them (kernels/shared_prefix.py).
#pragma once

#include "common.cuh"

// The kernels of a step do not depend on one another, so one that another of them follows lets it start at
// once (FOLLOWED), on the SMs' memory and slots that its own blocks leave; the last one lets the merge
// start when it is nearly done.  Those behind the first (BEHIND) need not wait before they begin: the first
// one's blocks let them start after their own wait, when what the step reads was complete.  They wait
// before they end instead, so that what waits for them has waited for all.  (Eight beams in
// float32, two kernels: 14.8 us; with the second started when the first is nearly done 25.2.)

namespace shared_prefix {

constexpr int BEHIND = 1, FOLLOWED = 2;                   // bits of `order`

constexpr int HALF_ROWS = 128;

// A tile of query rows with a range of keys.  Rows are (token, query head of the kv head's group),
// counted from the first token of the owner: all requests of a group for keys of its prefix, one
// request for its own keys.
struct Item {
    int tok0;        // the owner's first token
    int count;       // the tile's rows
    int row0;        // the tile's first row
    int seq;         // the request whose page table is read
    int begin;       // prefix: the range's first key; own keys: the prefix's length
    int end;         // prefix: behind the range's last key; own keys: -1
    int split;       // own keys: which of `splits` equal ranges this is, | splits << 16;
                     // prefix: 1 where the range has two places for up to HALF_ROWS rows each
    int base;        // the tile's place among the partial results, in rows
};

// Where the partial results of a request lie: row r of the group (of the request) is row r % rows of
// tile r / rows; a tile's chunks are consecutive.
struct Joined {
    int tok0, group_tok0;
    int prefix_base, prefix_chunks, prefix_rows;
    int own_base, own_chunks, own_rows;
};

struct Range {
    int begin, end;          // keys of the item
    int pos0;                // position of the owner's first token; prefix: beyond every key
    // behind the last key that row i of the tile sees; rows that do not exist see none
    __device__ __forceinline__ int row_end(const Item& it, int i, int g) const {
        if (i >= it.count) return begin;
        return pos0 < 0 ? end : min(end, pos0 + (it.row0 + i) / g + 1);
    }
};

// The keys of an item.  Own keys: from the prefix's end to the position of the tile's last token, in
// `splits` ranges of a multiple of `unit` keys.
__device__ __forceinline__ Range range_of(const Item& it, const int* seq_pos0, int g, int unit) {
    Range r;
    if (it.end >= 0) {
        r.begin = it.begin;
        r.end = it.end;
        r.pos0 = -1;
        return r;
    }
    r.pos0 = seq_pos0[it.seq];
    const int stop = max(it.begin, r.pos0 + (it.row0 + it.count - 1) / g + 1);
    const int splits = it.split >> 16, part = it.split & 0xffff;
    int each = (stop - it.begin + splits - 1) / splits;
    each = (each + unit - 1) / unit * unit;
    r.begin = min(stop, it.begin + part * each);
    r.end = min(stop, r.begin + each);
    return r;
}

// The second place of a range that has two, by a kernel that needs one: no key.
__device__ __forceinline__ bool has_second_place(const Item& it) { return it.end >= 0 && it.split; }

// A page of a request; -1, with the status set, where it has none.
__device__ __forceinline__ int page_of(const int* block_table, int table_stride, int num_pages,
                                       int slot, int logical, int* status) {
    int id = -1;
    if (logical < table_stride && slot >= 0) id = block_table[(size_t)slot * table_stride + logical];
    if (id < 0 || id >= num_pages) {
        atomicExch(status, 2);
        return -1;
    }
    return id;
}

}  // namespace shared_prefix
