// The list of rows and key ranges that the kernels of a shared prefix work from, made by the host (library.py,
// `SharedPrefixes`) as one array of 32-bit integers:
//   [0]  ranges in use, [1] row tiles in use, [2], [3] unused
//   own_start[num_seqs]    the first key that is a sequence's own (the length of its group's prefix; 0 without one)
//   place[num_seqs]        row tile * SP_ROWS + first row of the sequence in it; -1 without a prefix
//   members[num_seqs]      the sequences of the groups, one group after the other
//   parts[cap_tiles][2]    a row tile's first range and how many it has
//   (filled up to a multiple of four integers)
//   tiles[cap_tiles][4]    the sequence whose block table is read, the first of its members, how many, the prefix's length
//   items[cap_items][4]    row tile, first key (a multiple of 64), end of the keys, 0
// The capacities belong to the array, so that a captured launch serves other lists of the same shape.
#pragma once
#include <stdint.h>

#define SP_ROWS 128                // rows (sequence, head of the group) of a tile

struct SharedItem { int tile, key_begin, key_end, unused; };
struct SharedTile { int table_seq, first, count, prefix; };

struct SharedPlan {
    const int* base;
    int num_seqs, cap_tiles, cap_items, tiles_at;
    __device__ __forceinline__ int items_used() const { return min(base[0], cap_items); }
    __device__ __forceinline__ int own_start(int seq) const { return base[4 + seq]; }
    __device__ __forceinline__ int place(int seq) const { return base[4 + num_seqs + seq]; }
    __device__ __forceinline__ int member(int i) const { return base[4 + 2 * num_seqs + i]; }
    __device__ __forceinline__ int2 parts(int tile) const {
        const int* at = base + 4 + 3 * num_seqs + 2 * tile;
        return make_int2(at[0], at[1]);
    }
    __device__ __forceinline__ SharedTile tile(int t) const {
        const int4 v = *reinterpret_cast<const int4*>(base + tiles_at + 4 * t);
        return SharedTile{v.x, v.y, v.z, v.w};
    }
    __device__ __forceinline__ SharedItem item(int i) const {
        const int4 v = *reinterpret_cast<const int4*>(base + tiles_at + 4 * cap_tiles + 4 * i);
        return SharedItem{v.x, v.y, v.z, v.w};
    }
};

static inline SharedPlan shared_plan(const int* base, int num_seqs, int cap_tiles, int cap_items) {
    SharedPlan s;
    s.base = base; s.num_seqs = num_seqs; s.cap_tiles = cap_tiles; s.cap_items = cap_items;
    s.tiles_at = (4 + 3 * num_seqs + 2 * cap_tiles + 3) / 4 * 4;
    return s;
}
