// The list of rows and key ranges that the kernels of a shared prefix work from, made by the host (library.py,
// `SharedPrefixes`) as one array of 32-bit integers:
//   [0]  ranges in use, [1] row tiles in use, [2], [3] unused
//   own_start[num_seqs]    the first key that is a sequence's own (the length of its group's prefix; 0 without one)
//   place[num_seqs]        row tile * SP_ROWS + first row of the sequence in it; -1 without a prefix
//   members[num_seqs]      the sequences of the groups, one group after the other
//   parts[cap_tiles][2]    a row tile's first range and how many it has
//   (filled up to a multiple of four integers)
//   items[cap_items][8]    a range: first key (a multiple of 64), end of the keys (0: not in use), the sequence whose block table is
//                          read, the first of its row tile's members, how many they are, the row tile, 0, 0
// The capacities belong to the array, so that a captured launch serves other lists of the same shape.
#pragma once
#include <stdint.h>

#define SP_ROWS 128                // rows (sequence, head of the group) of a tile

struct SharedItem { int key_begin, key_end, table_seq, first, count; };

struct SharedPlan {
    const int* base;
    int num_seqs, items_at;
    __device__ __forceinline__ int own_start(int seq) const { return base[4 + seq]; }
    __device__ __forceinline__ int place(int seq) const { return base[4 + num_seqs + seq]; }
    __device__ __forceinline__ int member(int i) const { return base[4 + 2 * num_seqs + i]; }
    __device__ __forceinline__ int2 parts(int tile) const {
        const int* at = base + 4 + 3 * num_seqs + 2 * tile;
        return make_int2(at[0], at[1]);
    }
    __device__ __forceinline__ SharedItem item(int i) const {
        const int4* at = reinterpret_cast<const int4*>(base + items_at + 8 * i);
        const int4 v = at[0];
        return SharedItem{v.x, v.y, v.z, v.w, at[1].x};
    }
};

static inline SharedPlan shared_plan(const int* base, int num_seqs, int cap_tiles) {
    SharedPlan s;
    s.base = base; s.num_seqs = num_seqs;
    s.items_at = (4 + 3 * num_seqs + 2 * cap_tiles + 3) / 4 * 4;
    return s;
}
