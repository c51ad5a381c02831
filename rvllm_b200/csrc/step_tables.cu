// Block tables, slot maps and positions of a step, built on the device from the requests' lengths.
//
// A table of pages stays on the device, one row per request slot and cache group: [groups, table_rows, table_width].  A step
// brings, per sequence b, the row it owns, how many of that row's entries are already there (`held`), the position of its first
// token and how many tokens it brings; and one flat list of the pages that were handed out for the step, group by group and
// sequence by sequence.  With u(b) = ceil((start + q) / page) blocks in use, sequence b of group g takes the next
// max(0, u - held) pages of the list for the entries [held, u) of its row, and
//   block_tables[g][b][j] = row[j] for live <= j < u, else -1   (live: the first block that a window or chunk still sees)
//   slot_mapping[g][t]    = row[pos / page] * page + pos % page  for token t at position pos
//   positions, token_seq, cu_seqlens, ctx_lens                   as the step's kernels read them.
// A sequence without a row (-1) stands for no request: its context length is 0, its entries and slots are -1.
//
// One launch for the tables, no order between its CTAs: where a sequence's pages begin in the list, and its tokens in the step, are sums over
// the sequences before it, which every CTA forms for itself (integers: any order gives the same), and an entry that is new in
// this step is read from the list, never from the row that another CTA may be writing.  A CTA takes 1, 2, 4 or 8 neighbouring
// sequences of one group, with 256, 128, 64 or 32 threads each: one while the CTAs find room at once (four an SM), more where the
// sums, which a CTA forms once, would be what it spends its time on.  Every index that comes from device memory is checked against its
// bound; an entry that would lie outside counts as absent (-1).
// What bounds it is latency - a launch, the lengths, the sums, the entries, each behind the other - and from a few hundred sequences on
// the sums, not the bytes.  GPU time in graphs with 1 / 2 / 4 / 8 sequences a CTA, us: 64 decoded tokens in contexts up to 32,767 (0.6 MB)
// 4.5 / 6.5 / 8.7 / 14; 800 in contexts up to 8,000 7.2 / 5.7 / 6.7 / 8.7; 2,000 21 / 15.9 / 9.7 / 11.2; 1,024 in two groups with
// portions (18 MB) 16.9 / 13.5 / 12.3 / 18.7, which is 1.5 TB/s.  The empty launch behind it (see there) takes 0.8 us more, and the host 2.7.
#include "common.cuh"

#define TABLE_THREADS 256

struct TableParams {
    int* page_table;               // [groups, table_rows, table_width]
    const int* rows;               // [num_seqs]
    const int* held;               // [groups, num_seqs]
    const int* starts;             // [num_seqs]
    const int* q_lens;             // [num_seqs]
    const int* new_pages;          // [num_new]
    const int* spans;              // [groups, 2]: window, chunk (0: none)
    int* block_tables;             // [groups, num_seqs, max_blocks]
    int* slot_mapping;             // [groups, num_tokens]
    int* positions;                // [num_tokens]
    int* token_seq;                // [num_tokens]
    int* cu_seqlens;               // [num_seqs + 1]
    int* ctx_lens;                 // [num_seqs]
    int groups, num_seqs, table_rows, table_width, num_new, num_tokens, max_blocks, page_size;
};

__device__ __forceinline__ int blocks_in_use(const TableParams& p, int b) {
    const int row = p.rows[b];
    const unsigned end = (unsigned)max(p.starts[b], 0) + (unsigned)max(p.q_lens[b], 0);
    if (row < 0 || row >= p.table_rows) return 0;
    return (int)min((end + (unsigned)p.page_size - 1u) / (unsigned)p.page_size, (unsigned)p.table_width);
}

template <int PER>
__global__ void __launch_bounds__(TABLE_THREADS)
step_tables_kernel(const TableParams p) {
    constexpr int THREADS = TABLE_THREADS / PER;             // of a sequence
    __shared__ unsigned sums[2][TABLE_THREADS / 32];
    __shared__ unsigned own[2][PER];                         // new pages and tokens of this CTA's sequences
    rv_pdl_wait();
    const int tid = threadIdx.x, g = blockIdx.y, b0 = blockIdx.x * PER;
    // pages taken before this CTA's first sequence (all groups before g, then the sequences before b0), tokens before it (unsigned, as
    // every place that follows from them: lengths whose sums pass 31 bits give places that are out of range, or others' in it)
    unsigned pages = 0, tokens = 0;
    for (int s = tid; s < p.num_seqs; s += TABLE_THREADS) {
        const int used = blocks_in_use(p, s);
        const int until = s < b0 ? g + 1 : g;                // groups in which s comes before
        for (int i = 0; i < until; ++i) pages += max(0, used - max(p.held[(size_t)i * p.num_seqs + s], 0));
        if (s < b0) tokens += max(p.q_lens[s], 0);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        pages += __shfl_xor_sync(0xffffffffu, pages, o);
        tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
    }
    if ((tid & 31) == 0) { sums[0][tid >> 5] = pages; sums[1][tid >> 5] = tokens; }
    const int sub = tid / THREADS, at = tid - sub * THREADS, b = b0 + sub;
    const bool here = b < p.num_seqs;
    const int row = here ? p.rows[b] : -1;
    const bool real = row >= 0 && row < p.table_rows;
    const int start = here ? max(p.starts[b], 0) : 0, q = here ? max(p.q_lens[b], 0) : 0;
    const int used = here ? blocks_in_use(p, b) : 0;
    const int held = here ? min(max(p.held[(size_t)g * p.num_seqs + b], 0), p.table_width) : 0;
    if (PER > 1 && at == 0) { own[0][sub] = max(0, used - held); own[1][sub] = q; }
    __syncthreads();
    pages = tokens = 0;
#pragma unroll
    for (int w = 0; w < TABLE_THREADS / 32; ++w) { pages += sums[0][w]; tokens += sums[1][w]; }
    if (PER > 1)
        for (int i = 0; i < sub; ++i) { pages += own[0][i]; tokens += own[1][i]; }
    if (!here) return;

    int* mine = p.page_table + ((size_t)g * p.table_rows + (real ? row : 0)) * p.table_width;
    auto entry = [&](int j) -> int {                         // j < used
        if (j < held) return mine[j];
        const unsigned i = pages + (unsigned)(j - held);
        return i < (unsigned)p.num_new ? p.new_pages[i] : -1;
    };
    for (int j = held + at; j < used; j += THREADS) mine[j] = entry(j);
    const int window = p.spans[2 * g], chunk = p.spans[2 * g + 1];
    int first = window > 0 ? max(0, start - window + 1) : 0;
    if (chunk > 0) first = max(first, start / chunk * chunk);
    const int live = first / p.page_size;
    int* out = p.block_tables + ((size_t)g * p.num_seqs + b) * p.max_blocks;
#pragma unroll 4
    for (int j = at; j < p.max_blocks; j += THREADS) out[j] = (j >= live && j < used) ? entry(j) : -1;
    for (int i = at; i < q; i += THREADS) {
        const unsigned t = tokens + (unsigned)i;
        if (t >= (unsigned)p.num_tokens) break;
        const unsigned pos = real ? (unsigned)start + (unsigned)i : 0u;
        const unsigned block = pos / (unsigned)p.page_size;
        int slot = -1;
        if (real && block < (unsigned)used) {
            const int page = entry((int)block);
            if (page >= 0) slot = page * p.page_size + (int)(pos - block * (unsigned)p.page_size);
        }
        p.slot_mapping[(size_t)g * p.num_tokens + t] = slot;
        if (g == 0) { p.positions[t] = (int)pos; p.token_seq[t] = b; }
    }
    if (b == p.num_seqs - 1)                                 // places behind the last sequence's tokens belong to none
        for (unsigned t = tokens + (unsigned)q + (unsigned)at; t < (unsigned)p.num_tokens; t += THREADS) {
            p.slot_mapping[(size_t)g * p.num_tokens + t] = -1;
            if (g == 0) { p.positions[t] = 0; p.token_seq[t] = -1; }
        }
    if (g == 0 && at == 0) {
        p.cu_seqlens[b] = (int)tokens;
        if (b == p.num_seqs - 1) p.cu_seqlens[p.num_seqs] = (int)(tokens + (unsigned)q);
        p.ctx_lens[b] = real ? (int)((unsigned)start + (unsigned)q) : 0;
    }
    // (no early signal: the step's other kernels may read this metadata before they wait for their predecessor, see below)
}

// Nothing, launched without the early attribute: it starts when the tables are complete, and a kernel behind it may read them before its
// own wait.  A launch that asks to start early right behind the tables would be promised them only after that wait.
__global__ void tables_settled_kernel() {}

// The arguments, packed by the caller in the order of TableParams, then the stream, and whether the next launch on it may be an early one.
struct TableArgs {
    TableParams p;
    cudaStream_t stream;
    int settle;
};

RV_EXPORT int rv_step_tables(const TableArgs* a) {
    const TableParams& p = a->p;
    if (p.groups < 1 || p.num_seqs < 1 || p.table_rows < 1 || p.table_width < 1 || p.num_new < 0 || p.num_tokens < 0 || p.max_blocks < 1 ||
        p.page_size < 1)
        return RV_ERR_BAD_SIZE;
    if (p.groups > 65535) return RV_ERR_UNSUPPORTED;
    const long long pairs = (long long)p.num_seqs * p.groups, room = 4LL * rv_sm_count();
    const int per = pairs <= room ? 1 : pairs <= 2 * room ? 2 : pairs <= 4 * room ? 4 : 8;
    const dim3 grid((p.num_seqs + per - 1) / per, p.groups);
    if (per == 1) RV_LAUNCH_ST = rv_launch(step_tables_kernel<1>, grid, dim3(TABLE_THREADS), 0, a->stream, p);
    else if (per == 2) RV_LAUNCH_ST = rv_launch(step_tables_kernel<2>, grid, dim3(TABLE_THREADS), 0, a->stream, p);
    else if (per == 4) RV_LAUNCH_ST = rv_launch(step_tables_kernel<4>, grid, dim3(TABLE_THREADS), 0, a->stream, p);
    else RV_LAUNCH_ST = rv_launch(step_tables_kernel<8>, grid, dim3(TABLE_THREADS), 0, a->stream, p);
    const int st = rv_launch_status();
    if (st != RV_OK || !a->settle) return st;            // (whether others are launched early is not for this library's switch to say)
    RV_LAUNCH_ST = rv_launch_alone(tables_settled_kernel, dim3(1), dim3(32), 0, a->stream);
    return rv_launch_status();
}
