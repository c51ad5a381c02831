// Attention of a step's one-token sequences, groups of which begin with the same cached tokens (bfloat16): the keys of a group's
// prefix are read once for all of its sequences, on the fifth-generation tensor cores; the keys behind it sequence by sequence.
//
// The queries of a group for one key/value head are n G rows (n sequences, G = nh / nkv heads) against the same P keys:
//   S = scale Q K^T [n G x P],   m = max_j S,   l = sum_j e^(S - m),   O = e^(S - m) V
// a matrix product of the size of a prompt's attention, without a triangle.  The keys a sequence has to itself give another
// (m, l, O) by the same sums, and any number of them, over any ranges of the keys, are put together by
//   m' = max(m1, m2),   l' = l1 e^(m1 - m') + l2 e^(m2 - m'),   O' likewise,   out = O' / l'.
// Two kernels: the first has two kinds of CTAs, for ranges of the prefixes and for pieces of the own keys, all of which leave
// (O, m, l) unnormalised in 32 bits; the second adds them up row by row.
//
// One launch for both kinds, because neither fills the GPU alone: the prefixes' CTAs are few and busy with arithmetic, or many
// and waiting for memory; the own keys are a latency (lengths, pages, keys, each after the other) repeated for every sequence.  An
// SM holds two CTAs of either kind, the prefixes' are handed out first.  (As kernels of their own, one after the other, the 64
// sequences behind 2,048 shared keys with 1 to 700 of their own took 41 to 55 us in several forms; together they take 26.7.)
// Which rows and ranges there are is a list that the host makes once for a set of sequences: it changes when a request comes or
// goes, not from step to step (shared_prefix.cuh).
//
// A CTA of the prefixes owns up to 128 rows (floor(128 / G) whole sequences) of one kv head and one range of the keys: S = Q K^T of
// 64 keys into tensor memory, which is free again as soon as the softmax warps have read it, one thread per row of softmax, P into one of
// two buffers of tensor memory as bfloat16 pairs, read from there as the A operand of O += P V; two loader warps (keys, values: TMA
// boxes through the block table) and two warps that issue, as in attention_tcgen05.cu, which has the measurements behind this cut.
// What differs: rows come from sequences that lie anywhere in the batch (fetched by plain loads and swizzled by hand, while the first
// keys are on their way), keys behind the end of a prefix inside its last page belong to somebody else (their values are set to
// zero, so that a NaN there does not meet a probability of zero), and warps whose rows are all empty skip the softmax.
// P is rounded to bfloat16 (2^-8 relative at most), as in every attention kernel of this library: the tensor core takes no wider A
// beside a bfloat16 V; sums and maxima are float.
//
// The own keys: G rows against each key, so the bytes bound it (hd x 4 bytes a key and kv head) and what has to be won is latency: the
// lengths, the pages and the keys of a sequence follow from one another, and most sequences have few keys of their own.  All of
// them, cut into pieces, are one list, which the warps of a fixed number of CTAs take in turn; a warp works alone, on 16 keys at a time,
// and asks for the next chunks (TMA, into stages of its own) across the ends of pieces, so that their memory latencies overlap.  The
// products are turned over - S^T [16 keys x 8 heads] = K Q^T and O^T [16 dims x 8 heads] += V^T P^T on mma.sync, keys and values by
// ldmatrix - so that a group of up to eight heads fills the narrow side (a larger group is cut into blocks of eight); P^T gets from
// the layout of a result to that of an operand by two 8 x 8 transposes (movmatrix).  (The legacy matrix instruction, because its tile
// has a side of eight: a decoded token's G rows would leave most of tcgen05's 128 empty, and the time is the bytes'.  Before, the whole
// step of the example: a CTA per sequence and kv head, or several in a cluster, 41 to 70 us, most of it set-up; a list of pieces whose
// keys went from global memory straight into registers 50 us, 8 to 13 us a piece of 64.)
// Keys outside a sequence, and pages that do not exist, count as not there.
//
// What it takes (one B200, heads of 128; time of both kernels in a graph, bytes or products that it cannot do without):
//   4 sequences behind 32,768 keys, 32 heads on 8      33.2 us   136 MB, 4.1 TB/s (7 during the prefixes; the merge is 3 us)
//   64 behind 2,048 with 1 to 700 of their own         26.7 us    49 MB, 1.8 TB/s: filling, the own keys' second half, the merge
//   256 behind 16,384                                  93.7 us   69 GFLOP, 0.74 PFLOP/s (0.44 of measured): the softmax warps' chain, some
//                                                               1,900 cycles a tile of 64 keys with two CTAs an SM (tensor pipe busy 40 %)
//   8 behind 1,003, 28 heads on 4                      10.1 us   two launches and the latencies of one range
// Cache layer layout: [num_pages, 2 (k, v), nkv, page_size, HEAD_DIM].
#include "common.cuh"
#include "shared_prefix.cuh"
#include "tcgen05_attention.cuh"

#ifndef HEAD_DIM
#define HEAD_DIM 128
#endif
static_assert(HEAD_DIM == 64 || HEAD_DIM == 128, "this kernel is built for head sizes 64 and 128");

#define ROWS SP_ROWS
#define KV_TILE 64
#define SOFTMAX_WARPS 4
#define LOADER_WARP SOFTMAX_WARPS               // the keys
#define VLOADER_WARP (SOFTMAX_WARPS + 1)        // the values
#define QK_WARP (SOFTMAX_WARPS + 2)             // issues S = Q K^T (and allocates the tensor memory)
#define PV_WARP (SOFTMAX_WARPS + 3)             // issues O += P V
#define HALVES (HEAD_DIM / 64)
#define Q_BYTES (ROWS * HEAD_DIM * 2)
#define TILE_BYTES (KV_TILE * HEAD_DIM * 2)
#define NUM_THREADS (32 * (SOFTMAX_WARPS + 4))
// two CTAs an SM: 128 registers a thread at launch, (200 + 56) x 128 = 128 x 256 after the split
#define REGS_SOFTMAX 200
#define REGS_OTHERS 56
#define TMEM_COLS 256
#define S_COL 0                     // one S buffer of 64 columns: free again as soon as the softmax warps have read it
#define P_COL 64                    // two P buffers (bf16 pairs) of 32 columns
#define O_COL 128
#define NK (HEAD_DIM == 128 ? 3 : 4)
#define NV (HEAD_DIM == 128 ? 2 : 4)
// mbarriers, by their index
#define B_Q 0
#define B_K 1
#define B_KFREE (B_K + NK)
#define B_V (B_KFREE + NK)
#define B_VFREE (B_V + NV)
#define B_SFULL (B_VFREE + NV)
#define B_SFREE (B_SFULL + 1)
#define B_OFULL (B_SFREE + 1)      // [2] each from here on
#define B_PFULL (B_OFULL + 2)
#define NUM_BARS (B_PFULL + 2)
static_assert(SOFTMAX_WARPS * 32 * 36 * 4 <= NK * TILE_BYTES, "the softmax warps turn their rows over in the keys' ring");
static_assert(NUM_BARS <= 30, "the barriers, the tensor-memory address and the abort flag share 256 bytes");
#define RESCALE_LOG2 8.0f

struct SharedParams {
    SharedPlan plan;
    const __nv_bfloat16* q;        // [num_seqs, nh, HEAD_DIM]: sequence b brings row b
    const __nv_bfloat16* cache;
    const int* block_tables;       // [num_seqs, max_blocks]
    const int* ctx_lens;
    float* pre_o;                  // [items, nkv, ROWS, HEAD_DIM]: the prefixes' sums
    float* pre_ml;                 // [items, nkv, ROWS, 2]
    float* own_o;                  // [pieces, num_seqs, nh, HEAD_DIM]: those of the own keys
    float* own_ml;                 // [pieces, num_seqs, nh, 2]
    int* status;
    int num_seqs, nh, nkv, page_shift, page_size, max_blocks, num_pages;
    int prefix_ctas;               // nkv * items; the CTAs behind them are those of the own keys:
    int head_blocks;               // blocks of eight heads of a group
    int pieces, piece;             // the most pieces of a sequence, the keys of one
    float scale_log2e, cap_log2e, scale_over_cap;
};

// The running (maximum, denominator, four columns) of a row, and one more part's taken up into it.  One without keys (l = 0) may hold any sum; one whose
// scores are no numbers has a maximum of -inf and an l that is none either, and passes that on.
struct Merged {
    float m = -INFINITY, l = 0.f;
    float4 o = {0.f, 0.f, 0.f, 0.f};
    __device__ __forceinline__ void take(float pm, float pl, const float4& po) {
        if (pl == 0.f) return;
        const float m_new = fmaxf(m, pm);
        const float keep = fast_exp2(m - m_new), f = fast_exp2(pm - m_new);
        m = m_new;
        l = l * keep + pl * f;
        o.x = o.x * keep + po.x * f; o.y = o.y * keep + po.y * f;
        o.z = o.z * keep + po.z * f; o.w = o.w * keep + po.w * f;
    }
};

// Pieces that the own keys of a sequence are cut into: as many as its own length asks for, at most as many as there is room for.
__device__ __forceinline__ int pieces_of(int own, int piece, int most) { return max(1, min(most, (own + piece - 1) / piece)); }

// A wait of a whole warp, whose lanes all give up when one does.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, code));
}

__device__ __forceinline__ void own_keys(const SharedParams& p, const CUtensorMap& map, unsigned char* smem, int cta);

__global__ void __launch_bounds__(NUM_THREADS, 2)
shared_attention_kernel(const __grid_constant__ CUtensorMap map_kv, const __grid_constant__ CUtensorMap map_own, const SharedParams p) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* q_s = smem_raw;                           // [HALVES][128 rows x 128 B]
    unsigned char* k_s = q_s + Q_BYTES;                      // [NK stages][HALVES][KV_TILE keys x 128 B]
    unsigned char* v_s = k_s + NK * TILE_BYTES;              // [NV stages][HALVES][KV_TILE keys x 128 B]
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_s + NV * TILE_BYTES);
    uint32_t& tmem_base_slot = *reinterpret_cast<uint32_t*>(bars + 30);
    volatile int& abort_flag = *reinterpret_cast<volatile int*>(bars + 31);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) tma_prefetch_descriptor(&map_kv);
    const uint32_t bar_q = smem_u32(&bars[B_Q]);
    const uint32_t bar_k0 = smem_u32(&bars[B_K]), bar_kfree0 = smem_u32(&bars[B_KFREE]);
    const uint32_t bar_v0 = smem_u32(&bars[B_V]), bar_vfree0 = smem_u32(&bars[B_VFREE]);
    const uint32_t bar_s_full = smem_u32(&bars[B_SFULL]), bar_s_free = smem_u32(&bars[B_SFREE]);
    const uint32_t bar_o_full0 = smem_u32(&bars[B_OFULL]), bar_p_full0 = smem_u32(&bars[B_PFULL]);

    rv_pdl_wait();
    if ((int)blockIdx.x >= p.prefix_ctas) {
        own_keys(p, map_own, smem_raw, (int)blockIdx.x - p.prefix_ctas);
        return;
    }
    const int item = blockIdx.x / p.nkv, kvh = blockIdx.x - item * p.nkv;
    const int G = p.nh / p.nkv;
    const SharedItem tile = p.plan.item(item);
    const int key_lo = tile.key_begin, key_hi = tile.key_end;               // a multiple of KV_TILE; the end may lie inside a page
    const int tile_rows = min(tile.count, ROWS / G) * G;
    if (key_hi <= key_lo || tile_rows <= 0) return;
    const int t_begin = key_lo / KV_TILE, n_it = (key_hi + KV_TILE - 1) / KV_TILE - t_begin;
    const int* table = p.block_tables + (size_t)tile.table_seq * p.max_blocks;

    // a softmax thread's row (its lane of tensor memory), and the sequence that it belongs to
    const int row = warp * 32 + lane;
    const bool in_range = warp < SOFTMAX_WARPS && row < tile_rows;
    const int my_seq = in_range ? p.plan.member(tile.first + row / G) : -1;
    if (tid == 0) {
        abort_flag = 0;
        mbar_init(bar_q, SOFTMAX_WARPS);
        for (int i = 0; i < NK; ++i) { mbar_init(bar_k0 + 8 * i, 1); mbar_init(bar_kfree0 + 8 * i, 1); }
        for (int i = 0; i < NV; ++i) { mbar_init(bar_v0 + 8 * i, 1); mbar_init(bar_vfree0 + 8 * i, 1); }
        mbar_init(bar_s_full, 1); mbar_init(bar_s_free, SOFTMAX_WARPS);
        for (int i = 0; i < 2; ++i) {
            mbar_init(bar_o_full0 + 8 * i, 1);
            mbar_init(bar_p_full0 + 8 * i, SOFTMAX_WARPS);                  // one arrival per warp
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == QK_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_slot)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    }
    tcgen05_fence_before();
    __syncthreads();
    tcgen05_fence_after();
    const uint32_t tmem_base = tmem_base_slot;
    // (only now that this CTA holds its tensor memory: a kernel behind this one might allocate before it waits)
    rv_pdl_launch_dependents();

    const int box_keys = p.page_size < KV_TILE ? p.page_size : KV_TILE;     // keys one TMA box brings
    const int boxes = KV_TILE / box_keys;
    int tiles_issued = 0;             // by this warp, if it is a loader
    if (warp == LOADER_WARP || warp == VLOADER_WARP) {
        // ------------------------------------------------------------ loader warps: TMA, one for keys, one for values
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS));
        const int which = warp == LOADER_WARP ? 0 : 1;
        const int stages = which == 0 ? NK : NV;
        const uint32_t bar_full0 = which == 0 ? bar_k0 : bar_v0, bar_free0 = which == 0 ? bar_kfree0 : bar_vfree0;
        const uint32_t ring = smem_u32(which == 0 ? k_s : v_s);
        auto lookup = [&](int t) -> int {               // this lane's page of tile t, or -1
            const int key = t * KV_TILE + lane * box_keys;
            if (lane >= boxes || key >= key_hi || (key >> p.page_shift) >= p.max_blocks) return -1;
            const int page = __ldg(table + (key >> p.page_shift));
            return page < p.num_pages ? page : -1;
        };
        auto issue = [&](int t, int stage, int page) {
            const uint32_t bar = bar_full0 + 8 * stage;
            const int key = t * KV_TILE + lane * box_keys;
            const unsigned mask = __ballot_sync(0xffffffffu, page >= 0);
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)__popc(mask) * HALVES * (uint32_t)box_keys * 128u);
            __syncwarp();
            if (page >= 0) {
                const int row = ((page * 2 + which) * p.nkv + kvh) * p.page_size + (key & (p.page_size - 1));
#pragma unroll
                for (int h = 0; h < HALVES; ++h)
                    tma_load_2d(ring + (uint32_t)stage * TILE_BYTES + (uint32_t)h * (KV_TILE * 128) + (uint32_t)lane * box_keys * 128,
                                &map_kv, h * 64, row, bar);
            }
            __syncwarp();
        };
        for (int i = 0; i < stages && i < n_it; ++i, ++tiles_issued) issue(t_begin + i, i, lookup(t_begin + i));
        int page = stages < n_it ? lookup(t_begin + stages) : -1;
        int stage = 0;
        uint32_t phase = 0;
        for (int e = 0; e + stages < n_it; ++e) {
            const int next = e + 1 + stages < n_it ? lookup(t_begin + e + 1 + stages) : -1;     // a turn before it is needed
            int ok_l = 1;
            if (lane == 0) ok_l = mbar_wait(bar_free0 + 8 * stage, phase, &abort_flag, 3 + which) ? 1 : 0;
            if (!__shfl_sync(0xffffffffu, ok_l, 0)) break;
            issue(t_begin + e + stages, stage, page);
            ++tiles_issued;
            page = next;
            if (++stage == stages) { stage = 0; phase ^= 1; }
        }
    } else if (warp == QK_WARP) {
        // ------------------------------------------------------------ S = Q K^T
        // S(i) goes where S(i - 1) was, once the four warps have read that.  It is issued after the product with P(i - 2) has
        // finished, so a softmax warp that has seen S(i) may write P(i) where P(i - 2) was.
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS));
        if (lane == 0) {
            const uint32_t idesc_s = umma_idesc_bf16(ROWS, KV_TILE);
            int k_stage = 0;
            uint32_t k_phase = 0;
            const bool ready = mbar_wait(bar_q, 0, &abort_flag, 1);
            for (int i = 0; i < n_it && ready; ++i) {
                if (!mbar_wait(bar_k0 + 8 * k_stage, k_phase, &abort_flag, 5)) break;
                if (i >= 2 && !mbar_wait(bar_o_full0 + 8 * (i & 1), ((i - 2) >> 1) & 1, &abort_flag, 6)) break;
                if (i >= 1 && !mbar_wait(bar_s_free, (i - 1) & 1, &abort_flag, 13)) break;
                tcgen05_fence_after();
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    const uint64_t dq = umma_desc(smem_u32(q_s) + h * (ROWS * 128));
                    const uint64_t dk = umma_desc(smem_u32(k_s) + k_stage * TILE_BYTES + h * (KV_TILE * 128));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        tcgen05_mma_bf16(tmem_base + S_COL, dq + (uint64_t)(2 * j), dk + (uint64_t)(2 * j), idesc_s, (h | j) != 0);
                }
                tcgen05_commit(bar_s_full);
                tcgen05_commit(bar_kfree0 + 8 * k_stage);
                if (++k_stage == NK) { k_stage = 0; k_phase ^= 1; }
            }
        }
    } else if (warp == PV_WARP) {
        // ------------------------------------------------------------ O += P V
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OTHERS));
        if (lane == 0) {
            const uint32_t idesc_o = umma_idesc_bf16(ROWS, HEAD_DIM) | (1u << 16);          // B is MN-major
            int v_stage = 0;
            uint32_t v_phase = 0;
            for (int i = 0; i < n_it; ++i) {
                const int b = i & 1;
                if (!mbar_wait(bar_v0 + 8 * v_stage, v_phase, &abort_flag, 7)) break;
                if (!mbar_wait(bar_p_full0 + 8 * b, (i >> 1) & 1, &abort_flag, 8)) break;
                tcgen05_fence_after();
                const uint32_t tp = tmem_base + P_COL + b * (KV_TILE / 2);
                const uint64_t dv = umma_desc_mn(smem_u32(v_s) + v_stage * TILE_BYTES, KV_TILE * 128);
#pragma unroll
                for (int j = 0; j < KV_TILE / 16; ++j)
                    tcgen05_mma_bf16_ts(tmem_base + O_COL, tp + 8 * j, dv + (uint64_t)(128 * j), idesc_o, (i | j) != 0);
                tcgen05_commit(bar_vfree0 + 8 * v_stage);
                tcgen05_commit(bar_o_full0 + 8 * b);
                if (++v_stage == NV) { v_stage = 0; v_phase ^= 1; }
            }
        }
    } else {
        // ------------------------------------------------------------ softmax warps: one thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_SOFTMAX));
        const bool rows_here = warp * 32 < tile_rows;                // (a warp without rows only hands its buffers on)
        // The rows' queries, 16 bytes a lane, to their places in the 128-byte swizzle; rows without a sequence are zeros.  A warp fetches
        // its own 32 rows, all loads at a time.
        constexpr int LANES = HEAD_DIM / 8;                          // that bring a row
        const int my_row = in_range ? my_seq * p.nh + kvh * G + row % G : -1;
        uint4 qv[LANES];
#pragma unroll
        for (int i = 0; i < LANES; ++i) {
            const int from = __shfl_sync(0xffffffffu, my_row, i * (32 / LANES) + lane / LANES);
            qv[i] = from >= 0 ? *reinterpret_cast<const uint4*>(p.q + (size_t)from * HEAD_DIM + (lane % LANES) * 8) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < LANES; ++i) {
            const int r = warp * 32 + i * (32 / LANES) + lane / LANES, chunk = lane % LANES;
            *reinterpret_cast<uint4*>(q_s + (chunk >> 3) * (ROWS * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) = qv[i];
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_q);
        // a row sees the keys of the range that its sequence has
        const int limit = in_range ? min(key_hi, p.ctx_lens[my_seq]) : 0;
        const uint32_t t_lane = tmem_base + ((uint32_t)(warp * 32) << 16);
        float m_ref = -INFINITY, l_run = 0.f;
        bool ok = true;
        for (int it = 0; it < n_it; ++it) {
            const int pb = it & 1;
            const int key0 = (t_begin + it) * KV_TILE;
            if (!warp_wait(bar_s_full, it & 1, &abort_flag, 9)) { ok = false; break; }
            tcgen05_fence_after();
            uint32_t s0[32], s1[32];
            if (rows_here) {
                tmem_ld_32x32(t_lane + S_COL, s0);
                tmem_ld_32x32(t_lane + S_COL + 32, s1);
                tmem_ld_wait();
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_s_free);
            if (key0 + KV_TILE > key_hi) {
                // values of keys behind the range's end: zeros, before the product may read them (it waits for P of all four warps)
                if (!warp_wait(bar_v0 + 8 * (it % NV), (it / NV) & 1, &abort_flag, 12)) { ok = false; break; }
                const int from = key_hi - key0, n = (KV_TILE - from) * 8;
                unsigned char* vt = v_s + (it % NV) * TILE_BYTES;
                for (int i = tid; i < HALVES * n; i += 32 * SOFTMAX_WARPS) {
                    const int h = i / n;
                    reinterpret_cast<uint4*>(vt + h * (KV_TILE * 128) + from * 128)[i - h * n] = make_uint4(0, 0, 0, 0);
                }
                fence_async_smem();
            }
            if (rows_here) {
                // with a cap the scores become c log2(e) tanh(scale s / c) here (tanh as 1 - 2 / (e^2x + 1)), and the scale below is 1
                const float eff_scale = p.cap_log2e > 0.f ? 1.f : p.scale_log2e;
                if (p.cap_log2e > 0.f) {
                    const float k2 = p.scale_over_cap * 2.885390081777927f;
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        const float ea = fast_exp2(__uint_as_float(s0[e]) * k2), eb = fast_exp2(__uint_as_float(s1[e]) * k2);
                        s0[e] = __float_as_uint(p.cap_log2e * (1.f - __fdividef(2.f, ea + 1.f)));
                        s1[e] = __float_as_uint(p.cap_log2e * (1.f - __fdividef(2.f, eb + 1.f)));
                    }
                }
                if (key0 + KV_TILE > limit) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) {
                        if (key0 + e >= limit) s0[e] = 0xff800000u;               // -inf
                        if (key0 + 32 + e >= limit) s1[e] = 0xff800000u;
                    }
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    mx[0] = max3(mx[0], __uint_as_float(s0[e]), __uint_as_float(s0[e + 1]));
                    mx[1] = max3(mx[1], __uint_as_float(s0[e + 2]), __uint_as_float(s0[e + 3]));
                    mx[2] = max3(mx[2], __uint_as_float(s1[e]), __uint_as_float(s1[e + 1]));
                    mx[3] = max3(mx[3], __uint_as_float(s1[e + 2]), __uint_as_float(s1[e + 3]));
                }
                const float m_tile = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * eff_scale;
                // The reference maximum is raised only when it is more than 2^8 behind: O then needs a pass.  The exponentials do not
                // wait to know: they are formed under the old reference beside the maximum, and once more in the rare tile that raises it.
                // (The first tile has its maximum to begin with; the empty statement keeps this a branch, a selection would make every
                // tile's exponentials wait.)
                if (it == 0) { m_ref = m_tile; asm volatile("" : "+f"(m_ref)); }
                bool raise = m_tile > m_ref + RESCALE_LOG2 || (m_ref == -INFINITY && m_tile > -INFINITY);
                uint32_t pk[32];
                float l_tile, l_tile2;
                for (;;) {
                    const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
                    l_tile = l_tile2 = 0.f;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {               // keys 2j and 2j + 1 of the tile: one column of P
                        const int e = 2 * j;
                        float a0, a1;
                        fma2(a0, a1, __uint_as_float(e < 32 ? s0[e] : s1[e - 32]), __uint_as_float(e + 1 < 32 ? s0[e + 1] : s1[e + 1 - 32]),
                             eff_scale, neg_m);
                        const float x0 = fast_exp2(a0), x1 = fast_exp2(a1);
                        add2(l_tile, l_tile2, x0, x1);
                        const __nv_bfloat162 h2 = __floats2bfloat162_rn(x0, x1);
                        pk[j] = *reinterpret_cast<const uint32_t*>(&h2);
                    }
                    if (!__any_sync(0xffffffffu, raise)) break;
                    float factor = 1.f;
                    if (raise) {
                        factor = m_ref == -INFINITY ? 0.f : fast_exp2(m_ref - m_tile);
                        m_ref = m_tile;
                        l_run *= factor;
                        raise = false;
                    }
                    // the product of the tile before must have finished; the one after waits for this warp's P
                    if (!warp_wait(bar_o_full0 + 8 * (pb ^ 1), ((it - 1) >> 1) & 1, &abort_flag, 11)) { ok = false; break; }
                    tcgen05_fence_after();
#pragma unroll
                    for (int c = 0; c < HEAD_DIM; c += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32(t_lane + O_COL + c, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
                        tmem_st_32x32(t_lane + O_COL + c, o);
                    }
                    tmem_st_wait();
                    tcgen05_fence_before();
                }
                if (!ok) break;
                l_run += l_tile + l_tile2;
                tmem_st_32x32(t_lane + P_COL + pb * (KV_TILE / 2), pk);
                tmem_st_wait();
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_p_full0 + 8 * pb);
        }
        if (ok) {
            ok = warp_wait(bar_o_full0 + 8 * ((n_it - 1) & 1), ((n_it - 1) >> 1) & 1, &abort_flag, 10);
            tcgen05_fence_after();
            if (ok && rows_here) {
                // A thread holds a row, so its stores would be 16 bytes here and there: the warp turns 32 x 32 floats over in shared
                // memory (its share of the keys' ring, which no product reads any more) and stores whole lines of four rows.
                const size_t prow0 = ((size_t)item * p.nkv + kvh) * ROWS + warp * 32;
                if (in_range) *reinterpret_cast<float2*>(p.pre_ml + (prow0 + lane) * 2) = make_float2(m_ref, l_run);
                float* turn = reinterpret_cast<float*>(k_s) + warp * (32 * 36);
                const int last = min(32, tile_rows - warp * 32);
#pragma unroll
                for (int c = 0; c < HEAD_DIM; c += 32) {
                    uint32_t o[32];
                    tmem_ld_32x32(t_lane + O_COL + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        *reinterpret_cast<uint4*>(turn + lane * 36 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    __syncwarp();
#pragma unroll
                    for (int r0 = 0; r0 < 32; r0 += 4) {
                        const int r = r0 + (lane >> 3);
                        const uint4 v = *reinterpret_cast<const uint4*>(turn + r * 36 + (lane & 7) * 4);
                        if (r < last) *reinterpret_cast<uint4*>(p.pre_o + (prow0 + r) * HEAD_DIM + c + (lane & 7) * 4) = v;
                    }
                    __syncwarp();
                }
            }
        }
    }

    tcgen05_fence_before();
    __syncthreads();
    if (abort_flag != 0) {
        // A wait gave up somewhere: tiles may still be on their way into this CTA's shared memory with nobody left to wait for
        // them.  Their loaders do (bounded, without touching the flag) before the CTA ends.
        if ((warp == LOADER_WARP || warp == VLOADER_WARP) && lane == 0) {
            volatile int ignore = 0;
            const int stages = warp == LOADER_WARP ? NK : NV;
            const uint32_t full0 = warp == LOADER_WARP ? bar_k0 : bar_v0;
            for (int i = max(0, tiles_issued - stages); i < tiles_issued; ++i)
                mbar_wait(full0 + 8 * (i % stages), (i / stages) & 1, &ignore, 0);
        }
        __syncthreads();
    }
    if (warp == QK_WARP)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS));
    if (tid == 0 && abort_flag != 0 && p.status) atomicCAS(p.status, 0, abort_flag);
}

// ---------------------------------------------------------------------------------------------
// The own keys (see the top of the file).
#define OWN_WARPS 4
#define OWN_THREADS (32 * OWN_WARPS)
#define OWN_CHUNK 16                           // keys
#define OWN_STAGES 2                           // of a warp; two CTAs an SM have 8 warps x 2 x 8 KB on their way (head size 128; three: no faster)
#define DIM_BLOCKS (HEAD_DIM / 16)
#define KEY_BYTES (HEAD_DIM * 2)               // a key, or a value, in shared memory: HALVES rows of 128 bytes
#define QUERY_BYTES (8 * HEAD_DIM * 2)
#define STAGE_BYTES (2 * OWN_CHUNK * KEY_BYTES)                            // of a box (a page, or the 16 keys of it): its keys, then its values
#define RING_BYTES (OWN_STAGES * STAGE_BYTES + QUERY_BYTES)                // of a warp; the queries come with a piece's first chunk
#define MERGE_BATCH 8
#define MERGE_BLOCKS 7                         // of an SM
#define MAX_SEQS 2048                          // of a step: what the list of pieces has room for

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}

// A warp's place in the list of pieces: which piece, and which chunk of it comes next.
struct OwnCursor {
    unsigned at;                   // piece x block of heads, in the whole list
    int seq, rank, kvh, head0;
    int chunk, chunk_end, ctx, start;
    bool first;                    // no chunk of the piece has been asked for yet
    int page;                      // of this lane's box of the chunk, -1 without one
};

__device__ __forceinline__ void own_keys(const SharedParams& p, const CUtensorMap& map, unsigned char* smem, int cta) {
    constexpr int HD = HEAD_DIM;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    rv_pdl_launch_dependents();
    // No second CTA of a kernel with tensor memory is placed on an SM while the first may still ask for some, so a CTA that needs
    // none says so (without this line the own keys' CTAs ran one an SM).
    if (warp == OWN_WARPS) asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
    if (warp >= OWN_WARPS) return;
    const int G = p.nh / p.nkv, blocks = p.nkv * p.head_blocks;
    unsigned char* ring = smem + warp * RING_BYTES;                        // (stages start on 1,024-byte boundaries: see the swizzle)
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OWN_WARPS * RING_BYTES);
    int* of_warp = reinterpret_cast<int*>(bars + OWN_WARPS * OWN_STAGES);
    volatile int& abort_flag = *reinterpret_cast<volatile int*>(of_warp + OWN_WARPS);
    int* before = of_warp + OWN_WARPS + 1;                                 // [num_seqs + 1]: pieces of the sequences before one
    int* ends = before + p.num_seqs + 1;                                   // [num_seqs]: context lengths
    int* begins = ends + p.num_seqs;                                       // [num_seqs]: first own keys
    const uint32_t bar0 = smem_u32(bars + warp * OWN_STAGES);
    if (tid == 0) abort_flag = 0;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < OWN_STAGES; ++i) mbar_init(bar0 + 8 * i, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const int each = (p.num_seqs + OWN_THREADS - 1) / OWN_THREADS, s_lo = min(tid * each, p.num_seqs), s_hi = min(s_lo + each, p.num_seqs);
    int mine = 0;
    for (int s = s_lo; s < s_hi; ++s) {
        const int ctx = max(p.ctx_lens[s], 0), start = min(p.plan.own_start(s), ctx);
        before[s] = mine; ends[s] = ctx; begins[s] = start;
        mine += pieces_of(ctx - start, p.piece, p.pieces);
    }
    int upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += other;
    }
    if (lane == 31) of_warp[warp] = upto;
    asm volatile("bar.sync 1, %0;" ::"n"(OWN_THREADS) : "memory");
    int base = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < OWN_WARPS; ++w) {
        base += w < warp ? of_warp[w] : 0;
        total += of_warp[w];
    }
    for (int s = s_lo; s < s_hi; ++s) before[s] += base;
    if (tid == 0) before[p.num_seqs] = total;
    asm volatile("bar.sync 1, %0;" ::"n"(OWN_THREADS) : "memory");

    const int warps = ((int)gridDim.x - p.prefix_ctas) * OWN_WARPS;
    const unsigned all = (unsigned)total * blocks;
    auto enter = [&](OwnCursor& c) {                 // the piece at c.at
        if (c.at >= all) return;
        const int piece = (int)(c.at / (unsigned)blocks), block = (int)c.at - piece * blocks;
        int seq = 0;
        for (int hi = p.num_seqs - 1; seq < hi;) {                         // the last sequence that begins at or before it
            const int mid = (seq + hi + 1) >> 1;
            if (before[mid] <= piece) seq = mid; else hi = mid - 1;
        }
        c.seq = seq;
        c.rank = piece - before[seq];
        c.kvh = block / p.head_blocks;
        c.head0 = (block - c.kvh * p.head_blocks) * 8;
        c.ctx = ends[seq];
        c.start = begins[seq];
        const int pieces = before[seq + 1] - before[seq];
        const int lo = c.start / OWN_CHUNK, chunks = (c.ctx + OWN_CHUNK - 1) / OWN_CHUNK - lo, per = (chunks + pieces - 1) / pieces;
        c.chunk = min(lo + c.rank * per, lo + chunks);
        c.chunk_end = min(lo + chunks, c.chunk + per);
        c.first = true;
    };
    auto next = [&](OwnCursor& c) {                  // the chunk behind c's, of the next piece if need be (an empty piece counts as one)
        c.first = false;
        if (++c.chunk >= c.chunk_end) { c.at += warps; enter(c); }
    };
    const int box_keys = p.page_size < OWN_CHUNK ? p.page_size : OWN_CHUNK, boxes = OWN_CHUNK / box_keys;
    const int box_bytes = 2 * box_keys * KEY_BYTES;
    // Lane i < boxes has the i-th box of a chunk, keys and values in one copy.  Its page is looked up when the chunk before has been
    // asked for, and looked at when the copy is.
    auto look_up = [&](OwnCursor& c) {
        const int key = c.chunk * OWN_CHUNK + lane * box_keys;
        c.page = -1;
        if (c.at < all && lane < boxes && c.chunk < c.chunk_end && key < c.ctx && key + box_keys > c.start && (key >> p.page_shift) < p.max_blocks)
            c.page = __ldg(p.block_tables + (size_t)c.seq * p.max_blocks + (key >> p.page_shift));
    };
    auto ask = [&](const OwnCursor& c, int stage) -> unsigned {
        const int page = c.page < p.num_pages ? c.page : -1;
        const unsigned mask = __ballot_sync(0xffffffffu, page >= 0);
        const uint32_t bar = bar0 + 8 * stage;
        const uint32_t query_bytes = c.first ? (uint32_t)min(8, G - c.head0) * HD * 2u : 0u;
        if (lane == 0) {
            mbar_expect_tx(bar, (uint32_t)__popc(mask) * (uint32_t)box_bytes + query_bytes);
            if (c.first) bulk_load(smem_u32(ring) + OWN_STAGES * STAGE_BYTES, p.q + ((size_t)c.seq * p.nh + c.kvh * G + c.head0) * HD, query_bytes, bar);
        }
        __syncwarp();
        if (page >= 0)
            tma_load_4d(smem_u32(ring) + stage * STAGE_BYTES + lane * box_bytes, &map, 0, 0,
                        c.kvh * p.page_size + ((c.chunk * OWN_CHUNK + lane * box_keys) & (p.page_size - 1)), 2 * page, bar);
        return mask;                                 // the boxes that come
    };
    // where key r of a chunk is in its stage (its value lies box_bytes / 2 further)
    auto key_at = [&](int r) { return (r / box_keys) * box_bytes + (r % box_keys) * KEY_BYTES; };

    OwnCursor ahead, now, pending;
    ahead.at = now.at = cta * OWN_WARPS + warp;
    enter(ahead);
    now = pending = ahead;
    look_up(ahead);
    unsigned here = 0;                               // which boxes of a stage have keys, two bits a stage
    int asked = 0, taken = 0;
    bool queries = false;                            // those of a piece are on their way, or lie there unread: one piece's at a time
    auto ask_ahead = [&]() {
        while (ahead.at < all && asked - taken < OWN_STAGES && !(ahead.first && queries)) {
            const int stage = asked % OWN_STAGES;
            here = (here & ~(3u << (2 * stage))) | ask(ahead, stage) << (2 * stage);
            if (ahead.first) { queries = true; pending = ahead; }
            ++asked;
            next(ahead);
            look_up(ahead);
        }
    };
    ask_ahead();
    const int g = lane >> 2, tq = lane & 3;
    uint32_t qf[DIM_BLOCKS][2];
    float o[DIM_BLOCKS][4], m_run[2], l_run[2];      // heads 2 tq, 2 tq + 1
    bool ok = true;
    // a lane's row of the keys and of the values as ldmatrix takes them: its place in a stage, the eight columns it names
    const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_half = lane >> 4, v_row = (lane & 7) + (lane >> 4) * 8, v_half = (lane >> 3) & 1;
    const uint32_t k_at = key_at(k_row), v_at = key_at(v_row) + box_bytes / 2;
    auto column = [](uint32_t row, int i, int half) {                      // of 16 i + 8 half, in the 128-byte swizzle
        const uint32_t line = row + (i >> 2) * 128;
        return line + (((2 * (i & 3) + half) ^ ((line >> 7) & 7)) << 4);
    };
    bool fresh = true;                               // the next chunk is the first of a piece
    while (taken < asked) {
        const int stage = taken % OWN_STAGES;
        if (!warp_wait(bar0 + 8 * stage, (taken / OWN_STAGES) & 1, &abort_flag, 14)) { ok = false; break; }
        const uint32_t at = smem_u32(ring) + stage * STAGE_BYTES;
        if (fresh) {
            now = pending;
            // Q as the B operand: elements 2 tq, 2 tq + 1 (and 8 on) of head g in every 16; heads beyond the block are zeros
            const uint32_t* q = reinterpret_cast<const uint32_t*>(ring + OWN_STAGES * STAGE_BYTES) + g * (HD / 2) + tq;
            const bool have = g < G - now.head0;
#pragma unroll
            for (int i = 0; i < DIM_BLOCKS; ++i) {
                qf[i][0] = have ? q[8 * i] : 0u;
                qf[i][1] = have ? q[8 * i + 4] : 0u;
                o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
            }
            m_run[0] = m_run[1] = -INFINITY;
            l_run[0] = l_run[1] = 0.f;
            queries = false;
        }
        // which of the chunk's keys there are, a bit each
        const int key0 = now.chunk * OWN_CHUNK;
        unsigned see = 0;
        if (now.chunk < now.chunk_end) {
            const int lo = max(now.start - key0, 0), hi = min(now.ctx - key0, OWN_CHUNK);
            see = hi > lo ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
            const unsigned got = here >> (2 * stage) & 3u;
            if (got != (1u << boxes) - 1u)
                for (int i = 0; i < boxes; ++i)
                    if (!(got >> i & 1u)) see &= ~(((1u << box_keys) - 1u) << (i * box_keys));
        }
        if (see != 0xffffu) {
            // values of keys that are not there: zeros, so that what an earlier request left, a NaN for instance, does not meet a
            // probability of zero
            if (!(see >> (lane >> 1) & 1u)) {
                unsigned char* to = ring + stage * STAGE_BYTES + key_at(lane >> 1) + box_bytes / 2 + (lane & 1) * (KEY_BYTES / 2);
#pragma unroll
                for (int i = 0; i < KEY_BYTES / 32; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(0, 0, 0, 0);
            }
            fence_async_smem();                      // (the next copy into the stage comes behind these writes)
            __syncwarp();
        }
        if (see) {
            float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < DIM_BLOCKS; ++i) {
                uint32_t a[4];
                ldmatrix_4(a, at + column(k_at, i, k_half));
                mma_16816(s, a, qf[i][0], qf[i][1]);
            }
            float alpha[2];
#pragma unroll
            for (int e = 0; e < 4; ++e) {                                  // e: key g + 8 (e >> 1), head 2 tq + (e & 1)
                float v = s[e] * p.scale_log2e;
                if (p.cap_log2e > 0.f) {
                    const float x = fast_exp2(s[e] * p.scale_over_cap * 2.885390081777927f);
                    v = p.cap_log2e * (1.f - __fdividef(2.f, x + 1.f));
                }
                s[e] = see >> (g + 8 * (e >> 1)) & 1u ? v : -INFINITY;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float mx = fmaxf(s[h], s[h + 2]);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
                const float m_new = fmaxf(m_run[h], mx);
                const float m_s = m_new == -INFINITY ? 0.f : m_new;
                alpha[h] = fast_exp2(m_run[h] - m_s);                      // 0 while nothing has been seen
                m_run[h] = m_new;
                s[h] = fast_exp2(s[h] - m_s);
                s[h + 2] = fast_exp2(s[h + 2] - m_s);
                l_run[h] = l_run[h] * alpha[h] + s[h] + s[h + 2];          // this lane's keys; the lanes are added at the end
            }
            const __nv_bfloat162 lo2 = __floats2bfloat162_rn(s[0], s[1]), hi2 = __floats2bfloat162_rn(s[2], s[3]);
            const uint32_t p0 = transpose_8x8(*reinterpret_cast<const uint32_t*>(&lo2));         // keys 2 tq, 2 tq + 1 of head g
            const uint32_t p1 = transpose_8x8(*reinterpret_cast<const uint32_t*>(&hi2));         // ... + 8
#pragma unroll
            for (int i = 0; i < DIM_BLOCKS; ++i) {                         // columns 16 i + g and 8 on
                o[i][0] *= alpha[0]; o[i][1] *= alpha[1];
                o[i][2] *= alpha[0]; o[i][3] *= alpha[1];
                uint32_t a[4];
                ldmatrix_4t(a, at + column(v_at, i, v_half));
                mma_16816(o[i], a, p0, p1);
            }
        }
        __syncwarp();                                // the stage has been read, and so have a first chunk's queries
        ++taken;
        ask_ahead();
        fresh = now.chunk + 1 >= now.chunk_end;
        ++now.chunk;
        if (fresh) {                                 // that was the piece's last chunk
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float l = l_run[h];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
                const int head = now.head0 + 2 * tq + h;
                if (head >= G) continue;
                const size_t to_row = ((size_t)now.rank * p.num_seqs + now.seq) * p.nh + now.kvh * G + head;
                if (g == 0) *reinterpret_cast<float2*>(p.own_ml + to_row * 2) = make_float2(m_run[h], l);
                float* to = p.own_o + to_row * HD + g;
#pragma unroll
                for (int i = 0; i < DIM_BLOCKS; ++i) { to[16 * i] = o[i][h]; to[16 * i + 8] = o[i][h + 2]; }
            }
        }
    }
    // A wait gave up: copies may still be on their way into this CTA's shared memory.  Waited for (bounded) before it is given up.
    if (!ok && lane == 0) {
        volatile int ignore = 0;
        for (int i = taken; i < asked; ++i) mbar_wait(bar0 + 8 * (i % OWN_STAGES), (i / OWN_STAGES) & 1, &ignore, 0);
        if (p.status) atomicCAS(p.status, 0, abort_flag);
    }
}

// ---------------------------------------------------------------------------------------------
// The sums of a row put together: WARPS warps per (sequence, head), which take its parts in turn, four neighbouring columns a lane
// and MERGE_BATCH parts' loads in flight.  What it costs is round trips to L2 - a row of 45 parts takes one warp six - and waves of
// blocks: so as many warps a row as still leave one wave (both kernels with 1 / 2 / 4 warps a row, us: 8 sequences of 28 heads, 18 parts
// 11.8 / 10.7 / 10.1; 4 of 32, 57 parts 38.5 / 35.0 / 33.2; 64 of 32, 14 parts 28.9 / 26.7 / 29.8; 256 of 32, 6 parts 93.7 / 99 / 110).
template <int WARPS>
__global__ void __launch_bounds__(128, MERGE_BLOCKS)
shared_merge_kernel(const SharedParams p, const float* __restrict__ sinks, const float* __restrict__ gate, __nv_bfloat16* __restrict__ out) {
    rv_pdl_launch_dependents();
    constexpr int LANES = HEAD_DIM / 4;              // that hold a row
    constexpr int TURNS = WARPS == 1 ? 1 : WARPS * 32 / LANES;             // groups of lanes that share one
    constexpr int ROWS_HERE = 128 / LANES / TURNS;   // rows of a block
    __shared__ float4 sh_o[TURNS == 1 ? 1 : 128 / LANES][LANES];
    __shared__ float2 sh_ml[128 / LANES];
    const int tid = threadIdx.x, group = tid / LANES, d = (tid - group * LANES) * 4;
    const int turn = group % TURNS;
    const int rows = p.num_seqs * p.nh, row = blockIdx.x * ROWS_HERE + group / TURNS;
    const bool here = row < rows;
    const int seq = here ? row / p.nh : 0, head = here ? row - seq * p.nh : 0;
    const int G = p.nh / p.nkv, kvh = head / G;
    const int ctx = max(p.ctx_lens[seq], 0);
    const int pieces = pieces_of(ctx - min(p.plan.own_start(seq), ctx), p.piece, p.pieces);
    const int place = p.plan.place(seq);
    int2 parts = make_int2(0, 0);
    if (place >= 0) parts = p.plan.parts(place / SP_ROWS);
    rv_pdl_wait();
    // the parts, prefix first: `turn`, turn + TURNS, ...
    const int total = here ? parts.y + pieces : 0;
    const size_t pre_at = ((size_t)parts.x * p.nkv + kvh) * SP_ROWS + (place >= 0 ? place % SP_ROWS + head - kvh * G : 0);
    Merged v;
    for (int s0 = turn; s0 < total; s0 += TURNS * MERGE_BATCH) {
        float2 ml[MERGE_BATCH];
        float4 o[MERGE_BATCH];
#pragma unroll
        for (int k = 0; k < MERGE_BATCH; ++k) {
            const int i = min(s0 + k * TURNS, total - 1);
            const bool pre = i < parts.y;
            const size_t at = pre ? pre_at + (size_t)i * p.nkv * SP_ROWS : (size_t)(i - parts.y) * rows + row;
            ml[k] = __ldcg(reinterpret_cast<const float2*>(pre ? p.pre_ml : p.own_ml) + at);
            o[k] = __ldcg(reinterpret_cast<const float4*>((pre ? p.pre_o : p.own_o) + at * HEAD_DIM + d));
        }
#pragma unroll
        for (int k = 0; k < MERGE_BATCH; ++k)
            if (s0 + k * TURNS < total) v.take(ml[k].x, ml[k].y, o[k]);
    }
    if (TURNS > 1) {
        sh_o[group][d / 4] = v.o;
        if (d == 0) sh_ml[group] = make_float2(v.m, v.l);
        __syncthreads();
        if (turn > 0) return;
#pragma unroll
        for (int t = 1; t < TURNS; ++t) v.take(sh_ml[group + t].x, sh_ml[group + t].y, sh_o[group + t][d / 4]);
    }
    if (!here) return;
    float num = 1.f, den = v.l;
    if (sinks) {                                     // exp(sink) joins the denominator; it has no value
        const float sk = sinks[head] * 1.4426950408889634f;
        const float m_new = fmaxf(v.m, sk);
        num = v.m == -INFINITY ? 0.f : fast_exp2(v.m - m_new);
        den = v.l * num + fast_exp2(sk - m_new);
    }
    float inv = den == 0.f ? 0.f : num / den;        // (what is no number stays so)
    if (gate) inv *= gate[row];
    rv_store4(out, RV_DTYPE_BF16, (size_t)row * HEAD_DIM + d, make_float4(v.o.x * inv, v.o.y * inv, v.o.z * inv, v.o.w * inv));
}

// ---------------------------------------------------------------- host side
// A cache layer as [planes of all pages][rows of a plane][64-element parts of a row][64]: a box brings some keys of a page and head
// and their values, in 128-byte rows with 128-byte swizzle.
static int make_own_map(CUtensorMap* map, const void* cache, long long num_pages, int nkv, int page_size) {
    RvEncodeTiledFn fn = rv_encode_fn();
    if (!fn) return RV_ERR_UNSUPPORTED;
    const cuuint64_t dims[4] = {64, HALVES, (cuuint64_t)nkv * page_size, (cuuint64_t)num_pages * 2};
    const cuuint64_t strides[3] = {128, KEY_BYTES, (cuuint64_t)nkv * page_size * KEY_BYTES};
    const cuuint32_t box[4] = {64, HALVES, (cuuint32_t)(page_size < OWN_CHUNK ? page_size : OWN_CHUNK), 2};
    const cuuint32_t elem[4] = {1, 1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(cache), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? RV_OK : RV_ERR_BAD_SIZE;
}

// The arguments, packed by the caller in this order (a step makes this call once a layer).
struct SharedArgs {
    const void* q; const void* cache; const int* block_tables; const int* ctx_lens; const int* plan;
    float* pre_o; float* pre_ml; float* own_o; float* own_ml; void* out; const float* sinks; const float* gate; int* status;
    cudaStream_t stream; long long num_pages;
    int num_seqs, cap_tiles, cap_items, nh, nkv, hd, page_size, max_blocks, piece, pieces, own_ctas, most_parts;
    float scale, softcap;
};

// pre_o [cap_items, nkv, SP_ROWS, HEAD_DIM], pre_ml [.., 2], own_o [pieces, num_seqs, nh, HEAD_DIM] and own_ml [.., 2] receive the parts'
// sums.  `piece`: own keys of a (sequence, kv head) that a warp takes at a time, `pieces`: the most pieces of a sequence (a longer one has
// longer ones), `own_ctas`: CTAs that take them in turn; `most_parts`: about as many parts as a row has (it decides how the merge is laid out, nothing else).
RV_EXPORT int rv_shared_attention_tcgen05(const SharedArgs* a) {
    if (a->hd != HEAD_DIM) return RV_ERR_UNSUPPORTED;
    const int nh = a->nh, nkv = a->nkv, page_size = a->page_size;
    if (a->num_seqs < 0 || nh <= 0 || nkv <= 0 || nh % nkv || page_size <= 0 || a->max_blocks <= 0 || a->num_pages <= 0 || a->cap_tiles < 0 ||
        a->cap_items < 0 || a->piece < 1 || a->pieces < 1 || a->own_ctas < 1 || !a->plan || !a->pre_o || !a->pre_ml || !a->own_o || !a->own_ml)
        return RV_ERR_BAD_SIZE;
    const int G = nh / nkv;
    if (G > SP_ROWS || (page_size & (page_size - 1)) || page_size < 8) return RV_ERR_UNSUPPORTED;
    // a row of the tensor map, a CTA and a row of the result are ints in the kernels
    const int head_blocks = (G + 7) / 8;
    const long long prefix_ctas = (long long)nkv * a->cap_items;
    if (a->num_pages > 0x7fffffffLL / 2 / nkv / page_size || prefix_ctas + a->own_ctas > 0x7fffffffLL || (long long)a->num_seqs * nh > 0x7fffffffLL ||
        (long long)a->num_seqs * a->pieces > 0x7fffffffLL / (nkv * head_blocks) || a->num_seqs > MAX_SEQS)
        return RV_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->cache) | reinterpret_cast<uintptr_t>(a->pre_o) |
         reinterpret_cast<uintptr_t>(a->own_o) | reinterpret_cast<uintptr_t>(a->plan) | reinterpret_cast<uintptr_t>(a->out)) % 16 ||
        (reinterpret_cast<uintptr_t>(a->pre_ml) | reinterpret_cast<uintptr_t>(a->own_ml)) % 8)
        return RV_ERR_ALIGNMENT;
    if (a->num_seqs == 0) return RV_OK;
    alignas(64) CUtensorMap map_kv, map_own;
    int st = rv_make_bf16_map(&map_kv, a->cache, a->num_pages * 2 * nkv * page_size, HEAD_DIM, page_size < KV_TILE ? page_size : KV_TILE);
    if (st == RV_OK) st = make_own_map(&map_own, a->cache, a->num_pages, nkv, page_size);
    if (st != RV_OK) return st;
    SharedParams p;
    p.plan = shared_plan(a->plan, a->num_seqs, a->cap_tiles);
    p.q = (const __nv_bfloat16*)a->q; p.cache = (const __nv_bfloat16*)a->cache; p.block_tables = a->block_tables; p.ctx_lens = a->ctx_lens;
    p.pre_o = a->pre_o; p.pre_ml = a->pre_ml; p.own_o = a->own_o; p.own_ml = a->own_ml; p.status = a->status;
    p.num_seqs = a->num_seqs; p.nh = nh; p.nkv = nkv; p.page_size = page_size; p.max_blocks = a->max_blocks; p.num_pages = (int)a->num_pages;
    p.prefix_ctas = (int)prefix_ctas; p.head_blocks = head_blocks; p.pieces = a->pieces; p.piece = a->piece;
    p.page_shift = 0;
    while ((1 << p.page_shift) < page_size) ++p.page_shift;
    p.scale_log2e = a->scale * 1.4426950408889634f;
    p.cap_log2e = a->softcap > 0.f ? a->softcap * 1.4426950408889634f : 0.f;
    p.scale_over_cap = a->softcap > 0.f ? a->scale / a->softcap : 0.f;
    const int smem = Q_BYTES + NK * TILE_BYTES + NV * TILE_BYTES + 256;
    static_assert(OWN_WARPS * (RING_BYTES + 8 * OWN_STAGES) + (OWN_WARPS + 1 + 3 * MAX_SEQS + 1) * 4 <= Q_BYTES + (NK + NV) * TILE_BYTES + 256,
                  "the own keys' stages and their list lie in the same shared memory");
    static_assert(STAGE_BYTES % 1024 == 0 && RING_BYTES % 1024 == 0, "the swizzle goes by address bits 7 to 9");
    static RvPerDevice configured;
    if (int e = rv_configure_smem(configured, shared_attention_kernel, smem)) return e;
    RV_LAUNCH_ST = rv_launch(shared_attention_kernel, dim3((unsigned)(prefix_ctas + a->own_ctas)), dim3(NUM_THREADS), smem, a->stream, map_kv, map_own, p);
    if ((st = rv_launch_status()) != RV_OK) return st;
    const int rows = a->num_seqs * nh, wave = MERGE_BLOCKS * rv_sm_count();
    const auto merge = [&](auto kernel, int per_block) {
        return rv_launch(kernel, dim3((rows + per_block - 1) / per_block), dim3(128), 0, a->stream, p, a->sinks, a->gate, (__nv_bfloat16*)a->out);
    };
    if (a->most_parts <= MERGE_BATCH || rows > 2 * wave) RV_LAUNCH_ST = merge(shared_merge_kernel<1>, 128 / (HEAD_DIM / 4));
    else if (rows > wave) RV_LAUNCH_ST = merge(shared_merge_kernel<2>, 2);
    else RV_LAUNCH_ST = merge(shared_merge_kernel<4>, 1);
    return rv_launch_status();
}
