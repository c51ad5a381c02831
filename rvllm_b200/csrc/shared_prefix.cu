// Attention over a prefix that sequences share: the plain kernels (any type, head size and page size) and the merge.
//
// With the keys of a sequence cut at its prefix's end, (m1, l1, o1) over the prefix and (m2, l2, o2) over what lies behind it, each
// (maximum, sum of e^(s - m), sum of e^(s - m) v), the attention is (o1 e^(m1 - m) + o2 e^(m2 - m)) / (l1 e^(m1 - m) + l2 e^(m2 - m)),
// m = max(m1, m2); cutting either part into further ranges changes nothing.  Maxima are in units of log2 throughout.
#include "common.cuh"
#include "shared_prefix.cuh"

// ---------------------------------------------------------------------------------------------
// The plain kernel of both parts: 32-bit products and sums (no tensor core takes 32 bits), both parts in one launch, the prefixes' CTAs
// first.  Arithmetic bounds it, or rather how often a word has to be read from shared memory for it: a CTA of the prefixes takes 32
// rows and 64 keys at a time, in register tiles (2.2 us a tile at the rate of the multiply-adds of an SM; a tile more a CTA takes 5); the
// rows of a sequence's own keys are few, a warp has one.  16 sequences behind 777 shared keys, 28 heads of 128 on 4: 21.3 us in a
// graph, 15.7 of them in this kernel, for 181 MFLOP (2.4 us of the GPU's multiply-adds, 4.5 MB): launches and the latencies of one tile
// per CTA.  (Before, a lane per key and a warp per four rows, both operands read once per four multiply-adds: 31.2.)
#define PLAIN_THREADS 256
#define PLAIN_TILE 32
#define PLAIN_MAX_DIM 256

struct PlainParams {
    SharedPlan plan;
    const void* q;                 // [num_seqs, nh, hd]: sequence b brings row b
    const void* cache;             // [num_pages, 2, nkv, page_size, hd]
    const int* block_tables;       // [num_seqs, max_blocks]
    const int* ctx_lens;
    float* pre_o;                  // [items, cuts, nkv, SP_ROWS, hd]: the prefixes' sums
    float* pre_ml;                 // ... and the same with 2 in place of hd
    float* own_o;                  // [splits, num_seqs, nh, hd]: those of the own keys
    float* own_ml;
    int prefix_ctas;               // kv heads x row blocks x cuts x items; behind them kv heads x blocks of eight heads x splits x sequences
    long long num_pages;
    int num_seqs, nh, nkv, hd, page_size, max_blocks;
    int row_blocks, cuts, splits;  // blocks of 32 rows of an item, its parts, and those of a sequence's own keys
    float scale, softcap;          // softcap 0: none
};

// Four elements of a tile in shared memory, which holds the cache's own type.
__device__ __forceinline__ float4 tile4(const float* at) { return *reinterpret_cast<const float4*>(at); }
__device__ __forceinline__ float4 tile4(const __nv_bfloat16* at) {
    const float2 lo = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(at)[0]), hi = __bfloat1622float2(reinterpret_cast<const __nv_bfloat162*>(at)[1]);
    return make_float4(lo.x, lo.y, hi.x, hi.y);
}
// Asks for four elements; zeros where there are none.
template <typename T>
__device__ __forceinline__ void ask4(T* to, const T* from, bool have) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;"
                 ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "n"(4 * (int)sizeof(T)), "r"(have ? 4 * (int)sizeof(T) : 0) : "memory");
}
__device__ __forceinline__ void asked() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void wait_all_but_last() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

template <int DPL> struct Tile {
    static constexpr int KEYS = DPL == 4 ? 64 : 32;            // of a tile of the prefixes: what two CTAs an SM leave room for
    static constexpr int S_STRIDE = KEYS + 8;                  // (the four rows that a warp's lanes write are 8 banks apart)
};
#define PREFIX_ROWS 32

// A range of a group's prefix against up to 32 rows.  For the scores a lane has KEYS / 16 rows x 2 keys, of the 4 x 8 lanes of a warp
// (which reads every word of its rows and keys once for 4 KEYS x 16 products), then a warp has four rows' statistics, and for the
// sums a lane has four rows x DPL columns.  Keys and values come by asynchronous copies, each while the other is worked on.
template <typename T, int DPL>
__device__ __forceinline__ void prefix_part(const PlainParams& p, float* sh, int cta) {
    constexpr int KEYS = Tile<DPL>::KEYS, S = Tile<DPL>::S_STRIDE, RR = KEYS / 16;
    const int stride = p.hd + 16 / (int)sizeof(T), q_stride = p.hd + 4;       // (16 bytes apart in the banks for hd a multiple of 32)
    float* q_s = sh;                                        // [PREFIX_ROWS][q_stride]
    float* s_s = q_s + PREFIX_ROWS * q_stride;              // [PREFIX_ROWS][S]: scores, then weights
    float* keep_s = s_s + PREFIX_ROWS * S;                  // [PREFIX_ROWS] what a row's sums so far are multiplied by
    int* lim_s = reinterpret_cast<int*>(keep_s + PREFIX_ROWS);   // [PREFIX_ROWS] keys that a row sees end here
    int* there_s = lim_s + PREFIX_ROWS;                     // [2][KEYS] whether a key's page exists, of two tiles
    T* k_s = reinterpret_cast<T*>(there_s + 2 * KEYS);      // [KEYS][stride]
    T* v_s = k_s + KEYS * stride;                           // [KEYS][stride]

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.nh / p.nkv;
    const int kvh = cta % p.nkv, row0 = cta / p.nkv % p.row_blocks * PREFIX_ROWS, which = cta / (p.nkv * p.row_blocks);
    const SharedItem item = p.plan.item(which / p.cuts);
    const int rows = min(item.count, SP_ROWS / G) * G - row0;
    if (item.key_end <= item.key_begin || rows <= 0) return;
    const int per = ((item.key_end - item.key_begin + KEYS - 1) / KEYS + p.cuts - 1) / p.cuts * KEYS;
    const int key_lo = item.key_begin + which % p.cuts * per, key_hi = min(item.key_end, key_lo + per);      // (none left: a part without keys)

    constexpr int SHARE = PLAIN_THREADS / KEYS;             // threads that bring a key
    const int mine = tid / SHARE, from = tid % SHARE * 4;
    const int* table = p.block_tables + (size_t)item.table_seq * p.max_blocks;
    auto page_of = [&](int key0) -> int {                   // of this thread's key of a tile
        const int key = key0 + mine;
        const int page = key < key_hi && key / p.page_size < p.max_blocks ? table[key / p.page_size] : -1;
        return page < p.num_pages ? page : -1;
    };
    const size_t plane = (size_t)p.nkv * p.page_size * p.hd;
    auto ask = [&](T* to, int key0, int page, size_t offset) {
        if (key0 < key_hi) {
            const T* at = reinterpret_cast<const T*>(p.cache) + offset +
                          (((size_t)max(page, 0) * 2 * p.nkv + kvh) * p.page_size + (key0 + mine) % p.page_size) * p.hd;
            for (int d = from; d < p.hd; d += 4 * SHARE) ask4(to + mine * stride + d, at + d, page >= 0);
        }
        asked();
    };
    int page = page_of(key_lo);
    ask(k_s, key_lo, page, 0);
    if (from == 0) there_s[mine] = page >= 0;
    ask(v_s, key_lo, page, plane);

    constexpr int dt = sizeof(T) == 4 ? RV_DTYPE_F32 : RV_DTYPE_BF16;
    {
        const int r = tid / 8, seq = r < rows ? p.plan.member(item.first + (row0 + r) / G) : -1;
        if (tid % 8 == 0) lim_s[r] = seq >= 0 ? min(key_hi, p.ctx_lens[seq]) : 0;
        const size_t at = ((size_t)max(seq, 0) * p.nh + kvh * G + (row0 + r) % G) * p.hd;
#pragma unroll 4
        for (int d = tid % 8 * 4; d < p.hd; d += 32) {
            const float4 v = seq >= 0 ? rv_load4(p.q, dt, at + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(q_s + r * q_stride + d) = make_float4(v.x * p.scale, v.y * p.scale, v.z * p.scale, v.w * p.scale);
        }
    }
    float m[4], l[4], acc[4][DPL];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[i][d] = 0.f;
    }
    constexpr int KEY_BLOCKS = KEYS / 16;
    const int s_row = warp / KEY_BLOCKS * (4 * RR) + lane / 8, s_key = warp % KEY_BLOCKS * 16 + lane % 8;      // and 4 i rows, 8 keys further
    const int o_row = warp % 4 * 8 + lane / 16, o_col = warp / 4 * 64 + lane % 16 * 4;                        // and 2 i rows, 128 c columns further
    int turn = 0;
    for (int key0 = key_lo; key0 < key_hi; key0 += KEYS, turn ^= 1) {
        const int next = page_of(key0 + KEYS), here = min(KEYS, key_hi - key0);
        wait_all_but_last();                                // the keys are there
        __syncthreads();
        if (warp / KEY_BLOCKS * (4 * RR) < rows && warp % KEY_BLOCKS * 16 < here) {
            float s[RR][2];
#pragma unroll
            for (int i = 0; i < RR; ++i) s[i][0] = s[i][1] = 0.f;
#pragma unroll 2
            for (int d = 0; d < p.hd; d += 4) {
                const float4 a0 = tile4(k_s + s_key * stride + d), a1 = tile4(k_s + (s_key + 8) * stride + d);
#pragma unroll
                for (int i = 0; i < RR; ++i) {
                    const float4 b = tile4(q_s + (s_row + 4 * i) * q_stride + d);
                    s[i][0] = fmaf(a0.x, b.x, s[i][0]); s[i][1] = fmaf(a1.x, b.x, s[i][1]);
                    s[i][0] = fmaf(a0.y, b.y, s[i][0]); s[i][1] = fmaf(a1.y, b.y, s[i][1]);
                    s[i][0] = fmaf(a0.z, b.z, s[i][0]); s[i][1] = fmaf(a1.z, b.z, s[i][1]);
                    s[i][0] = fmaf(a0.w, b.w, s[i][0]); s[i][1] = fmaf(a1.w, b.w, s[i][1]);
                }
            }
#pragma unroll
            for (int i = 0; i < RR; ++i) {
                s_s[(s_row + 4 * i) * S + s_key] = s[i][0];
                s_s[(s_row + 4 * i) * S + s_key + 8] = s[i][1];
            }
        }
        __syncthreads();                                    // the keys have been read
        ask(k_s, key0 + KEYS, next, 0);
        if (from == 0) there_s[(turn ^ 1) * KEYS + mine] = next >= 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = warp * 4 + i;
            if (r >= rows) break;
            float v[KEYS / 32], top = -INFINITY;
#pragma unroll
            for (int h = 0; h < KEYS / 32; ++h) {
                v[h] = s_s[r * S + 32 * h + lane];
                if (p.softcap > 0.f) v[h] = p.softcap * tanhf(v[h] / p.softcap);
                v[h] = key0 + 32 * h + lane < lim_s[r] && there_s[turn * KEYS + 32 * h + lane] ? v[h] * 1.4426950408889634f : -INFINITY;
                top = fmaxf(top, v[h]);
            }
            const float m_new = fmaxf(m[i], rv_warp_max(top));
            const float m_s = m_new == -INFINITY ? 0.f : m_new;
            const float keep = exp2f(m[i] - m_s);
            float sum = 0.f;
#pragma unroll
            for (int h = 0; h < KEYS / 32; ++h) {
                v[h] = exp2f(v[h] - m_s);
                s_s[r * S + 32 * h + lane] = v[h];
                sum += v[h];
            }
            l[i] = l[i] * keep + rv_warp_sum(sum);
            m[i] = m_new;
            if (lane == 0) keep_s[r] = keep;
        }
        wait_all_but_last();                                // the values are there
        __syncthreads();
        if (warp % 4 * 8 < rows) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float keep = keep_s[o_row + 2 * i];
#pragma unroll
                for (int d = 0; d < DPL; ++d) acc[i][d] *= keep;
            }
#pragma unroll 2
            for (int k = 0; k < here; k += 4) {         // (weights behind the last key are zeros)
                float4 w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = tile4(s_s + (o_row + 2 * i) * S + k);
#pragma unroll
                for (int c = 0; c < DPL; c += 4) {
                    const int d = o_col + c * 32;
                    if (d >= p.hd) continue;
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        const float4 v = tile4(v_s + (k + kk) * stride + d);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float e = kk == 0 ? w[i].x : kk == 1 ? w[i].y : kk == 2 ? w[i].z : w[i].w;
                            acc[i][c] = fmaf(e, v.x, acc[i][c]); acc[i][c + 1] = fmaf(e, v.y, acc[i][c + 1]);
                            acc[i][c + 2] = fmaf(e, v.z, acc[i][c + 2]); acc[i][c + 3] = fmaf(e, v.w, acc[i][c + 3]);
                        }
                    }
                }
            }
        }
        __syncthreads();                                    // the values and weights have been read
        ask(v_s, key0 + KEYS, next, plane);
    }
    const size_t out = ((size_t)which * p.nkv + kvh) * SP_ROWS + row0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = o_row + 2 * i;
#pragma unroll
        for (int c = 0; c < DPL; c += 4) {
            const int d = o_col + c * 32;
            if (r < rows && d < p.hd)
                *reinterpret_cast<float4*>(p.pre_o + (out + r) * p.hd + d) = make_float4(acc[i][c], acc[i][c + 1], acc[i][c + 2], acc[i][c + 3]);
        }
        if (lane == 0 && warp * 4 + i < rows) *reinterpret_cast<float2*>(p.pre_ml + (out + warp * 4 + i) * 2) = make_float2(m[i], l[i]);
    }
}

// A piece of the keys behind the prefix of one sequence, against up to eight of its heads: a warp has a row, its lanes the keys of the
// tile for the scores and hd / 32 columns for the sums; the next tile's words wait in registers.  Warps beyond the heads of a group only load.
template <typename T, int DPL>
__device__ __forceinline__ void own_part(const PlainParams& p, float* sh, int cta) {
    constexpr int R = PLAIN_THREADS / 32;
    const int stride = p.hd + 4;                            // (a multiple of four that is odd in units of 16 bytes for hd a multiple of 8)
    float* q_s = sh;                                        // [R][hd]
    float* k_s = q_s + R * p.hd;                            // [PLAIN_TILE][stride]
    float* v_s = k_s + PLAIN_TILE * stride;                 // [PLAIN_TILE][stride]
    float* p_s = v_s + PLAIN_TILE * stride;                 // [R][PLAIN_TILE]
    int* there_s = reinterpret_cast<int*>(p_s + R * PLAIN_TILE);   // [PLAIN_TILE] whether a key's page exists

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.nh / p.nkv;
    const int row_blocks = (G + R - 1) / R;
    const int kvh = cta % p.nkv, row0 = cta / p.nkv % row_blocks * R, which = cta / (p.nkv * row_blocks);
    const int seq = which % p.num_seqs, split = which / p.num_seqs, rows = G - row0;
    const int ctx = p.ctx_lens[seq], start = p.plan.own_start(seq);
    const int tiles = ctx > start ? (ctx - start + PLAIN_TILE - 1) / PLAIN_TILE : 0;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int key_lo = start + split * per * PLAIN_TILE, key_hi = min(ctx, key_lo + per * PLAIN_TILE);
    const size_t head = (size_t)seq * p.nh + kvh * G + row0;               // the first row's
    // an eighth of the columns of key tid / 8 (of row tid / 8) per thread
    constexpr int dt = sizeof(T) == 4 ? RV_DTYPE_F32 : RV_DTYPE_BF16;
    constexpr int SHARE = PLAIN_THREADS / PLAIN_TILE;
    const int mine = tid / SHARE, from = tid % SHARE * 4;
    if (mine < R) {
#pragma unroll 4
        for (int d = from; d < p.hd; d += 4 * SHARE) {
            const float4 v = mine < rows ? rv_load4(p.q, dt, (head + mine) * p.hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(q_s + mine * p.hd + d) = make_float4(v.x * p.scale, v.y * p.scale, v.z * p.scale, v.w * p.scale);
        }
    }
    const int* table = p.block_tables + (size_t)seq * p.max_blocks;
    auto page_of = [&](int key) -> int {
        return key < key_hi && key / p.page_size < p.max_blocks ? table[key / p.page_size] : -1;
    };
    float m = -INFINITY, l = 0.f, acc[DPL];
#pragma unroll
    for (int d = 0; d < DPL; ++d) acc[d] = 0.f;
    const size_t plane = (size_t)p.nkv * p.page_size * p.hd;
    float4 next_k[DPL], next_v[DPL];
    bool there = false;
    auto fetch = [&](int key0, int page) {
        there = page >= 0 && page < p.num_pages;
        const size_t at = (((size_t)max(page, 0) * 2 * p.nkv + kvh) * p.page_size + (key0 + mine) % p.page_size) * p.hd;
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            const int d = from + 4 * SHARE * i;
            next_k[i] = next_v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (there && d < p.hd) { next_k[i] = rv_load4(p.cache, dt, at + d); next_v[i] = rv_load4(p.cache, dt, at + plane + d); }
        }
    };
    fetch(key_lo, page_of(key_lo + mine));
    int page = page_of(key_lo + PLAIN_TILE + mine);
    for (int key0 = key_lo; key0 < key_hi; key0 += PLAIN_TILE) {
        __syncthreads();                                    // the tile before has been read
#pragma unroll
        for (int i = 0; i < DPL; ++i) {
            const int d = from + 4 * SHARE * i;
            if (d < p.hd) {
                *reinterpret_cast<float4*>(k_s + mine * stride + d) = next_k[i];
                *reinterpret_cast<float4*>(v_s + mine * stride + d) = next_v[i];
            }
        }
        if (from == 0) there_s[mine] = there;
        __syncthreads();
        fetch(key0 + PLAIN_TILE, page);
        page = page_of(key0 + 2 * PLAIN_TILE + mine);
        if (warp >= rows) continue;                         // (it brings its keys, and has no row to put them to)
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int d = 0; d < p.hd; d += 4) {
            const float4 a = tile4(k_s + lane * stride + d), b = tile4(q_s + warp * p.hd + d);
            s[0] = fmaf(a.x, b.x, s[0]); s[1] = fmaf(a.y, b.y, s[1]); s[2] = fmaf(a.z, b.z, s[2]); s[3] = fmaf(a.w, b.w, s[3]);
        }
        float v = (s[0] + s[1]) + (s[2] + s[3]);
        if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
        v = key0 + lane < key_hi && there_s[lane] ? v * 1.4426950408889634f : -INFINITY;
        const float m_new = fmaxf(m, rv_warp_max(v));
        const float m_s = m_new == -INFINITY ? 0.f : m_new;
        const float keep = exp2f(m - m_s), e = exp2f(v - m_s);
        l = l * keep + rv_warp_sum(e);
        m = m_new;
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[d] *= keep;
        p_s[warp * PLAIN_TILE + lane] = e;
        __syncwarp();
#pragma unroll 4
        for (int k = 0; k < PLAIN_TILE; ++k) {
            const float w = p_s[warp * PLAIN_TILE + k];
#pragma unroll
            for (int c = 0; c < DPL; c += 4) {
                const int d = c * 32 + lane * 4;
                if (d >= p.hd) continue;
                const float4 x = tile4(v_s + k * stride + d);
                acc[c] = fmaf(w, x.x, acc[c]); acc[c + 1] = fmaf(w, x.y, acc[c + 1]);
                acc[c + 2] = fmaf(w, x.z, acc[c + 2]); acc[c + 3] = fmaf(w, x.w, acc[c + 3]);
            }
        }
    }
    if (warp >= rows) return;
    const size_t out = (size_t)split * p.num_seqs * p.nh + head + warp;
#pragma unroll
    for (int c = 0; c < DPL; c += 4) {
        const int d = c * 32 + lane * 4;
        if (d < p.hd) *reinterpret_cast<float4*>(p.own_o + out * p.hd + d) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
    }
    if (lane == 0) *reinterpret_cast<float2*>(p.own_ml + out * 2) = make_float2(m, l);
}

template <typename T, int DPL>
__global__ void __launch_bounds__(PLAIN_THREADS, 2)
shared_plain_kernel(const PlainParams p) {
    extern __shared__ __align__(16) float sh[];
    rv_pdl_wait();
    rv_pdl_launch_dependents();                             // (only now: the merge reads the plan before it waits for this kernel)
    if ((int)blockIdx.x < p.prefix_ctas) prefix_part<T, DPL>(p, sh, blockIdx.x);
    else own_part<T, DPL>(p, sh, (int)blockIdx.x - p.prefix_ctas);
}

// Bytes of shared memory: what the larger of the two parts holds.
template <typename T, int DPL>
static int plain_bytes(int hd) {
    constexpr int KEYS = Tile<DPL>::KEYS, R = PLAIN_THREADS / 32;
    const int prefix = (PREFIX_ROWS * (hd + 4 + Tile<DPL>::S_STRIDE + 2) + 2 * KEYS) * 4 + 2 * KEYS * (hd * (int)sizeof(T) + 16);
    const int own = (R * hd + 2 * PLAIN_TILE * (hd + 4) + R * PLAIN_TILE + PLAIN_TILE) * 4;
    return prefix > own ? prefix : own;
}

template <typename T, int DPL>
static int launch_plain(const PlainParams& p, unsigned ctas, cudaStream_t stream) {
    static RvPerDevice configured;
    if (int e = rv_configure_smem(configured, shared_plain_kernel<T, DPL>, plain_bytes<T, DPL>(32 * DPL))) return e;
    RV_LAUNCH_ST = rv_launch(shared_plain_kernel<T, DPL>, dim3(ctas), dim3(PLAIN_THREADS), plain_bytes<T, DPL>(p.hd), stream, p);
    return rv_launch_status();
}

// ---------------------------------------------------------------------------------------------
// The merge: hd / 4 threads per (token, head) row, four neighbouring elements each, eight ranges' loads in flight at a time.
struct MergeParams {
    SharedPlan plan;
    const float* pre_o;            // [cap_items, cuts, nkv, SP_ROWS, hd]
    const float* pre_ml;
    const float* own_o;            // [splits, num_seqs, nh, hd]
    const float* own_ml;
    const float* sinks;            // [nh] or null
    const float* gate;             // [num_seqs, nh] or null
    void* out;                     // [num_seqs, nh, hd]
    int num_seqs, nh, nkv, hd, cuts, splits, rows_per_block;
};

template <typename T>
__global__ void __launch_bounds__(128)
shared_merge_kernel(const MergeParams p) {
    rv_pdl_launch_dependents();
    const int per = p.hd / 4;
    const int r = threadIdx.x / per, d = (threadIdx.x - r * per) * 4;
    const long long row = (long long)blockIdx.x * p.rows_per_block + r;           // (sequence, head)
    const bool live = r < p.rows_per_block && row < (long long)p.num_seqs * p.nh;
    const int seq = live ? (int)(row / p.nh) : 0, head = live ? (int)(row - (long long)seq * p.nh) : 0;
    const int G = p.nh / p.nkv, kvh = head / G;
    const int place = p.plan.place(seq);
    int2 parts = make_int2(0, 0);
    if (place >= 0) parts = p.plan.parts(place / SP_ROWS);
    rv_pdl_wait();
    if (!live) return;
    const size_t out_row = (size_t)seq * p.nh + head;
    const size_t pre_row = ((size_t)parts.x * p.cuts * p.nkv + kvh) * SP_ROWS + (place >= 0 ? place % SP_ROWS + head - kvh * G : 0);
    float m_all = -INFINITY, l_all = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    // the parts, prefix first, eight at a time
    const int from_prefix = parts.y * p.cuts, total = from_prefix + p.splits;
    for (int s0 = 0; s0 < total; s0 += 8) {
        float m[8], l[8];
        float4 o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool have = s0 + k < total;
            const int i = have ? s0 + k : total - 1;
            const bool pre = i < from_prefix;
            const size_t at = pre ? pre_row + (size_t)i * p.nkv * SP_ROWS : (size_t)(i - from_prefix) * p.num_seqs * p.nh + out_row;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(pre ? p.pre_ml : p.own_ml) + at);
            m[k] = have ? ml.x : -INFINITY;
            l[k] = have ? ml.y : 0.f;
            o[k] = __ldcg(reinterpret_cast<const float4*>((pre ? p.pre_o : p.own_o) + at * p.hd + d));
        }
        float m_new = m_all;
#pragma unroll
        for (int k = 0; k < 8; ++k) m_new = fmaxf(m_new, m[k]);
        const float m_s = m_new == -INFINITY ? 0.f : m_new;
        const float keep = exp2f(m_all - m_s);               // 0 while nothing has been seen
        l_all *= keep;
        sum.x *= keep; sum.y *= keep; sum.z *= keep; sum.w *= keep;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float f = exp2f(m[k] - m_s);               // 0 for an empty or absent part, whose sum may hold anything
            l_all += l[k] * f;
            if (f > 0.f) { sum.x += o[k].x * f; sum.y += o[k].y * f; sum.z += o[k].z * f; sum.w += o[k].w * f; }
        }
        m_all = m_new;
    }
    float num = 1.f, den = l_all;
    if (p.sinks) {                                       // exp(sink) joins the denominator; it has no value
        const float sk = p.sinks[head] * 1.4426950408889634f;
        const float m_new = fmaxf(m_all, sk);
        num = exp2f(m_all - m_new);
        den = l_all * num + exp2f(sk - m_new);
    }
    float inv = den == 0.f ? 0.f : num / den;            // (what is no number stays so)
    if (p.gate) inv *= p.gate[out_row];
    constexpr int dt = sizeof(T) == 4 ? RV_DTYPE_F32 : RV_DTYPE_BF16;
    rv_store4(p.out, dt, out_row * p.hd + d, make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv));
}

// The arguments, packed by the caller in this order (a step makes this call once a layer).
struct PlainArgs {
    const void* q; const void* cache; const int* block_tables; const int* ctx_lens; const int* plan;
    float* pre_o; float* pre_ml; float* own_o; float* own_ml; void* out; const float* sinks; const float* gate; cudaStream_t stream;
    long long num_pages;
    int num_seqs, cap_tiles, cap_items, nh, nkv, hd, page_size, max_blocks, row_blocks, cuts, splits, dtype;
    float scale, softcap;
};

// pre_o [cap_items, cuts, nkv, SP_ROWS, hd], own_o [splits, num_seqs, nh, hd] and the same with 2 in place of hd receive the parts' sums.
// `row_blocks`: of 32 rows, as many as the widest item has.
RV_EXPORT int rv_shared_attention_plain(const PlainArgs* a) {
    const int nh = a->nh, nkv = a->nkv, hd = a->hd;
    if (a->num_seqs < 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || a->page_size <= 0 || a->max_blocks <= 0 || a->num_pages <= 0 ||
        a->cap_tiles < 0 || a->cap_items <= 0 || a->row_blocks < 1 || a->cuts < 1 || a->splits < 1 || !a->plan || !a->pre_o || !a->pre_ml || !a->own_o || !a->own_ml)
        return RV_ERR_BAD_SIZE;
    if (a->dtype != RV_DTYPE_F32 && a->dtype != RV_DTYPE_BF16) return RV_ERR_BAD_DTYPE;
    if (hd % 4 || hd > PLAIN_MAX_DIM || nh / nkv > SP_ROWS) return RV_ERR_UNSUPPORTED;
    const int G = nh / nkv;
    const long long prefix_ctas = (long long)a->cap_items * a->cuts * nkv * a->row_blocks;
    const long long own_ctas = (long long)a->num_seqs * a->splits * nkv * ((G + 7) / 8);
    if (prefix_ctas + own_ctas > 0x7fffffffLL) return RV_ERR_UNSUPPORTED;       // (blocks of the launch)
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->cache) | reinterpret_cast<uintptr_t>(a->pre_o) |
         reinterpret_cast<uintptr_t>(a->own_o) | reinterpret_cast<uintptr_t>(a->plan) | reinterpret_cast<uintptr_t>(a->out)) % 16 ||
        (reinterpret_cast<uintptr_t>(a->pre_ml) | reinterpret_cast<uintptr_t>(a->own_ml)) % 8)
        return RV_ERR_ALIGNMENT;
    if (a->num_seqs == 0) return RV_OK;
    PlainParams p;
    p.plan = shared_plan(a->plan, a->num_seqs, a->cap_tiles);
    p.q = a->q; p.cache = a->cache; p.block_tables = a->block_tables; p.ctx_lens = a->ctx_lens;
    p.num_pages = a->num_pages; p.num_seqs = a->num_seqs;
    p.nh = nh; p.nkv = nkv; p.hd = hd; p.page_size = a->page_size; p.max_blocks = a->max_blocks; p.splits = a->splits; p.row_blocks = a->row_blocks; p.cuts = a->cuts;
    p.scale = a->scale; p.softcap = a->softcap;
    const bool wide = a->dtype == RV_DTYPE_F32;
    p.pre_o = a->pre_o; p.pre_ml = a->pre_ml; p.own_o = a->own_o; p.own_ml = a->own_ml; p.prefix_ctas = (int)prefix_ctas;
    const unsigned ctas = (unsigned)(prefix_ctas + own_ctas);
    int st = hd <= 128 ? (wide ? launch_plain<float, 4>(p, ctas, a->stream) : launch_plain<__nv_bfloat16, 4>(p, ctas, a->stream))
                       : (wide ? launch_plain<float, 8>(p, ctas, a->stream) : launch_plain<__nv_bfloat16, 8>(p, ctas, a->stream));
    if (st != RV_OK) return st;
    MergeParams m;
    m.plan = p.plan; m.pre_o = a->pre_o; m.pre_ml = a->pre_ml; m.own_o = a->own_o; m.own_ml = a->own_ml;
    m.sinks = a->sinks; m.gate = a->gate; m.out = a->out;
    m.num_seqs = a->num_seqs; m.nh = nh; m.nkv = nkv; m.hd = hd; m.cuts = a->cuts; m.splits = a->splits;
    m.rows_per_block = 128 / (hd / 4);
    const long long blocks = ((long long)a->num_seqs * nh + m.rows_per_block - 1) / m.rows_per_block;
    if (blocks > 0x7fffffffLL) return RV_ERR_UNSUPPORTED;
    if (wide) RV_LAUNCH_ST = rv_launch(shared_merge_kernel<float>, dim3((unsigned)blocks), dim3(128), 0, a->stream, m);
    else RV_LAUNCH_ST = rv_launch(shared_merge_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(128), 0, a->stream, m);
    return rv_launch_status();
}
