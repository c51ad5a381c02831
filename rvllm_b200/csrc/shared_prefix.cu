// Attention over a prefix that sequences share: the plain kernels (any type, head size and page size) and the merge.
//
// With the keys of a sequence cut at its prefix's end, (m1, l1, o1) over the prefix and (m2, l2, o2) over what lies behind it, each
// (maximum, sum of e^(s - m), sum of e^(s - m) v), the attention is (o1 e^(m1 - m) + o2 e^(m2 - m)) / (l1 e^(m1 - m) + l2 e^(m2 - m)),
// m = max(m1, m2); cutting either part into further ranges changes nothing.  Maxima are in units of log2 throughout.
#include "common.cuh"
#include "shared_prefix.cuh"

// ---------------------------------------------------------------------------------------------
// The plain kernel of both parts: 32-bit products and sums, one CTA per (row block, kv head, range of keys).  The rows of a CTA share
// the keys, so a tile of 32 keys and values goes to shared memory once and meets 8 * RPW rows: a warp owns RPW rows, its lanes the
// 32 keys of the tile for the scores and hd / 32 columns for the sums.  In float32 the arithmetic bounds it (no tensor core takes
// 32 bits); RPW = 4 reads five shared words per four multiply-adds each, RPW = 1 serves the few rows of one sequence.  Both parts are
// one launch, the prefixes' CTAs first.
#define PLAIN_THREADS 256
#define PLAIN_TILE 32
#define PLAIN_MAX_DIM 256

struct PlainParams {
    SharedPlan plan;
    const void* q;                 // [num_seqs, nh, hd]: sequence b brings row b
    const void* cache;             // [num_pages, 2, nkv, page_size, hd]
    const int* block_tables;       // [num_seqs, max_blocks]
    const int* ctx_lens;
    float* pre_o;                  // [items, nkv, SP_ROWS, hd]: the prefixes' sums
    float* pre_ml;                 // ... and the same with 2 in place of hd
    float* own_o;                  // [splits, num_seqs, nh, hd]: those of the own keys
    float* own_ml;
    int prefix_ctas;               // kv heads x row blocks x items; behind them kv heads x blocks of eight heads x splits x sequences
    long long num_pages;
    int num_seqs, nh, nkv, hd, page_size, max_blocks, splits;
    float scale, softcap;          // softcap 0: none
};

// OWN: the keys behind the prefix of one sequence; else a range of a group's prefix
template <typename T, int RPW, int DPL, bool OWN>
__device__ __forceinline__ void plain_part(const PlainParams& p, float* sh, int cta) {
    constexpr int R = PLAIN_THREADS / 32 * RPW;
    const int stride = p.hd + 4;                            // (a multiple of four that is odd in units of 16 bytes for hd a multiple of 8)
    float* q_s = sh;                                        // [R][hd]
    float* k_s = q_s + R * p.hd;                            // [PLAIN_TILE][stride]
    float* v_s = k_s + PLAIN_TILE * stride;                 // [PLAIN_TILE][stride]
    float* p_s = v_s + PLAIN_TILE * stride;                 // [R][PLAIN_TILE]
    int* tok_s = reinterpret_cast<int*>(p_s + R * PLAIN_TILE);   // [R] token of a row, -1 without one
    int* lim_s = tok_s + R;                                 // [R] keys that a row sees end here
    int* there_s = lim_s + R;                               // [PLAIN_TILE] whether a key's page exists

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int G = p.nh / p.nkv;
    const int row_blocks = ((OWN ? G : SP_ROWS / G * G) + R - 1) / R;
    const int kvh = cta % p.nkv, row0 = cta / p.nkv % row_blocks * R, which = cta / (p.nkv * row_blocks);
    int key_lo, key_hi, table_seq, rows, first = 0;
    if (OWN) {
        table_seq = which % p.num_seqs;
        rows = G;
        const int ctx = p.ctx_lens[table_seq], start = p.plan.own_start(table_seq);
        const int tiles = ctx > start ? (ctx - start + PLAIN_TILE - 1) / PLAIN_TILE : 0;
        const int per = (tiles + p.splits - 1) / p.splits;
        key_lo = start + which / p.num_seqs * per * PLAIN_TILE;
        key_hi = min(ctx, key_lo + per * PLAIN_TILE);
    } else {
        const SharedItem tile = p.plan.item(which);
        table_seq = tile.table_seq; first = tile.first;
        rows = min(tile.count, SP_ROWS / G) * G;
        key_lo = tile.key_begin; key_hi = tile.key_end;
        if (key_hi <= key_lo) return;
    }
    if (row0 >= rows) return;
    if (tid < R) {
        int tok = -1, lim = 0;
        if (row0 + tid < rows) {
            const int seq = OWN ? table_seq : p.plan.member(first + (row0 + tid) / G);
            tok = seq;
            lim = min(key_hi, p.ctx_lens[seq]);
        }
        tok_s[tid] = tok; lim_s[tid] = lim;
    }
    __syncthreads();
    // an eighth of the columns of key tid / 8 (of row tid / 8) per thread
    constexpr int dt = sizeof(T) == 4 ? RV_DTYPE_F32 : RV_DTYPE_BF16;
    constexpr int SHARE = PLAIN_THREADS / PLAIN_TILE;
    const int mine = tid / SHARE, from = tid % SHARE * 4;
    if (mine < R) {
        const int tok = tok_s[mine];
        const size_t at = ((size_t)max(tok, 0) * p.nh + kvh * G + (row0 + mine) % G) * p.hd;
#pragma unroll 4
        for (int d = from; d < p.hd; d += 4 * SHARE) {
            const float4 v = rv_load4(p.q, dt, at + d);
            *reinterpret_cast<float4*>(q_s + mine * p.hd + d) =
                tok >= 0 ? make_float4(v.x * p.scale, v.y * p.scale, v.z * p.scale, v.w * p.scale) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    }
    const int* table = p.block_tables + (size_t)table_seq * p.max_blocks;
    auto page_of = [&](int key) -> int {
        return key < key_hi && key / p.page_size < p.max_blocks ? table[key / p.page_size] : -1;
    };
    float m[RPW], l[RPW], acc[RPW][DPL];
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[i][d] = 0.f;
    }
    const size_t plane = (size_t)p.nkv * p.page_size * p.hd;
    // the next tile's words wait in registers while this one is worked on
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
        float s[RPW];
#pragma unroll
        for (int i = 0; i < RPW; ++i) s[i] = 0.f;
#pragma unroll 4
        for (int d = 0; d < p.hd; d += 4) {
            const float4 a = *reinterpret_cast<const float4*>(k_s + lane * stride + d);
#pragma unroll
            for (int i = 0; i < RPW; ++i) {
                const float4 b = *reinterpret_cast<const float4*>(q_s + (warp * RPW + i) * p.hd + d);
                s[i] = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, s[i]))));
            }
        }
#pragma unroll
        for (int i = 0; i < RPW; ++i) {
            const int r = warp * RPW + i;
            float v = s[i];
            if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
            v = key0 + lane < lim_s[r] && there_s[lane] ? v * 1.4426950408889634f : -INFINITY;
            const float m_new = fmaxf(m[i], rv_warp_max(v));
            const float m_s = m_new == -INFINITY ? 0.f : m_new;
            const float keep = exp2f(m[i] - m_s), e = exp2f(v - m_s);
            l[i] = l[i] * keep + rv_warp_sum(e);
            m[i] = m_new;
#pragma unroll
            for (int d = 0; d < DPL; ++d) acc[i][d] *= keep;
            p_s[r * PLAIN_TILE + lane] = e;
        }
        __syncwarp();
#pragma unroll 4
        for (int k = 0; k < PLAIN_TILE; ++k) {
#pragma unroll
            for (int c = 0; c < DPL; c += 4) {
                const int d = c * 32 + lane * 4;
                if (d >= p.hd) continue;
                const float4 v = *reinterpret_cast<const float4*>(v_s + k * stride + d);
#pragma unroll
                for (int i = 0; i < RPW; ++i) {
                    const float e = p_s[(warp * RPW + i) * PLAIN_TILE + k];
                    acc[i][c] = fmaf(e, v.x, acc[i][c]); acc[i][c + 1] = fmaf(e, v.y, acc[i][c + 1]);
                    acc[i][c + 2] = fmaf(e, v.z, acc[i][c + 2]); acc[i][c + 3] = fmaf(e, v.w, acc[i][c + 3]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RPW; ++i) {
        const int r = warp * RPW + i;
        if (row0 + r >= rows || tok_s[r] < 0) continue;
        const size_t prow = OWN ? ((size_t)(which / p.num_seqs) * p.num_seqs + tok_s[r]) * p.nh + kvh * G + row0 + r
                                : ((size_t)which * p.nkv + kvh) * SP_ROWS + row0 + r;
        float* sums = (OWN ? p.own_o : p.pre_o) + prow * p.hd;
#pragma unroll
        for (int c = 0; c < DPL; c += 4) {
            const int d = c * 32 + lane * 4;
            if (d < p.hd) *reinterpret_cast<float4*>(sums + d) = make_float4(acc[i][c], acc[i][c + 1], acc[i][c + 2], acc[i][c + 3]);
        }
        if (lane == 0) *reinterpret_cast<float2*>((OWN ? p.own_ml : p.pre_ml) + prow * 2) = make_float2(m[i], l[i]);
    }
}

template <typename T, int DPL>
__global__ void __launch_bounds__(PLAIN_THREADS)
shared_plain_kernel(const PlainParams p) {
    extern __shared__ __align__(16) float sh[];
    rv_pdl_launch_dependents();
    rv_pdl_wait();
    if ((int)blockIdx.x < p.prefix_ctas) plain_part<T, 4, DPL, false>(p, sh, blockIdx.x);
    else plain_part<T, 1, DPL, true>(p, sh, (int)blockIdx.x - p.prefix_ctas);
}

template <typename T, int DPL>
static int launch_plain(const PlainParams& p, unsigned ctas, cudaStream_t stream) {
    constexpr int R = PLAIN_THREADS / 32 * 4;
    const auto bytes = [](int hd) { return (R * hd + 2 * PLAIN_TILE * (hd + 4) + R * PLAIN_TILE + 2 * R + PLAIN_TILE) * 4; };
    static RvPerDevice configured;
    if (int e = rv_configure_smem(configured, shared_plain_kernel<T, DPL>, bytes(PLAIN_MAX_DIM))) return e;
    RV_LAUNCH_ST = rv_launch(shared_plain_kernel<T, DPL>, dim3(ctas), dim3(PLAIN_THREADS), bytes(p.hd), stream, p);
    return rv_launch_status();
}

// ---------------------------------------------------------------------------------------------
// The merge: hd / 4 threads per (token, head) row, four neighbouring elements each, eight ranges' loads in flight at a time.
struct MergeParams {
    SharedPlan plan;
    const float* pre_o;            // [cap_items, nkv, SP_ROWS, hd]
    const float* pre_ml;
    const float* own_o;            // [splits, num_seqs, nh, hd]
    const float* own_ml;
    const float* sinks;            // [nh] or null
    const float* gate;             // [num_seqs, nh] or null
    void* out;                     // [num_seqs, nh, hd]
    int num_seqs, nh, nkv, hd, splits, rows_per_block;
};

struct Running {
    float m, l;
    float4 o;
};

// Takes up `n` ranges, `step` rows apart from `row` on.
__device__ __forceinline__ void merge_ranges(Running& r, const float* __restrict__ part_o, const float* __restrict__ part_ml, size_t row,
                                             size_t step, int n, int hd, int d) {
    for (int s0 = 0; s0 < n; s0 += 8) {
        float m[8], l[8];
        float4 o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool have = s0 + i < n;
            const size_t at = row + (size_t)(have ? s0 + i : s0) * step;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_ml) + at);
            m[i] = have ? ml.x : -INFINITY;
            l[i] = have ? ml.y : 0.f;
            o[i] = __ldcg(reinterpret_cast<const float4*>(part_o + at * hd + d));
        }
        float m_new = r.m;
#pragma unroll
        for (int i = 0; i < 8; ++i) m_new = fmaxf(m_new, m[i]);
        const float m_s = m_new == -INFINITY ? 0.f : m_new;
        const float keep = exp2f(r.m - m_s);             // 0 while nothing has been seen
        r.l *= keep;
        r.o.x *= keep; r.o.y *= keep; r.o.z *= keep; r.o.w *= keep;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float f = exp2f(m[i] - m_s);           // 0 for an empty or absent range, whose sum may hold anything
            r.l += l[i] * f;
            if (f > 0.f) { r.o.x += o[i].x * f; r.o.y += o[i].y * f; r.o.z += o[i].z * f; r.o.w += o[i].w * f; }
        }
        r.m = m_new;
    }
}

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
    rv_pdl_wait();
    if (!live) return;
    Running v;
    v.m = -INFINITY; v.l = 0.f; v.o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int place = p.plan.place(seq);
    if (place >= 0) {
        const int2 parts = p.plan.parts(place / SP_ROWS);
        merge_ranges(v, p.pre_o, p.pre_ml, ((size_t)parts.x * p.nkv + kvh) * SP_ROWS + place % SP_ROWS + (head - kvh * G),
                     (size_t)p.nkv * SP_ROWS, parts.y, p.hd, d);
    }
    const size_t out_row = (size_t)seq * p.nh + head;
    merge_ranges(v, p.own_o, p.own_ml, out_row, (size_t)p.num_seqs * p.nh, p.splits, p.hd, d);
    float num = 1.f, den = v.l;
    if (p.sinks) {                                       // exp(sink) joins the denominator; it has no value
        const float sk = p.sinks[head] * 1.4426950408889634f;
        const float m_new = fmaxf(v.m, sk);
        num = exp2f(v.m - m_new);
        den = v.l * num + exp2f(sk - m_new);
    }
    float inv = den == 0.f ? 0.f : num / den;            // (what is no number stays so)
    if (p.gate) inv *= p.gate[out_row];
    constexpr int dt = sizeof(T) == 4 ? RV_DTYPE_F32 : RV_DTYPE_BF16;
    rv_store4(p.out, dt, out_row * p.hd + d, make_float4(v.o.x * inv, v.o.y * inv, v.o.z * inv, v.o.w * inv));
}

// The arguments, packed by the caller in this order (a step makes this call once a layer).
struct PlainArgs {
    const void* q; const void* cache; const int* block_tables; const int* ctx_lens; const int* plan;
    float* pre_o; float* pre_ml; float* own_o; float* own_ml; void* out; const float* sinks; const float* gate; cudaStream_t stream;
    long long num_pages;
    int num_seqs, cap_tiles, cap_items, nh, nkv, hd, page_size, max_blocks, splits, dtype;
    float scale, softcap;
};

// pre_o [cap_items, nkv, SP_ROWS, hd], own_o [splits, num_seqs, nh, hd] and the same with 2 in place of hd receive the parts' sums.
RV_EXPORT int rv_shared_attention_plain(const PlainArgs* a) {
    const int nh = a->nh, nkv = a->nkv, hd = a->hd;
    if (a->num_seqs < 0 || nh <= 0 || nkv <= 0 || nh % nkv || hd <= 0 || a->page_size <= 0 || a->max_blocks <= 0 || a->num_pages <= 0 ||
        a->cap_tiles < 0 || a->cap_items <= 0 || a->splits < 1 || !a->plan || !a->pre_o || !a->pre_ml || !a->own_o || !a->own_ml)
        return RV_ERR_BAD_SIZE;
    if (a->dtype != RV_DTYPE_F32 && a->dtype != RV_DTYPE_BF16) return RV_ERR_BAD_DTYPE;
    if (hd % 4 || hd > PLAIN_MAX_DIM || nh / nkv > SP_ROWS) return RV_ERR_UNSUPPORTED;
    const int G = nh / nkv;
    const long long prefix_ctas = (long long)a->cap_items * nkv * ((SP_ROWS / G * G + 31) / 32);
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
    p.nh = nh; p.nkv = nkv; p.hd = hd; p.page_size = a->page_size; p.max_blocks = a->max_blocks; p.splits = a->splits;
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
    m.num_seqs = a->num_seqs; m.nh = nh; m.nkv = nkv; m.hd = hd; m.splits = a->splits;
    m.rows_per_block = 128 / (hd / 4);
    const long long blocks = ((long long)a->num_seqs * nh + m.rows_per_block - 1) / m.rows_per_block;
    if (blocks > 0x7fffffffLL) return RV_ERR_UNSUPPORTED;
    if (wide) RV_LAUNCH_ST = rv_launch(shared_merge_kernel<float>, dim3((unsigned)blocks), dim3(128), 0, a->stream, m);
    else RV_LAUNCH_ST = rv_launch(shared_merge_kernel<__nv_bfloat16>, dim3((unsigned)blocks), dim3(128), 0, a->stream, m);
    return rv_launch_status();
}
