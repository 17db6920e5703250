// Attention over listed blocks, backward.  With p_ij = exp(scale q_i.k_j - lse_i) again (nothing of the forward is kept
// but o and lse) and delta_i = do_i.o_i:
//
//   ds_ij = p_ij (do_i.v_j - delta_i) scale,   dq_i = sum_j ds_ij k_j,   dk_j = sum_i ds_ij q_i,   dv_j = sum_i p_ij do_i
//
// dq walks the lists as the forward does.  dk and dv need, for every block of keys, the query blocks that list it: the
// lists are turned over into one bit per (block of keys, query block), so that every block of keys is one work item that
// sums over its queries in ascending order and writes its rows once.  No atomics on gradients: the same inputs give the
// same bits.  A block that very many queries list (the first one often is on every list) is cut into items of `chunk`
// query blocks each, whose float partial sums a last kernel adds up in order.
//
// p and ds are rounded to the type for their products.  bf16 has float's range; half loses digits below 2^-14, where ds lies
// for output gradients of 1e-3 already (4096 keys of like weight and output gradients of 1e-4: every digit), so half's
// operands are multiplied by powers of two on the way, which the float results are divided by: p by 2^10 (p <= 1, but for scores
// so large, from 10^7 on, that their float error is felt in p: room for 2^6), ds without its scale by the 2^n that brings its
// bound, twice the longest do times the longest v (o_i is a mean of rows of v), near half's largest numbers.
#include <type_traits>
#include "attn_tc.cuh"

namespace spamm {

constexpr int TK_MAX_CHUNK = 640;            // query blocks of a work item: their list lies in what the tiles leave of shared memory

struct BackwardPlan {
    int nqb, nkb, words;        // query blocks, blocks of keys, 32-bit words of a block's bits
    int chunk;                  // query blocks of a work item
    int item_cap, slot_cap;     // items and partial sums of one (sequence, key head)
    int64_t groups;             // batch * kv_heads
    FastDiv per, G;             // rows of a full query block, heads of a key head
    int box_tokens;             // queries of a tensor copy of q and do (0: rows are copied one by one)
    int64_t n_norms;            // blocks of threads of attn_delta_kernel
    size_t delta, bits, counts, slots, items, n_items, partial, norms, factor, bytes;   // scratch offsets (the last two: half)
};

struct Item {
    int kb, chunk, slot, pad;   // block of keys, which chunk of its query blocks, partial sum to write (-1: the rows)
};

// A plan counts the rows of a query block in 32 bits.
static bool backward_fits(const spamm_attn &a)
{
    return (int64_t)min(a.query_block, a.max_q) * (a.heads / a.kv_heads) <= (1 << 28);
}

static BackwardPlan backward_plan(const spamm_attn &a)
{
    BackwardPlan p;
    const int G = a.heads / a.kv_heads;
    p.nqb = attn_query_blocks(a);
    p.nkb = ceil_div(a.max_q, a.block);
    p.words = ceil_div(p.nqb, 32);
    const int64_t rows = (int64_t)min(a.query_block, a.max_q) * G;
    p.chunk = (int)max((int64_t)1, min((int64_t)TK_MAX_CHUNK, 8192 / rows));
    p.per = fast_div((uint32_t)rows);
    p.G = fast_div((uint32_t)G);
    // a tensor copy takes the heads of a key head of as many queries as fit a tile or make up a query block, when that
    // cuts tiles of 128 rows evenly and begins on a group of 8 rows
    const int64_t fit = G <= 128 && 128 % G == 0 ? min((int64_t)min(a.query_block, a.max_q), (int64_t)128 / G) : 0;
    p.box_tokens = fit && 128 % (fit * G) == 0 && fit * G % 8 == 0 && min(a.query_block, a.max_q) % fit == 0 ? (int)fit : 0;
    const int64_t pairs = (int64_t)p.nqb * min(a.n_select, p.nkb);
    p.item_cap = (int)min((int64_t)INT32_MAX / 4, p.nkb + pairs / p.chunk);
    p.slot_cap = (int)min((int64_t)INT32_MAX / 4, 2 * pairs / p.chunk);
    p.groups = (int64_t)a.batch * a.kv_heads;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t o = at; at += (n + 255) / 256 * 256; return o; };
    p.delta = take((size_t)a.tokens * a.heads * 4);
    p.bits = take((size_t)p.groups * p.nkb * p.words * 4);          // bits and counts lie together: attn_delta_kernel clears them
    p.counts = take((size_t)p.groups * p.nkb * 4);
    p.slots = take((size_t)p.groups * p.nkb * 4);
    p.items = take((size_t)p.groups * p.item_cap * sizeof(Item));
    p.n_items = take((size_t)p.groups * 4);
    p.partial = take((size_t)p.groups * p.slot_cap * a.block * a.dim * 2 * 4);
    const bool half = a.dtype == SPAMM_ATTN_HALF;
    p.n_norms = ((int64_t)a.tokens * a.heads + 31) / 32;
    p.norms = take(half ? (size_t)p.n_norms * sizeof(float2) : 0);
    p.factor = take(half ? 4 : 0);
    p.bytes = at;
    return p;
}

// delta = do.o for every row; a quarter of a warp for each.  Rows of no sequence get zero gradients here, and the bits and
// counts of the lists that are turned over next are cleared (`clear`, one launch less).  For half every block of threads leaves
// the largest squared norms of its rows of do and of v.  (Rows with infinities and NaN do not count: what meets them is not
// finite in any case.)  Bound by the reading of do, o and the low part of o: 18000 tokens of 32 heads of 128 (440 MB) take
// 66 us, 6.7 TB/s; half with the norms 5196 tokens (128 MB) 24.5 us, 5.2 TB/s (22 us without).
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_delta_kernel(const __grid_constant__ spamm_attn a, FastDiv div_heads, FastDiv div_g, const T *d_do,
                                                         int64_t do_token, int64_t do_head, float *delta, T *dq, T *dk, T *dv,
                                                         uint4 *clear, size_t n_clear, float2 *norms)
{
    constexpr bool HALF = std::is_same<T, __half>::value;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n_clear; i += (size_t)gridDim.x * 256) clear[i] = make_uint4(0, 0, 0, 0);
    const int sub = threadIdx.x & 7;
    const int64_t w = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
    const bool there = w < (int64_t)a.tokens * a.heads;
    const int row = w <= INT32_MAX ? (int)div_heads.quotient((uint32_t)w) : (int)(w / a.heads), head = (int)(w - (int64_t)row * a.heads);
    const int h = (int)div_g.quotient(head);
    const bool first = head == h * (int)div_g.d;      // of the heads of its key head
    bool held = false;
    if (there) {
        // the sequence that holds the row
        int lo = 0, hi = a.batch;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (a.d_cu[mid + 1] > row) hi = mid; else lo = mid + 1;
        }
        if (lo < a.batch) {
            const Seq sq = attn_seq(a, lo);
            held = row >= sq.row0 && row < sq.row0 + sq.nq;
        }
    }
    if (there && !held) {
        const uint4 z = make_uint4(0, 0, 0, 0);
        for (int c = sub; c < D / 8; c += 8) {
            reinterpret_cast<uint4 *>(dq + ((int64_t)row * a.heads + head) * D)[c] = z;
            if (first) {
                reinterpret_cast<uint4 *>(dk + ((int64_t)row * a.kv_heads + h) * D)[c] = z;
                reinterpret_cast<uint4 *>(dv + ((int64_t)row * a.kv_heads + h) * D)[c] = z;
            }
        }
    }
    float sum = 0.f, norm_do = 0.f, norm_v = 0.f;
    if (held) {
#pragma unroll
        for (int c = 0; c < D / 64; c++) {
            const int d = (c * 8 + sub) * 8;
            const uint4 x = *reinterpret_cast<const uint4 *>(d_do + row * do_token + head * do_head + d);
            const uint4 y = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.d_o) + row * a.o_token + head * a.o_head + d);
            uint4 z = make_uint4(0, 0, 0, 0), k = z;
            if (a.d_o_low) z = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.d_o_low) + w * D + d);
            if (HALF && first) k = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.d_v) + row * a.v_token + h * a.v_head + d);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, ks[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 u = Pack<T>::to2(xs[i]);
                float2 v = Pack<T>::to2(ys[i]);
                if (a.d_o_low) {
                    const float2 w = Pack<T>::to2(reinterpret_cast<const uint32_t *>(&z)[i]);
                    v.x += w.x;
                    v.y += w.y;
                }
                sum = fmaf(u.x, v.x, fmaf(u.y, v.y, sum));
                if constexpr (HALF) {
                    norm_do = fmaf(u.x, u.x, fmaf(u.y, u.y, norm_do));
                    if (first) {
                        const float2 t = Pack<T>::to2(ks[i]);
                        norm_v = fmaf(t.x, t.x, fmaf(t.y, t.y, norm_v));
                    }
                }
            }
        }
    }
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) sum += __shfl_xor_sync(~0u, sum, d, 8);
    if (held && sub == 0) delta[w] = sum;
    if constexpr (HALF) {
        __shared__ uint2 met[8];
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) {
            norm_do += __shfl_xor_sync(~0u, norm_do, d, 8);
            norm_v += __shfl_xor_sync(~0u, norm_v, d, 8);
        }
        // floats from zero on are in the order of their bits
        const uint32_t x = __reduce_max_sync(~0u, isfinite(norm_do) ? __float_as_uint(norm_do) : 0u);
        const uint32_t y = __reduce_max_sync(~0u, isfinite(norm_v) ? __float_as_uint(norm_v) : 0u);
        if ((threadIdx.x & 31) == 0) met[threadIdx.x >> 5] = make_uint2(x, y);
        __syncthreads();
        if (threadIdx.x < 8) {
            const uint2 m = met[threadIdx.x];
            const uint32_t most_do = __reduce_max_sync(0xffu, m.x), most_v = __reduce_max_sync(0xffu, m.y);
            if (threadIdx.x == 0) norms[blockIdx.x] = make_float2(__uint_as_float(most_do), __uint_as_float(most_v));
        }
    }
}

// What half's ds is multiplied by: the power of two that brings its bound, 2 |do| |v|, to 2^13 .. 2^14, from the largest squared
// norms.
static __device__ float ds_factor(float norm_do, float norm_v)
{
    const float bound = 2.f * sqrtf(norm_do) * sqrtf(norm_v);
    int e = 14;
    if (bound > 0.f) frexpf(bound, &e);               // bound < 2^e
    return ldexpf(1.f, 14 - e);
}
constexpr float P_UP = 10.f, P_DOWN = 0x1p-10f;       // log2 of what half's p is multiplied by, and what takes it back

// How ds enters its products and what their results are multiplied by.
struct DsScale { float in, out; };
template <typename T> static __device__ __forceinline__ DsScale ds_scale(const spamm_attn &a, const float *factor)
{
    if constexpr (std::is_same<T, __half>::value) return {*factor, a.scale / *factor};
    else return {a.scale, 1.f};
}

// Turns the lists over: one warp reads a list and sets the bit of its query block in every listed block of keys.  (The bits and
// counts do not depend on the order of the atomics.)  5 us for query blocks of 64; one list for each of 5000 queries and 2 key
// heads 16 us, the atomics of the blocks that all of them list.
__global__ __launch_bounds__(128) void attn_turn_kernel(const __grid_constant__ spamm_attn a, int nqb, int nkb, int words,
                                                        unsigned *bits, int *counts)
{
    __shared__ int lists[4][SPAMM_ATTN_MAX_SELECT];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t w = (int64_t)blockIdx.x * 4 + warp;
    if (w >= (int64_t)a.batch * nqb * a.kv_heads) return;
    const int h = (int)(w % a.kv_heads), qb = (int)(w / a.kv_heads % nqb), s = (int)(w / a.kv_heads / nqb);
    const Seq sq = attn_seq(a, s);
    const int last = min((int)min((int64_t)(qb + 1) * a.query_block, (int64_t)sq.nq), sq.nq) - 1;
    if ((int64_t)qb * a.query_block >= sq.nq) return;
    const int blocks = ceil_div(attn_limit(a, sq, last), a.block);
    const int n = attn_load_list(a, s, qb, nqb, h, blocks, blocks, lists[warp], lane);
    const int64_t group = (int64_t)s * a.kv_heads + h;
    for (int i = lane; i < n; i += 32) {
        const int64_t at = group * nkb + lists[warp][i];
        atomicOr(bits + at * words + (qb >> 5), 1u << (qb & 31));
        atomicAdd(counts + at, 1);
    }
}

// The work items of one (sequence, key head), in the order of the blocks: a running sum over the blocks of how many
// items and partial sums each needs.  The first block of threads also takes the factor of half's ds from `norms`.
__global__ __launch_bounds__(1024) void attn_items_kernel(const __grid_constant__ spamm_attn a, const BackwardPlan p,
                                                          const int *counts, int *slots, Item *items, int *n_items,
                                                          const float2 *norms, float *factor)
{
    __shared__ int2 warp_sum[32];
    __shared__ int2 carry;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t group = blockIdx.x;
    const int s = (int)(group / a.kv_heads);
    const int n_blocks = ceil_div(attn_seq(a, s).nk, a.block);
    if (norms && blockIdx.x == 0) {
        float2 most = make_float2(0.f, 0.f);
        for (int64_t i = tid; i < p.n_norms; i += 1024) most = make_float2(fmaxf(most.x, norms[i].x), fmaxf(most.y, norms[i].y));
        const uint32_t x = __reduce_max_sync(~0u, __float_as_uint(most.x)), y = __reduce_max_sync(~0u, __float_as_uint(most.y));
        if (lane == 0) warp_sum[warp] = make_int2((int)x, (int)y);
        __syncthreads();
        if (warp == 0) {
            const int2 m = warp_sum[lane];
            const uint32_t most_do = __reduce_max_sync(~0u, (uint32_t)m.x), most_v = __reduce_max_sync(~0u, (uint32_t)m.y);
            if (lane == 0) *factor = ds_factor(__uint_as_float(most_do), __uint_as_float(most_v));
        }
    }
    if (tid == 0) carry = make_int2(0, 0);
    __syncthreads();
    for (int b0 = 0; b0 < n_blocks; b0 += 1024) {
        const int b = b0 + tid;
        const int n = b < n_blocks ? counts[group * p.nkb + b] : 0;
        const int chunks = b < n_blocks ? max(1, ceil_div(n, p.chunk)) : 0;
        int x = chunks, y = chunks > 1 ? chunks : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(~0u, x, d), v = __shfl_up_sync(~0u, y, d);
            if (lane >= d) { x += u; y += v; }
        }
        if (lane == 31) warp_sum[warp] = make_int2(x, y);
        __syncthreads();
        if (warp == 0) {
            int2 t = warp_sum[lane];
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u = __shfl_up_sync(~0u, t.x, d), v = __shfl_up_sync(~0u, t.y, d);
                if (lane >= d) { t.x += u; t.y += v; }
            }
            warp_sum[lane] = t;
        }
        __syncthreads();
        const int2 c = carry, before = warp ? warp_sum[warp - 1] : make_int2(0, 0);
        int at = c.x + before.x + x - chunks, slot = c.y + before.y + y - (chunks > 1 ? chunks : 0);
        if (b < n_blocks) {
            slots[group * p.nkb + b] = slot;
            for (int i = 0; i < chunks; i++)
                if (at + i < p.item_cap) items[group * p.item_cap + at + i] = Item{b, i, chunks > 1 ? slot + i : -1, 0};
        }
        __syncthreads();
        if (tid == 0) carry = make_int2(c.x + warp_sum[31].x, c.y + warp_sum[31].y);
        __syncthreads();
    }
    if (tid == 0) n_items[group] = min(carry.x, p.item_cap);
}

// Whether no ds of a row is finite in any case.
static __device__ __forceinline__ bool no_finite_ds(float lse, float delta)
{
    return lse != lse || (not_finite(__float_as_uint(delta)) && lse != -CUDART_INF_F);
}

// dq of one row over its own keys alone, by one warp: y[0 .. D/32).
template <typename T, int D, typename Block>
static __device__ __forceinline__ void dq_row(const spamm_attn &a, const Seq &sq, int s, int h, int query, int head, const T *d_do,
                                              int64_t do_token, int64_t do_head, const float *delta, int n, Block block, int lane, float *y)
{
    const int64_t row = sq.row0 + query, at = row * a.heads + head;
    const float lse = a.d_lse[at], dl = delta[at], minus_lse = lse == -CUDART_INF_F ? -CUDART_INF_F : -lse * LOG2E;
    float q[D / 32], g[D / 32], k[D / 32], v[D / 32];
    row_load<T, D>(static_cast<const T *>(a.d_q) + row * a.q_token + head * a.q_head, lane, q);
    row_load<T, D>(d_do + row * do_token + head * do_head, lane, g);
    row_keys<T>(a, sq, s, h, n, attn_limit(a, sq, query), block, [&](const T *kr, const T *vr) {
        row_load<T, D>(kr, lane, k);
        row_load<T, D>(vr, lane, v);
        const float p = fast_exp2(fmaf(row_dot<D>(q, k), a.scale * LOG2E, minus_lse));
        const float ds = p * (row_dot<D>(g, v) - dl) * a.scale;
#pragma unroll
        for (int i = 0; i < D / 32; i++) y[i] = fmaf(ds, k[i], y[i]);
    });
}

constexpr int DQ_STAGES = 3;
constexpr int DQ_WARPS = 4;

// dq of 16 rows (queries x heads) of one key head; the layout of attn_rows_kernel.  64 sequences of 16 rows, 8 key heads of 128,
// lists of up to 16 blocks of 64: 13 us (26 us in tiles of 128 rows).
template <typename T, int D>
__global__ __launch_bounds__(128) void attn_dq_rows_kernel(const __grid_constant__ spamm_attn a, int nqb, int tiles, const T *d_do,
                                                           int64_t do_token, int64_t do_head, const float *delta, const float *factor,
                                                           T *dq)
{
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int TILE16 = 16 * D * 2;
    uint8_t *ring = smem;
    uint8_t *q_tile = ring + DQ_WARPS * DQ_STAGES * 2 * TILE16;
    uint8_t *do_tile = q_tile + TILE16;
    int *blk = reinterpret_cast<int *>(do_tile + TILE16);
    __shared__ int shared_count;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned idx = blockIdx.x;
    const int tile = idx % tiles; idx /= tiles;
    const int qb = idx % nqb; idx /= nqb;
    const int h = idx % a.kv_heads;
    const int s = idx / a.kv_heads;
    const int G = a.heads / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    const int bq = min(a.query_block, a.max_q);
    const int n_tok = min(bq, sq.nq - qb * bq);
    const int64_t n_rows = (int64_t)max(n_tok, 0) * G;
    if ((int64_t)tile * 16 >= n_rows) return;
    const int rows = (int)min((int64_t)16, n_rows - tile * 16);
    const int first_query = qb * bq + tile * 16 / G, last_query = qb * bq + (tile * 16 + rows - 1) / G;
    const int limit_max = attn_limit(a, sq, last_query), limit_min = attn_limit(a, sq, first_query);

    for (int i = tid; i < 16 * D / 8; i += 128) {
        const int r = i / (D / 8), c = i % (D / 8);
        const int x = tile * 16 + r;
        const bool ok = r < rows;
        const int64_t row = sq.row0 + qb * bq + (int64_t)(ok ? x / G : 0), head = h * G + (ok ? x % G : 0);
        cp_async16(smem_addr(q_tile) + tile_off<D>(r, c), static_cast<const T *>(a.d_q) + row * a.q_token + head * a.q_head + c * 8, ok);
        cp_async16(smem_addr(do_tile) + tile_off<D>(r, c), d_do + row * do_token + head * do_head + c * 8, ok);
    }
    cp_commit();
    if (warp == 0) {
        const int all_blocks = ceil_div(attn_limit(a, sq, qb * bq + n_tok - 1), a.block);
        const int n = attn_load_list(a, s, qb, nqb, h, all_blocks, ceil_div(limit_max, a.block), blk, lane);
        if (lane == 0) shared_count = n;
    }
    __syncthreads();
    const int chunks_per_block = a.block >> 4;
    const int n_chunks = shared_count * chunks_per_block;
    const uint32_t my_ring = smem_addr(ring) + warp * DQ_STAGES * 2 * TILE16;

    auto issue = [&](int c, int stage) {
        if (c < n_chunks) {
            const int e = c / chunks_per_block;
            const int pos = blk[e] * a.block + (c - e * chunks_per_block) * 16;
            const int n = min(16, limit_max - pos);
            const T *kp = static_cast<const T *>(a.d_k) + (int64_t)(sq.row0 + pos) * a.k_token + h * a.k_head;
            const T *vp = static_cast<const T *>(a.d_v) + (int64_t)(sq.row0 + pos) * a.v_token + h * a.v_head;
            const uint32_t kt = my_ring + stage * 2 * TILE16, vt = kt + TILE16;
#pragma unroll
            for (int i = 0; i < 16 * D / 8 / 32; i++) {
                const int x = i * 32 + lane, r = x / (D / 8), c8 = x % (D / 8);
                const bool ok = r < n;
                cp_async16(kt + tile_off<D>(r, c8), (ok ? kp + r * a.k_token : static_cast<const T *>(a.d_k)) + c8 * 8, ok);
                cp_async16(vt + tile_off<D>(r, c8), (ok ? vp + r * a.v_token : static_cast<const T *>(a.d_v)) + c8 * 8, ok);
            }
        }
        cp_commit();
    };
    for (int i = 0; i < DQ_STAGES - 1; i++) issue(warp + DQ_WARPS * i, i);
    cp_wait<DQ_STAGES - 1>();
    __syncthreads();
    uint32_t qf[D / 16][4], df[D / 16][4];
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) {
        a_frag<D>(smem_addr(q_tile), 0, ks, lane, qf[ks]);
        a_frag<D>(smem_addr(do_tile), 0, ks, lane, df[ks]);
    }
    int limit[2];
    float lse2[2], dl[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = (lane >> 2) + 8 * x;
        const int y = tile * 16 + min(r, rows - 1);
        const int64_t row = sq.row0 + qb * bq + y / G;
        const int64_t at = row * a.heads + h * G + y % G;
        limit[x] = attn_limit(a, sq, qb * bq + y / G);
        const float z = a.d_lse[at];
        lse2[x] = z == -CUDART_INF_F ? CUDART_INF_F : z * LOG2E;       // a row without keys: every p zero
        dl[x] = delta[at];
    }
    const float scale2 = a.scale * LOG2E;
    const DsScale dss = ds_scale<T>(a, factor);
    float o[D / 8][4] = {};
    int stage = 0;
    for (int c = warp; c < n_chunks; c += DQ_WARPS) {
        issue(c + DQ_WARPS * (DQ_STAGES - 1), (stage + DQ_STAGES - 1) % DQ_STAGES);
        cp_wait<DQ_STAGES - 1>();
        __syncwarp();
        const uint32_t kt = my_ring + stage * 2 * TILE16, vt = kt + TILE16;
        stage = stage + 1 == DQ_STAGES ? 0 : stage + 1;
        float sc[2][4] = {}, dp[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++) {
            uint32_t b[4];
            b_frag2<D>(kt, 0, ks, lane, b);
            mma16816<T>(sc[0], qf[ks], b[0], b[1]);
            mma16816<T>(sc[1], qf[ks], b[2], b[3]);
            b_frag2<D>(vt, 0, ks, lane, b);
            mma16816<T>(dp[0], df[ks], b[0], b[1]);
            mma16816<T>(dp[1], df[ks], b[2], b[3]);
        }
        const int p0 = blk[c / chunks_per_block] * a.block + (c % chunks_per_block) * 16;
        const bool masked = p0 > limit_min - 16;
#pragma unroll
        for (int nt = 0; nt < 2; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int x = i >> 1;
                float pr = fast_exp2(sc[nt][i] * scale2 - lse2[x]);
                float ds = pr * (dp[nt][i] - dl[x]) * dss.in;
                if (masked && p0 + nt * 8 + (lane & 3) * 2 + (i & 1) >= limit[x]) ds = 0.f;
                sc[nt][i] = ds;
            }
        const uint32_t pf[4] = {Pack<T>::two(sc[0][0], sc[0][1]), Pack<T>::two(sc[0][2], sc[0][3]),
                                Pack<T>::two(sc[1][0], sc[1][1]), Pack<T>::two(sc[1][2], sc[1][3])};
#pragma unroll
        for (int n = 0; n < D / 16; n++) {
            uint32_t b[4];
            bt_frag2<D>(kt, 0, n * 16, lane, b);
            mma16816<T>(o[2 * n], pf, b[0], b[1]);
            mma16816<T>(o[2 * n + 1], pf, b[2], b[3]);
        }
        __syncwarp();
    }
    cp_wait<0>();
    __syncthreads();
    float *so = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int n = 0; n < D / 8; n++)
#pragma unroll
        for (int x = 0; x < 2; x++)
            *reinterpret_cast<float2 *>(so + ((warp * 16 + (lane >> 2) + 8 * x) * D + n * 8 + (lane & 3) * 2)) =
                make_float2(o[n][2 * x], o[n][2 * x + 1]);
    __syncthreads();
    const int r = tid >> 3, c0 = (tid & 7) * (D / 8);
    __shared__ unsigned odd_rows;
    if (tid == 0) odd_rows = 0;
    bool odd = false;
    if (r < rows) {
        float y[D / 8] = {};
#pragma unroll
        for (int w = 0; w < DQ_WARPS; w++)
#pragma unroll
            for (int i = 0; i < D / 8; i++) y[i] += so[(w * 16 + r) * D + c0 + i];
#pragma unroll
        for (int i = 0; i < D / 8; i++) y[i] *= dss.out;
#pragma unroll
        for (int i = 0; i < D / 8; i++) odd |= not_finite(__float_as_uint(y[i]));
        uint32_t out[D / 16];
#pragma unroll
        for (int i = 0; i < D / 16; i++) out[i] = Pack<T>::two(y[2 * i], y[2 * i + 1]);
        const int x = tile * 16 + r;
        const int64_t at = ((int64_t)sq.row0 + qb * bq + x / G) * a.heads + h * G + x % G;
        if (odd) odd = !no_finite_ds(a.d_lse[at], delta[at]);
        T *dst = dq + at * D + c0;
#pragma unroll
        for (int i = 0; i < D / 64; i++) reinterpret_cast<uint4 *>(dst)[i] = *reinterpret_cast<uint4 *>(out + 4 * i);
    }
    if (!__syncthreads_or(odd)) return;
    // rows that are not finite once more, over their own keys alone (see row_keys)
    __shared__ uint32_t sure[D];
    if (odd) atomicOr(&odd_rows, 1u << r);
    if (tid < D) sure[tid] = 0;
    __syncthreads();
    sure_columns<T, D>(a, sq, s, h, static_cast<const T *>(a.d_k), a.k_token, a.k_head, shared_count, 0, nullptr, blk, nullptr, limit_min, sure,
                       tid, 128);
    __syncthreads();
#pragma unroll 1
    for (int sr = warp; sr < rows; sr += DQ_WARPS) {
        if (!(odd_rows >> sr & 1)) continue;
        const int x = tile * 16 + sr, query = qb * bq + x / G, head = h * G + x % G;
        const uint32_t *got = reinterpret_cast<const uint32_t *>(dq + (((int64_t)sq.row0 + query) * a.heads + head) * D + lane * (D / 32));
        bool open = false;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) open |= unsure(Pack<T>::to2(got[i / 2]), sure, lane * (D / 32) + i, ~0u);
        if (!__any_sync(~0u, open)) continue;
        float y[D / 32] = {};
        dq_row<T, D>(a, sq, s, h, query, head, d_do, do_token, do_head, delta, shared_count, [&](int e) { return blk[e]; }, lane, y);
        T *dst = dq + (((int64_t)sq.row0 + query) * a.heads + head) * D + lane * (D / 32);
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) *reinterpret_cast<uint32_t *>(dst + i) = Pack<T>::two(y[i], y[i + 1]);
    }
}

// The set bits [want0, want0 + room) of a block's query blocks, in order, to `list`; how many there are.  All threads.
template <int THREADS>
static __device__ __forceinline__ int expand_bits(const unsigned *my_bits, int words, int want0, int room, int *list, int *warp_sum)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, want1 = want0 + room;
    int found = 0;
    for (int w0 = 0; w0 < words && found < want1; w0 += THREADS) {
        unsigned word = w0 + tid < words ? my_bits[w0 + tid] : 0;
        const int n = __popc(word);
        int run = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(~0u, run, d);
            if (lane >= d) run += u;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = run;
        __syncthreads();
        int at = found + run - n, all = 0;
        for (int w = 0; w < THREADS / 32; w++) {
            if (w < warp) at += warp_sum[w];
            all += warp_sum[w];
        }
        while (word && at < want1) {
            const int bit = __ffs(word) - 1;
            word &= word - 1;
            if (at >= want0) list[at - want0] = (w0 + tid) * 32 + bit;
            at++;
        }
        found += all;
    }
    __syncthreads();
    return min(max(found - want0, 0), room);
}

// ---- tiles of 128 rows on the tensor memory path
//
// dq: 128 rows (queries x heads of a key head), 64 listed keys at a time.  S = Q K^T and dP = dO V^T go to tensor memory, a
// pair of threads for each row writes ds over S, dQ += ds K takes it from there.  Half the tensor memory and half the shared
// memory: two blocks of threads share an SM, one's exponentials run beside the other's products.  Bound by the chain of a
// step, products, then ds, then products, of which only two are under way on an SM (three tiles of K and V at D = 128 leave no
// room for a third): 3 sequences of up to 8192, 32 heads of 128, 16 blocks of 64 (414 GFLOP) take 550 us, 0.75 PFLOP/s.
constexpr int TQ_ROWS = 128, TQ_KEYS = 64, TQ_SOFTMAX = 256, TQ_THREADS = TQ_SOFTMAX + 64, TQ_COLS = 256;

// Blocks of keys whose marks fit the room of the key tiles.
template <int D> constexpr int TQ_BLOCKS = 3 * TQ_KEYS * D * 2 / 4 < UNION_BLOCKS ? 3 * TQ_KEYS * D * 2 / 4 : UNION_BLOCKS;

struct TqCtrl {
    uint64_t q_full, k_full[2], k_empty[2], v_full, v_empty, s_full, ds_full, dq_done;
    uint32_t tmem_base;
    uint32_t abort_flag;
    int32_t err;
    int32_t count;
    uint32_t odd[4];                    // rows whose result is not finite
};

template <typename T, int D>
__global__ __launch_bounds__(TQ_THREADS, 2) void attn_dq_tc_kernel(const __grid_constant__ spamm_attn a, int tiles,
                                                                   const TileShape shape, int max_entries,
                                                                   const __grid_constant__ RowMap k_map,
                                                                   const __grid_constant__ RowMap v_map, const T *d_do,
                                                                   int64_t do_token, int64_t do_head, const float *delta,
                                                                   const float *factor, T *dq)
{
    extern __shared__ __align__(1024) uint8_t smem_tc[];
    uint8_t *const smem = smem_tc;
    constexpr int RT = TQ_ROWS * D * 2, KT = TQ_KEYS * D * 2;
    const uint32_t q_tile = smem_u32(smem), do_tile = q_tile + RT, k_ring = do_tile + RT, v_tile = k_ring + 2 * KT;
    TqCtrl *ctrl = reinterpret_cast<TqCtrl *>(smem + 2 * RT + 3 * KT);
    uint32_t *bits = reinterpret_cast<uint32_t *>(ctrl + 1);           // [max_entries]
    uint16_t *blk = reinterpret_cast<uint16_t *>(bits + max_entries);

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned idx = blockIdx.x;
    const int tile = tiles - 1 - idx % tiles; idx /= tiles;
    const int h = idx % a.kv_heads;
    const int s = idx / a.kv_heads;
    const int G = a.heads / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    const TileRows tr = attn_tile(a, shape, sq, tile);
    if (!tr.rows) return;
    const int rows = tr.rows;
    const int limit_max = attn_limit(a, sq, tr.last), limit_min = attn_limit(a, sq, tr.first);

    if (warp < 8) {
        constexpr int PASS = TQ_SOFTMAX / (D / 8);                     // rows at a time
        const int c = tid % (D / 8);
        const T *q_src = static_cast<const T *>(a.d_q) + (int64_t)sq.row0 * a.q_token + (int64_t)h * G * a.q_head + c * 8;
        const T *do_src = d_do + (int64_t)sq.row0 * do_token + (int64_t)h * G * do_head + c * 8;
#pragma unroll
        for (int qr = tid / (D / 8); qr < TQ_ROWS; qr += PASS) {
            const bool ok = qr < rows;
            const int qy = tr.row0 + (ok ? qr : 0), tok = (int)shape.G.quotient(qy), head = qy - tok * G;
            const uint32_t off = panel_off(TQ_ROWS, qr, c);
            cp_async16(q_tile + off, q_src + tok * a.q_token + head * a.q_head, ok);
            cp_async16(do_tile + off, do_src + tok * do_token + head * do_head, ok);
        }
        cp_commit();
    } else if (warp == 8) {
        if (lane == 0) {
            mbar_init(smem_u32(&ctrl->q_full), TQ_SOFTMAX);
            for (int i = 0; i < 2; i++) {
                mbar_init(smem_u32(&ctrl->k_full[i]), 32);
                mbar_init(smem_u32(&ctrl->k_empty[i]), 1);
            }
            mbar_init(smem_u32(&ctrl->v_full), 32);
            mbar_init(smem_u32(&ctrl->v_empty), 1);
            mbar_init(smem_u32(&ctrl->s_full), 1);
            mbar_init(smem_u32(&ctrl->ds_full), TQ_SOFTMAX);
            mbar_init(smem_u32(&ctrl->dq_done), 1);
            ctrl->abort_flag = 0;
            ctrl->err = 0;
            for (int i = 0; i < 4; i++) ctrl->odd[i] = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        tmem_alloc<TQ_COLS>(smem_u32(&ctrl->tmem_base));
        tc_fence_before();
    }
    const int n_entries = attn_union<TQ_THREADS>(a, sq, s, h, tr, 0, ceil_div(limit_max, a.block),
                                                 reinterpret_cast<uint32_t *>(smem + 2 * RT), blk, bits, &ctrl->count);
    tc_fence_after();
    const int log_block = 31 - __clz(a.block);
    const int n_keys = n_entries << log_block;
    const int n_tiles = (n_keys + TQ_KEYS - 1) / TQ_KEYS;
    const uint32_t tmem = ctrl->tmem_base, tmem_dq = tmem + 2 * TQ_KEYS;
    const WaitState ws{&ctrl->abort_flag, &ctrl->err};

    if (warp == 9) {
        const int piece = min(a.block, TQ_KEYS), pieces = TQ_KEYS / piece;     // a piece: keys of one block, one tensor copy
        auto load = [&](int j, uint32_t dst, bool value, uint64_t *full) {
            const uint32_t bar = smem_u32(full);
            const RowMap &rm = value ? v_map : k_map;
            bool by_hand = false;
            for (int x = lane; x < pieces * (D / 64); x += 32) {
                const int i = x / (D / 64), panel = x % (D / 64), key = j * TQ_KEYS + i * piece, e = key >> log_block;
                if (e >= n_entries) continue;
                const int pos = blk[e] * a.block + (key & (a.block - 1));
                if (!rm.usable || pos + piece > sq.nk) { by_hand = true; continue; }
                mbar_expect_tx(bar, piece * 128);
                tma_box(dst + panel * (TQ_KEYS * 128) + i * piece * 128, &rm.map, panel * 64, rm.swapped ? sq.row0 + pos : h,
                        rm.swapped ? h : sq.row0 + pos, bar);
            }
            if (__any_sync(~0u, by_hand)) {
                const T *src = static_cast<const T *>(value ? a.d_v : a.d_k);
                const int64_t tok = value ? a.v_token : a.k_token, head = value ? a.v_head : a.k_head;
                for (int i = 0; i < pieces; i++) {
                    const int key = j * TQ_KEYS + i * piece, e = key >> log_block;
                    if (e >= n_entries) break;
                    const int pos = blk[e] * a.block + (key & (a.block - 1));
                    if (rm.usable && pos + piece <= sq.nk) continue;
                    const int n = sq.nk - pos;
                    const int64_t at = n > 0 ? (int64_t)(sq.row0 + pos) * tok + h * head : 0;
                    for (int x = lane; x < piece * (D / 8); x += 32) {
                        const int r = x / (D / 8), c = x % (D / 8);
                        cp_async16(dst + panel_off(TQ_KEYS, i * piece + r, c), src + (r < n ? at + r * tok : 0) + c * 8, r < n);
                    }
                }
                cp_commit();
                cp_wait<0>();
                fence_async_smem();
            }
            mbar_arrive(bar);
        };
        bool fine = true;
        for (int j = 0; j < n_tiles; j++) {
            if (j > 1) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->k_empty[j & 1]), (j >> 1) - 1, 1));
            if (!fine) break;
            load(j, k_ring + (j & 1) * KT, false, &ctrl->k_full[j & 1]);
            if (j) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->v_empty), j - 1, 2));
            if (!fine) break;
            load(j, v_tile, true, &ctrl->v_full);
        }
        __syncthreads();
    } else if (warp == 8) {
        if (n_tiles) {
            constexpr uint32_t s_desc = mma_desc<T>(128, TQ_KEYS, false, false), o_desc = mma_desc<T>(128, D, false, true);
            const uint32_t base = __shfl_sync(~0u, tmem, 0);
            const uint64_t q_desc = desc_k_major(q_tile), do_desc = desc_k_major(do_tile), v_desc = desc_k_major(v_tile);
            const uint64_t k_desc = desc_k_major(k_ring), kt_desc = desc_mn_major(k_ring, TQ_KEYS);
            bool fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->q_full), 0, 3));
            for (int j = 0; j < n_tiles && fine; j++) {
                const uint32_t stage = (j & 1) * (KT >> 4);
                fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->k_full[j & 1]), j >> 1, 4) && ws.wait(smem_u32(&ctrl->v_full), j, 5));
                if (!fine) break;
                tc_fence_after();
                if (elect_one()) {
                    // dP first: the buffer of V comes free the earlier
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++)
                        mma_ss(base + TQ_KEYS, do_desc + step_k_major(TQ_ROWS, ks), v_desc + step_k_major(TQ_KEYS, ks), s_desc, ks != 0);
                    umma_commit(smem_u32(&ctrl->v_empty));
#pragma unroll
                    for (int ks = 0; ks < D / 16; ks++)
                        mma_ss(base, q_desc + step_k_major(TQ_ROWS, ks), k_desc + stage + step_k_major(TQ_KEYS, ks), s_desc, ks != 0);
                    umma_commit(smem_u32(&ctrl->s_full));
                }
                __syncwarp();
                fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->ds_full), j, 6));
                if (!fine) break;
                tc_fence_after();
                const int steps = min(TQ_KEYS, n_keys - j * TQ_KEYS) / 16;      // rows of K behind were never written
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < TQ_KEYS / 16; ks++)
                        if (ks < steps)
                            mma_ts(base + 2 * TQ_KEYS, base + (ks >> 1) * 32 + (ks & 1) * 8, kt_desc + stage + step_mn_major(ks), o_desc, j || ks);
                    umma_commit(smem_u32(&ctrl->k_empty[j & 1]));
                    umma_commit(smem_u32(&ctrl->dq_done));
                }
                __syncwarp();
            }
        }
        __syncwarp();
        __syncthreads();
    } else {
        const int r = tid & 127, half = warp >> 2, y = tr.row0 + min(r, rows - 1), my_query = (int)shape.G.quotient(y);
        const int limit = attn_limit(a, sq, my_query);
        const uint32_t my_bit = 1u << (my_query / a.query_block - tr.qb0), all_bits = tr.n_qb == 32 ? ~0u : (1u << tr.n_qb) - 1;
        const int64_t at = (int64_t)(sq.row0 + my_query) * a.heads + h * G + y - my_query * G;
        const float z = a.d_lse[at];
        const float minus_lse = z == -CUDART_INF_F ? -CUDART_INF_F : -z * LOG2E;       // a row without keys: every p zero
        const DsScale dss = ds_scale<T>(a, factor);
        const float minus_delta = -delta[at] * dss.in;
        cp_wait<0>();
        fence_async_smem();
        mbar_arrive(smem_u32(&ctrl->q_full));
        const uint32_t lane_s = tmem + ((uint32_t)((warp & 3) * 32) << 16) + half * 32, lane_dp = lane_s + TQ_KEYS;
        const uint32_t lane_dq = tmem_dq + ((uint32_t)((warp & 3) * 32) << 16) + half * (D / 2);
        const float scale2 = a.scale * LOG2E;
        const float2 sc2 = make_float2(scale2, scale2), ml2 = make_float2(minus_lse, minus_lse);
        const float2 sc = make_float2(dss.in, dss.in), md = make_float2(minus_delta, minus_delta);
        bool fine = true;
        for (int j = 0; j < n_tiles; j++) {
            // lanes 0 and 1: position and lists of this half's groups of 16 keys
            int group_pos = INT32_MAX / 2;
            uint32_t group_bits = all_bits;
            if (lane < 2) {
                const int key = j * TQ_KEYS + half * 32 + lane * 16, e = key >> log_block;
                if (e < n_entries) {
                    group_pos = blk[e] * a.block + (key & (a.block - 1));
                    group_bits = bits[e];
                }
            }
            const bool masked = __any_sync(~0u, (lane < 2 && group_pos > limit_min - 16) || group_bits != all_bits);
            fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->s_full), j, 7));
            if (!fine) break;
            tc_fence_after();
            uint32_t v[32], d[32], w[16];
            tmem_ld32(lane_s, v);
            tmem_ld32(lane_dp, d);
            tmem_wait_ld();
            tmem_landed<32>(v);
            tmem_landed<32>(d);
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const float2 x = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sc2, ml2);
                const float2 g = fma2(make_float2(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])), sc, md);
                v[2 * i] = __float_as_uint(fast_exp2(x.x) * g.x);
                v[2 * i + 1] = __float_as_uint(fast_exp2(x.y) * g.y);
            }
            if (masked) {
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    const int pos = __shfl_sync(~0u, group_pos, g);
                    const int n = __shfl_sync(~0u, group_bits, g) & my_bit ? limit - pos : 0;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (i >= n) v[g * 16 + i] = 0u;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i++) w[i] = Pack<T>::two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
            tmem_st16(lane_s, w);                               // over this thread's scores, which have been read
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&ctrl->ds_full));
        }
        if (n_tiles && fine) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->dq_done), n_tiles - 1, 8));
        tc_fence_after();
        __syncthreads();                                       // every copy has landed, every product is done
        bool odd = false;
#pragma unroll 1
        for (int c = 0; c < D / 64; c++) {
            uint32_t v[32];
            if (n_tiles) {
                tmem_ld32(lane_dq + c * 32, v);
                tmem_wait_ld();
                tmem_landed<32>(v);
            }
#pragma unroll
            for (int i = 0; i < 32; i++) v[i] = !fine ? 0x7fc00000u : n_tiles ? __float_as_uint(__uint_as_float(v[i]) * dss.out) : 0u;
#pragma unroll
            for (int i = 0; i < 32; i++) odd |= not_finite(v[i]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                uint32_t x[4];
#pragma unroll
                for (int k = 0; k < 4; k++)
                    x[k] = Pack<T>::two(__uint_as_float(v[8 * i + 2 * k]), __uint_as_float(v[8 * i + 2 * k + 1]));
                *reinterpret_cast<uint4 *>(smem + row_piece(D * 2, r, half * (D / 16) + c * 4 + i)) = *reinterpret_cast<uint4 *>(x);
            }
        }
        const unsigned rows_odd = __ballot_sync(~0u, odd && fine && r < rows && !no_finite_ds(z, minus_delta));
        if (rows_odd && lane == 0) atomicOr(&ctrl->odd[warp & 3], rows_odd);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ctrl->odd[0] | ctrl->odd[1] | ctrl->odd[2] | ctrl->odd[3]) {
            uint32_t *const sure = reinterpret_cast<uint32_t *>(smem + RT);         // behind the rows
            if (tid < D) sure[tid] = 0;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            sure_columns<T, D>(a, sq, s, h, static_cast<const T *>(a.d_k), a.k_token, a.k_head, n_entries, 0, blk, nullptr, bits, limit_min, sure,
                               tid, 256);
            asm volatile("bar.sync 1, 256;" ::: "memory");
#pragma unroll 1
            for (int sr = warp; sr < rows; sr += 8) {
                if (!(ctrl->odd[sr >> 5] >> (sr & 31) & 1)) continue;
                const int sy = tr.row0 + sr, tok = (int)shape.G.quotient(sy), head = h * G + sy - tok * G;
                const uint32_t bit = 1u << (tok / a.query_block - tr.qb0);
                bool open = false;
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) {
                    const int d = lane * (D / 32) + i, piece = d * 2;
                    open |= unsure(Pack<T>::to2(*reinterpret_cast<const uint32_t *>(smem + row_piece(D * 2, sr, piece >> 4) + (piece & 15))), sure, d, bit);
                }
                if (!__any_sync(~0u, open)) continue;
                float y2[D / 32] = {};
                dq_row<T, D>(a, sq, s, h, tok, head, d_do, do_token, do_head, delta, n_entries,
                             [&](int e) { return bits[e] & bit ? (int)blk[e] : -1; }, lane, y2);
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) {
                    const int piece = (lane * (D / 32) + i) * 2;
                    *reinterpret_cast<uint32_t *>(smem + row_piece(D * 2, sr, piece >> 4) + (piece & 15)) = Pack<T>::two(y2[i], y2[i + 1]);
                }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        const int c = tid % (D / 8);
        for (int sr = tid / (D / 8); sr < rows; sr += TQ_SOFTMAX / (D / 8)) {
            const int sy = tr.row0 + sr, tok = (int)shape.G.quotient(sy);
            *reinterpret_cast<uint4 *>(dq + ((int64_t)(sq.row0 + tok) * a.heads + h * G + sy - tok * G) * D + c * 8) =
                *reinterpret_cast<const uint4 *>(smem + row_piece(D * 2, sr, c));
        }
        if (!fine && a.d_status) *a.d_status = SPAMM_ERR_DEVICE_WAIT;
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        if (ctrl->abort_flag) drain_products();
        __syncwarp();
        tc_fence_after();
        tmem_free<TQ_COLS>(tmem);
    }
}

// dk and dv of a block's keys (of half a block of 128) from one chunk of the query blocks that list it, 128 gathered rows at a
// time.
//
//   S = Q K^T, dP = dO V^T   [128 rows x keys]        from shared memory, two buffers each in tensor memory
//   dV^T += dO^T P,  dK^T += Q^T ds   [D x keys]      the tiles of dO and Q once more, as operands whose rows are K
//
// P and ds pass through shared memory.  One block of threads per SM: while eight warps work on the exponentials of one
// tile, the products of the tile before and of the one behind it run, and four warps gather the rows of the one after.
// With D = 64 the tiles of dO and Q together are the 128 rows of the second products' A: dV^T comes out in the upper half
// of one accumulator, dK^T in the lower half of the other (the other halves are not used).
//
// Bound by the chain of a tile, scores to p and ds to the second products, whose steps the roles hand one another through
// barriers: 3 sequences of up to 8192, 32 heads of 128, lists of 16 blocks of 64 (553 GFLOP) take 843 to 891 us from run to
// run, 0.62 to 0.66 PFLOP/s, and with every product cut to a single step still about 690 us, with the exponentials left out
// 820 us.  Four threads for a row 942 us; a few exponentials by the polynomial of attn_tc.cuh 880 to 895 us, no gain.  Five
// buffers of rows instead of two pairs 905 -> 892 us.  Chunks of 8192 rows for one item: 4096 906 us and 2048 980 us against
// 909 us, 269, 260 and 286 us with a list for each query.
constexpr int TK_ROWS = 128, TK_MAX_KEYS = 64, TK_SOFTMAX = 256, TK_THREADS = TK_SOFTMAX + 32 + 128;
// Tensor memory columns, and blocks of threads per SM: short blocks of small heads leave room for two.
__host__ __device__ constexpr int tk_cols(int keys) { return keys == 64 ? 512 : keys == 32 ? 256 : 128; }
__host__ __device__ constexpr int tk_per_sm(int dim, int keys) { return dim == 64 && keys < 64 ? 2 : 1; }
// Buffers of the ring that the tiles of dO and Q pass through in turn (dO of tile j is the ring's 2 j-th, Q its 2 j + 1-st).
// An even number where the two of a tile must lie side by side.
__host__ __device__ constexpr int tk_slots(int dim, int keys) { return dim == 128 ? 5 : keys < 64 ? 4 : 8; }
constexpr int TK_MAX_SLOTS = 8;

struct TkCtrl {
    uint64_t kv_full, full[TK_MAX_SLOTS], empty[TK_MAX_SLOTS], s_full[2], p_full, dv_done, ds_full, dk_done;
    uint32_t tmem_base;
    uint32_t abort_flag;
    int32_t err;
    int32_t warp_sum[TK_THREADS / 32];
};

template <typename T, int D, int TK_KEYS>
__global__ __launch_bounds__(TK_THREADS, tk_per_sm(D, TK_KEYS)) void attn_dkv_tc_kernel(const __grid_constant__ spamm_attn a, const __grid_constant__ BackwardPlan p,
                                                                    const __grid_constant__ RowMap q_map,
                                                                    const __grid_constant__ RowMap do_map,
                                                                    const T *d_do, int64_t do_token, int64_t do_head,
                                                                    const float *delta, const float *factor, const unsigned *bits,
                                                                    const Item *items, const int *n_items, float *partial, T *dk, T *dv)
{
    extern __shared__ __align__(1024) uint8_t smem_tc[];
    uint8_t *const smem = smem_tc;
    constexpr int KT = TK_KEYS * D * 2, RT = TK_ROWS * D * 2, PT = TK_ROWS * 128;     // rows of p and ds take a panel's 128 bytes
    constexpr int HALF = TK_KEYS / 2;                           // keys of a thread
    constexpr int SLOTS = tk_slots(D, TK_KEYS);
    const uint32_t k_tile = smem_u32(smem), v_tile = k_tile + KT, ring = v_tile + KT;
    const uint32_t p_tile = ring + SLOTS * RT, ds_tile = p_tile + PT;
    TkCtrl *ctrl = reinterpret_cast<TkCtrl *>(smem + 2 * KT + SLOTS * RT + 2 * PT);
    int *list = reinterpret_cast<int *>(ctrl + 1);

    const int halves = a.block / TK_KEYS;
    const int half = blockIdx.x % halves;
    const unsigned rest = blockIdx.x / halves;
    const int64_t group = rest / p.item_cap;
    const int item_i = rest % p.item_cap;
    if (item_i >= n_items[group]) return;
    const Item item = items[group * p.item_cap + item_i];
    const int s = (int)(group / a.kv_heads), h = (int)(group % a.kv_heads);
    const Seq sq = attn_seq(a, s);
    const int G = a.heads / a.kv_heads;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int pos0 = item.kb * a.block + half * TK_KEYS;
    const int keys = min(TK_KEYS, sq.nk - pos0);
    if (keys <= 0) return;

    if (warp == 8) {
        if (lane == 0) {
            mbar_init(smem_u32(&ctrl->kv_full), 128);
            for (int i = 0; i < SLOTS; i++) {
                mbar_init(smem_u32(&ctrl->full[i]), 64);
                mbar_init(smem_u32(&ctrl->empty[i]), 1);
            }
            for (int i = 0; i < 2; i++) mbar_init(smem_u32(&ctrl->s_full[i]), 1);
            mbar_init(smem_u32(&ctrl->p_full), TK_SOFTMAX);
            mbar_init(smem_u32(&ctrl->ds_full), TK_SOFTMAX);
            mbar_init(smem_u32(&ctrl->dv_done), 1);
            mbar_init(smem_u32(&ctrl->dk_done), 1);
            ctrl->abort_flag = 0;
            ctrl->err = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        tmem_alloc<tk_cols(TK_KEYS)>(smem_u32(&ctrl->tmem_base));
        tc_fence_before();
    }
    const int n_list = expand_bits<TK_THREADS>(bits + (group * p.nkb + item.kb) * p.words, p.words, item.chunk * p.chunk, p.chunk,
                                               list, ctrl->warp_sum);
    tc_fence_after();
    const int bq = min(a.query_block, a.max_q), per = bq * G;
    // all listed query blocks are full but the sequence's last one, which can only be the last of the list
    const int n_rows = n_list ? (n_list - 1) * per + min(bq, sq.nq - list[n_list - 1] * bq) * G : 0;
    const int n_tiles = (n_rows + TK_ROWS - 1) / TK_ROWS;
    const uint32_t tmem = ctrl->tmem_base, tmem_dv = tmem + 4 * TK_KEYS, tmem_dk = tmem_dv + TK_KEYS;
    const WaitState ws{&ctrl->abort_flag, &ctrl->err};
    // row x of the gathered rows: its row of q and its head; false when there is none
    auto locate = [&](int x, int *query, int *head) {
        if (x >= n_rows) return false;
        const int e = (int)p.per.quotient(x), y = x - e * per, tok = (int)p.G.quotient(y);
        *query = list[e] * bq + tok;
        *head = h * G + y - tok * G;
        return true;
    };

    if (warp > 8) {
        // ---- rows: two warps bring those of dO (and V first), two those of Q (and K first), each as its buffers come free
        const int t = (tid - TK_SOFTMAX - 32) & 63, lw = t >> 5;
        const bool is_q = tid - TK_SOFTMAX - 32 >= 64;
        const T *src = is_q ? static_cast<const T *>(a.d_q) : d_do;
        const int64_t token = is_q ? a.q_token : do_token, stride = is_q ? a.q_head : do_head;
        // waits until the buffer of tile j is free: the n-th of the ring takes the place of the (n - SLOTS)-th
        auto number = [&](int j) { return 2 * j + (is_q ? 1 : 0); };
        auto buffer_free = [&](int j) {
            const int n = number(j);
            return n < SLOTS || __all_sync(~0u, ws.wait(smem_u32(&ctrl->empty[n % SLOTS]), n / SLOTS - 1, 1));
        };
        {
            const T *kv = is_q ? static_cast<const T *>(a.d_k) : static_cast<const T *>(a.d_v);
            const int64_t kv_token = is_q ? a.k_token : a.v_token, kv_head = is_q ? a.k_head : a.v_head;
            const uint32_t tile = is_q ? k_tile : v_tile;
            for (int x = t; x < TK_KEYS * (D / 8); x += 64) {
                const int r = x / (D / 8), c = x % (D / 8);
                const bool ok = r < keys;
                cp_async16(tile + panel_off(TK_KEYS, r, c), kv + (int64_t)(sq.row0 + pos0 + (ok ? r : 0)) * kv_token + h * kv_head + c * 8, ok);
            }
            cp_commit();
        }
        constexpr int PASS = 32 / (D / 8);                      // rows of a warp's copy
        const int col = lane % (D / 8), sub = lane / (D / 8);
        bool fine = true;
        auto signal = [&](uint64_t *bar) {
            fence_async_smem();
            mbar_arrive(smem_u32(bar));
        };
        // whole tiles by tensor copies; the one in which the rows end, or all when the strides do not allow it, row by row
        const RowMap &map = is_q ? q_map : do_map;
        const int by_map = p.box_tokens && map.usable && !map.swapped ? n_rows / TK_ROWS : 0;
        if (by_map) {
            const int box_rows = p.box_tokens * G, boxes = TK_ROWS / box_rows;
            const int i = t % boxes, panel = t / boxes;
            for (int j = 0; j < by_map; j++) {
                fine = buffer_free(j);
                if (!fine) break;
                const int slot = number(j) % SLOTS;
                const uint32_t bar = smem_u32(&ctrl->full[slot]);
                if (panel < D / 64) {
                    int query, head;
                    locate(j * TK_ROWS + i * box_rows, &query, &head);
                    mbar_expect_tx(bar, box_rows * 128);
                    tma_box(ring + slot * RT + panel * (TK_ROWS * 128) + i * box_rows * 128, &map.map, panel * 64, head,
                            sq.row0 + query, bar);
                }
                mbar_arrive(bar);
                if (j == 0) {
                    cp_wait<0>();
                    signal(&ctrl->kv_full);
                }
            }
        }
        int waiting = by_map ? -1 : -2;                         // what was requested and not announced: a tile, -2: K or V
        auto announce = [&] {
            if (waiting != -1) signal(waiting == -2 ? &ctrl->kv_full : &ctrl->full[number(waiting) % SLOTS]);
            waiting = -1;
        };
        for (int j = by_map; j <= n_tiles && fine; j++) {
            if (j < n_tiles) {
                if (number(j) >= SLOTS && waiting != -1) {
                    // the buffer comes free only when tiles before have been worked on: announce them first
                    cp_wait<0>();
                    announce();
                }
                fine = buffer_free(j);
                if (!fine) break;
                const uint32_t dst = ring + number(j) % SLOTS * RT;
#pragma unroll 1
                for (int half_tile = 0; half_tile < 2; half_tile++) {
                    // each lane finds one of 32 rows, the copies take the addresses from it
                    const int r0 = lw * 64 + half_tile * 32;
                    int query = 0, head = 0;
                    const bool there = locate(j * TK_ROWS + r0 + lane, &query, &head);
                    const int64_t at = there ? (int64_t)(sq.row0 + query) * token + head * stride : -1;
#pragma unroll 4
                    for (int i = 0; i < 32; i += PASS) {
                        const int r = i + sub;
                        const int64_t from = __shfl_sync(~0u, at, r);
                        cp_async16(dst + panel_off(TK_ROWS, r0 + r, col), src + (from < 0 ? 0 : from) + col * 8, from >= 0);
                    }
                }
            }
            cp_commit();
            if (waiting != -1) {
                cp_wait<1>();                                   // the group before this one
                announce();
            }
            if (j < n_tiles) waiting = j;
        }
        cp_wait<0>();
    } else if (warp == 8) {
        // ---- products
        if (n_tiles) {
            constexpr uint32_t s_desc = mma_desc<T>(128, TK_KEYS, false, false), o_desc = mma_desc<T>(128, TK_KEYS, true, true);
            const uint32_t base = __shfl_sync(~0u, tmem, 0);
            const uint64_t k_desc = desc_k_major(k_tile), v_desc = desc_k_major(v_tile), row_desc = desc_k_major(ring);
            // A of the second products: 128 values of dO (of Q) x 128 rows; with D = 64 the tiles of dO and Q one behind the other
            const uint64_t turned_desc = desc_mn_major(ring, TK_ROWS);
            const uint64_t p_desc = desc_mn_major(p_tile, TK_ROWS), ds_desc = desc_mn_major(ds_tile, TK_ROWS);
            bool fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->kv_full), 0, 2));
            // Whichever is ready: dP of the next tile (at most one tile under way), its S, or the second products of the oldest
            // tile under way.  dO comes free after dV, before Q does, and returns before it: hence dP before S.  (In a fixed
            // order the second products would wait for the copies of the next tile, which wait for the buffers that they free.)
            int next_dp = 0, next_s = 0, second = 0, idle = 0;
            unsigned long long t0 = 0;
            auto do_slot = [](int j) { return 2 * j % SLOTS; };
            auto q_slot = [](int j) { return (2 * j + 1) % SLOTS; };
            while (second < n_tiles) {
                const uint32_t dp_stage = do_slot(next_dp) * (RT >> 4), s_stage = q_slot(next_s) * (RT >> 4);
                if (next_s < next_dp && __all_sync(~0u, mbar_test(smem_u32(&ctrl->full[q_slot(next_s)]), (2 * next_s + 1) / SLOTS & 1))) {
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < D / 16; ks++)
                            mma_ss(base + (next_s & 1) * 2 * TK_KEYS, row_desc + s_stage + step_k_major(TK_ROWS, ks), k_desc + step_k_major(TK_KEYS, ks),
                                   s_desc, ks != 0);
                        umma_commit(smem_u32(&ctrl->s_full[next_s & 1]));
                    }
                    __syncwarp();
                    next_s++;
                    t0 = 0;
                } else if (next_dp < n_tiles && next_dp - second < 2 &&
                           __all_sync(~0u, mbar_test(smem_u32(&ctrl->full[do_slot(next_dp)]), 2 * next_dp / SLOTS & 1))) {
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < D / 16; ks++)
                            mma_ss(base + (next_dp & 1) * 2 * TK_KEYS + TK_KEYS, row_desc + dp_stage + step_k_major(TK_ROWS, ks),
                                   v_desc + step_k_major(TK_KEYS, ks), s_desc, ks != 0);
                    }
                    __syncwarp();
                    next_dp++;
                    t0 = 0;
                } else if (second < next_s && __all_sync(~0u, mbar_test(smem_u32(&ctrl->p_full), second & 1))) {
                    tc_fence_after();
                    const int do_at = do_slot(second), q_at = q_slot(second);
                    const uint32_t do_stage = do_at * (RT >> 4), q_stage = (D == 64 ? do_at : q_at) * (RT >> 4);
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < TK_ROWS / 16; ks++)
                            mma_ss(base + 4 * TK_KEYS, turned_desc + do_stage + step_mn_major(ks), p_desc + step_mn_major(ks), o_desc, second || ks);
                        if (D == 128) umma_commit(smem_u32(&ctrl->empty[do_at]));
                        umma_commit(smem_u32(&ctrl->dv_done));
                    }
                    __syncwarp();
                    fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->ds_full), second, 5));
                    if (!fine) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int ks = 0; ks < TK_ROWS / 16; ks++)
                            mma_ss(base + 5 * TK_KEYS, turned_desc + q_stage + step_mn_major(ks), ds_desc + step_mn_major(ks), o_desc, second || ks);
                        if (D == 64) umma_commit(smem_u32(&ctrl->empty[do_at]));      // dO is half of this A too
                        umma_commit(smem_u32(&ctrl->empty[q_at]));
                        umma_commit(smem_u32(&ctrl->dk_done));
                    }
                    __syncwarp();
                    second++;
                    t0 = 0;
                } else {
                    if (++idle & 63) continue;                   // the clock is slow to read
                    if (__any_sync(~0u, !fine || *ws.abort_flag)) break;
                    if (!t0) t0 = global_ns();
                    if (__any_sync(~0u, global_ns() - t0 > WAIT_LIMIT_NS)) {
                        *ws.abort_flag = 1;
                        break;
                    }
                }
            }
        }
        __syncwarp();
    } else {
        // ---- p and ds: thread = row, the upper four warps the second half of the keys
        const int r = tid & 127, part = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const float scale2 = a.scale * LOG2E;
        // half: p times 2^P_UP, and ds = p (dP - delta) with it times the factor
        constexpr bool IS_HALF = std::is_same<T, __half>::value;
        const DsScale dss = ds_scale<T>(a, factor);
        const float p_up = IS_HALF ? P_UP : 0.f, p_down = IS_HALF ? P_DOWN : 1.f, ds_in = dss.in * p_down;
        const float2 sc2 = make_float2(scale2, scale2), sc = make_float2(ds_in, ds_in);
        // lse and delta of the row in tile j as they are, and how many of this thread's keys it sees: requested a tile ahead,
        // and not touched before they are needed
        auto row_of = [&](int j, float *lse, float *dl, int *n_visible) {
            int query, head;
            *lse = -CUDART_INF_F;                               // a row that is none, or has no keys: every p zero
            *dl = 0.f;
            *n_visible = 0;
            if (j < n_tiles && locate(j * TK_ROWS + r, &query, &head)) {
                const int64_t at = (int64_t)(sq.row0 + query) * a.heads + head;
                *lse = a.d_lse[at];
                *dl = delta[at];
                *n_visible = min(a.causal ? query + 1 - pos0 : TK_KEYS, keys) - part * HALF;
            }
        };
        float lse, dl;
        int n_visible;
        row_of(0, &lse, &dl, &n_visible);
        bool fine = true;
        for (int j = 0; j < n_tiles; j++) {
            const float minus_lse = lse == -CUDART_INF_F ? lse : IS_HALF ? fmaf(-lse, LOG2E, p_up) : -lse * LOG2E, minus_delta = -dl * ds_in;
            int next_visible;
            row_of(j + 1, &lse, &dl, &next_visible);
            fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->s_full[j & 1]), j >> 1, 6));
            if (!fine) break;
            tc_fence_after();
            const uint32_t s_at = tmem + (j & 1) * 2 * TK_KEYS + lanes + part * HALF;
            uint32_t v[HALF], d[HALF], w[HALF / 2];
            tmem_ld<HALF>(s_at, v);
            tmem_ld<HALF>(s_at + TK_KEYS, d);
            tmem_wait_ld();
            tmem_landed<HALF>(v);
            tmem_landed<HALF>(d);
            const float2 ml2 = make_float2(minus_lse, minus_lse), md = make_float2(minus_delta, minus_delta);
#pragma unroll
            for (int i = 0; i < HALF / 2; i++) {
                const float2 x = fma2(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), sc2, ml2);
                const float2 g = fma2(make_float2(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1])), sc, md);
                const float e0 = fast_exp2(x.x), e1 = fast_exp2(x.y);
                v[2 * i] = __float_as_uint(e0);
                v[2 * i + 1] = __float_as_uint(e1);
                d[2 * i] = __float_as_uint(e0 * g.x);
                d[2 * i + 1] = __float_as_uint(e1 * g.y);
            }
            if (__any_sync(~0u, n_visible < HALF)) {
#pragma unroll
                for (int i = 0; i < HALF; i++)
                    if (i >= n_visible) { v[i] = 0u; d[i] = 0u; }
            }
#pragma unroll
            for (int i = 0; i < HALF / 2; i++) w[i] = Pack<T>::two(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
            if (j) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->dv_done), j - 1, 7));
            if (!fine) break;
#pragma unroll
            for (int c = 0; c < HALF / 8; c++)
                *reinterpret_cast<uint4 *>(smem + (p_tile - k_tile) + panel_off(TK_ROWS, r, part * (HALF / 8) + c)) =
                    make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            fence_async_smem();
            tc_fence_before();
            mbar_arrive(smem_u32(&ctrl->p_full));
#pragma unroll
            for (int i = 0; i < HALF / 2; i++) w[i] = Pack<T>::two(__uint_as_float(d[2 * i]), __uint_as_float(d[2 * i + 1]));
            if (j) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->dk_done), j - 1, 8));
            if (!fine) break;
#pragma unroll
            for (int c = 0; c < HALF / 8; c++)
                *reinterpret_cast<uint4 *>(smem + (ds_tile - k_tile) + panel_off(TK_ROWS, r, part * (HALF / 8) + c)) =
                    make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            fence_async_smem();
            tc_fence_before();
            mbar_arrive(smem_u32(&ctrl->ds_full));
            n_visible = next_visible;
        }
        if (n_tiles && fine) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->dk_done), n_tiles - 1, 9));
        tc_fence_after();
        // rows of the accumulators are the D values, columns the keys: four warps write dv, four dk
        const bool is_k = part != 0;
        const float out = is_k ? dss.out : p_down;
        const int row = r, d0 = D == 64 && is_k ? row - 64 : row;
        const bool mine = D == 128 || (is_k ? row >= 64 : row < 64);            // whole warps
        constexpr int COLS = TK_KEYS < 32 ? TK_KEYS : 32;
#pragma unroll 1
        for (int c = 0; c < TK_KEYS / COLS; c++) {
            uint32_t v[COLS];
            if (n_tiles) {
                tmem_ld<COLS>((is_k ? tmem_dk : tmem_dv) + lanes + c * COLS, v);
                tmem_wait_ld();
                tmem_landed<COLS>(v);
            }
#pragma unroll
            for (int i = 0; i < COLS; i++) v[i] = !fine ? 0x7fc00000u : n_tiles ? __float_as_uint(__uint_as_float(v[i]) * out) : 0u;
            if (!mine) continue;
            if (item.slot >= 0) {
                float *dst = partial + (group * p.slot_cap + item.slot) * (int64_t)(2 * a.block * D) + (is_k ? 0 : a.block * D) +
                             (half * TK_KEYS + c * COLS) * D + d0;
#pragma unroll
                for (int i = 0; i < COLS; i++) dst[i * D] = __uint_as_float(v[i]);
            } else {
                T *dst = (is_k ? dk : dv) + ((int64_t)(sq.row0 + pos0 + c * COLS) * a.kv_heads + h) * D + d0;
#pragma unroll
                for (int i = 0; i < COLS; i++)
                    if (c * COLS + i < keys) dst[(int64_t)i * a.kv_heads * D] = Pack<T>::one(__uint_as_float(v[i]));
            }
        }
        if (!fine && a.d_status) *a.d_status = SPAMM_ERR_DEVICE_WAIT;
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        if (ctrl->abort_flag) drain_products();
        __syncwarp();
        tc_fence_after();
        tmem_free<tk_cols(TK_KEYS)>(tmem);
    }
}

// Adds up the partial sums of the blocks of keys that were cut into several items, in the order of the items.  Bound by the
// reading of the sums: 23 us in the case of attn_dkv_tc_kernel's figures.
template <typename T>
__global__ __launch_bounds__(128) void attn_dkv_join_kernel(const __grid_constant__ spamm_attn a, const BackwardPlan p,
                                                            const int *counts, const int *slots, const float *partial,
                                                            T *dk, T *dv)
{
    const int64_t group = blockIdx.x / p.nkb;
    const int kb = blockIdx.x % p.nkb;
    const int s = (int)(group / a.kv_heads), h = (int)(group % a.kv_heads);
    const Seq sq = attn_seq(a, s);
    const int keys = min(a.block, sq.nk - kb * a.block);
    const int chunks = keys > 0 ? ceil_div(counts[group * p.nkb + kb], p.chunk) : 0;
    if (chunks <= 1) return;
    const int64_t tile = 2 * (int64_t)a.block * a.dim;
    const float *src = partial + (group * p.slot_cap + slots[group * p.nkb + kb]) * tile;
    for (int i = blockIdx.y * 128 + threadIdx.x; i < 2 * keys * a.dim / 4; i += 128 * gridDim.y) {
        const int which = i >= keys * a.dim / 4;
        const int x = (i - which * (keys * a.dim / 4)) * 4;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = 0; c < chunks; c++) {
            const float4 z = *reinterpret_cast<const float4 *>(src + c * tile + which * a.block * a.dim + x);
            y.x += z.x; y.y += z.y; y.z += z.z; y.w += z.w;
        }
        T *dst = (which ? dv : dk) + ((int64_t)(sq.row0 + kb * a.block + x / a.dim) * a.kv_heads + h) * a.dim + x % a.dim;
        *reinterpret_cast<uint2 *>(dst) = make_uint2(Pack<T>::two(y.x, y.y), Pack<T>::two(y.z, y.w));
    }
}

template <typename T, int D, int KEYS>
static int dkv_launch(const spamm_attn &a, const BackwardPlan &p, const T *d_do, int64_t do_token, int64_t do_head,
                      const float *delta, const float *factor, const unsigned *bits, const Item *items, const int *n_items,
                      float *partial, T *dk, T *dv, cudaStream_t stream)
{
    const size_t smem = 2 * KEYS * D * 2 + tk_slots(D, KEYS) * TK_ROWS * D * 2 + 2 * TK_ROWS * 128 + sizeof(TkCtrl) + p.chunk * 4;
    int st = attn_set_smem((const void *)attn_dkv_tc_kernel<T, D, KEYS>);
    if (st) return st;
    RowMap q_map, do_map;
    const int G = a.heads / a.kv_heads;
    attn_row_map(a, a.d_q, a.q_token, a.q_head, a.heads, G, max(1, p.box_tokens), &q_map);
    attn_row_map(a, d_do, do_token, do_head, a.heads, G, max(1, p.box_tokens), &do_map);
    attn_dkv_tc_kernel<T, D, KEYS><<<(unsigned)(p.groups * p.item_cap * (a.block / KEYS)), TK_THREADS, smem, stream>>>(
        a, p, q_map, do_map, d_do, do_token, do_head, delta, factor, bits, items, n_items, partial, dk, dv);
    return SPAMM_OK;
}

template <typename T, int D>
static int backward_launch(const spamm_attn &a, const BackwardPlan &p, const T *d_do, int64_t do_token, int64_t do_head, T *dq,
                           T *dk, T *dv, uint8_t *scratch, cudaStream_t stream)
{
    float *delta = reinterpret_cast<float *>(scratch + p.delta);
    unsigned *bits = reinterpret_cast<unsigned *>(scratch + p.bits);
    int *counts = reinterpret_cast<int *>(scratch + p.counts), *slots = reinterpret_cast<int *>(scratch + p.slots);
    Item *items = reinterpret_cast<Item *>(scratch + p.items);
    int *n_items = reinterpret_cast<int *>(scratch + p.n_items);
    float *partial = reinterpret_cast<float *>(scratch + p.partial);
    const bool half = std::is_same<T, __half>::value;
    float2 *norms = half ? reinterpret_cast<float2 *>(scratch + p.norms) : nullptr;
    float *factor = half ? reinterpret_cast<float *>(scratch + p.factor) : nullptr;
    const int64_t rows = (int64_t)a.tokens * a.heads, lists = (int64_t)a.batch * p.nqb * a.kv_heads;
    const int bq = min(a.query_block, a.max_q);
    const int tiles = (int)(((int64_t)bq * (a.heads / a.kv_heads) + 15) / 16);
    const int64_t dq_grid = p.groups * p.nqb * tiles;
    if ((rows + 31) / 32 > INT32_MAX || (lists + 3) / 4 > INT32_MAX || dq_grid > INT32_MAX || p.groups * p.item_cap > INT32_MAX / 2 ||
        p.groups * p.nkb > INT32_MAX)
        return attn_too_large();

    attn_delta_kernel<T, D><<<(unsigned)((rows + 31) / 32), 256, 0, stream>>>(a, fast_div(a.heads), p.G, d_do, do_token, do_head, delta, dq, dk, dv,
                                                                             reinterpret_cast<uint4 *>(bits), (p.slots - p.bits) / 16, norms);
    attn_turn_kernel<<<(unsigned)((lists + 3) / 4), 128, 0, stream>>>(a, p.nqb, p.nkb, p.words, bits, counts);
    attn_items_kernel<<<(unsigned)p.groups, 1024, 0, stream>>>(a, p, counts, slots, items, n_items, norms, factor);

    // (over more blocks than a union is built over, tiles of 16 rows whatever their number)
    int st;
    const int tq = attn_tiles(a);
    if (attn_big_tiles(a, (int64_t)min(a.n_select, p.nkb) * a.block) && attn_tile_fits(a) && p.nkb <= TQ_BLOCKS<D> && p.groups * tq <= INT32_MAX) {
        RowMap k_map, v_map;
        attn_row_maps(a, min(a.block, TQ_KEYS), &k_map, &v_map);
        const int entries = (int)min((int64_t)p.nkb, (int64_t)attn_tile_lists(a) * a.n_select);
        const size_t smem = 2 * TQ_ROWS * D * 2 + 3 * TQ_KEYS * D * 2 + sizeof(TqCtrl) + 6 * (size_t)entries;
        st = attn_set_smem((const void *)attn_dq_tc_kernel<T, D>);
        if (st) return st;
        attn_dq_tc_kernel<T, D><<<(unsigned)(p.groups * tq), TQ_THREADS, smem, stream>>>(
            a, tq, attn_tile_shape(a), entries, k_map, v_map, d_do, do_token, do_head, delta, factor, dq);
    } else {
        const size_t smem = (size_t)DQ_WARPS * DQ_STAGES * 2 * 16 * D * 2 + 2 * 16 * D * 2 + a.n_select * 4;
        st = attn_set_smem((const void *)attn_dq_rows_kernel<T, D>);
        if (st) return st;
        attn_dq_rows_kernel<T, D><<<(unsigned)dq_grid, 128, smem, stream>>>(a, p.nqb, tiles, d_do, do_token, do_head, delta, factor, dq);
    }

    switch (a.block) {
    case 16: st = dkv_launch<T, D, 16>(a, p, d_do, do_token, do_head, delta, factor, bits, items, n_items, partial, dk, dv, stream); break;
    case 32: st = dkv_launch<T, D, 32>(a, p, d_do, do_token, do_head, delta, factor, bits, items, n_items, partial, dk, dv, stream); break;
    default: st = dkv_launch<T, D, TK_MAX_KEYS>(a, p, d_do, do_token, do_head, delta, factor, bits, items, n_items, partial, dk, dv, stream); break;
    }
    if (st) return st;
    if (p.nqb > p.chunk)
        attn_dkv_join_kernel<T><<<dim3((unsigned)(p.groups * p.nkb), 8), 128, 0, stream>>>(a, p, counts, slots, partial, dk, dv);
    SPAMM_CUDA_TRY(cudaGetLastError());
    return SPAMM_OK;
}

}  // namespace spamm

using namespace spamm;

extern "C" size_t spamm_attn_backward_scratch_bytes(const spamm_attn *a)
{
    if (attn_check(a, false) || !a->batch || !a->max_q || !a->tokens || !backward_fits(*a)) return 0;
    return backward_plan(*a).bytes;
}

extern "C" int spamm_attn_backward_dev(const spamm_attn *a, const void *d_do, int64_t do_token, int64_t do_head, void *d_dq,
                                       void *d_dk, void *d_dv, void *d_scratch, size_t scratch_bytes, void *stream)
{
    int st = attn_check(a, true);
    if (st) return st;
    if (a->n_pages || !a->n_select)
        return attn_refuse("gradients need packed keys and lists");
    if (!(a->scale > 0.f) || !(a->scale <= 3e38f))
        return attn_refuse("scale is not a positive number");
    if (!a->tokens) return SPAMM_OK;
    if (!attn_rows_ok(a->d_q, a->q_token, a->q_head) || !attn_rows_ok(a->d_k, a->k_token, a->k_head) ||
        !attn_rows_ok(a->d_v, a->v_token, a->v_head) || !attn_rows_ok(a->d_o, a->o_token, a->o_head) || !a->d_lse ||
        !attn_rows_ok(d_do, do_token, do_head) || !attn_rows_ok(d_dq, 0, 0) || !attn_rows_ok(d_dk, 0, 0) || !attn_rows_ok(d_dv, 0, 0))
        return attn_refuse("q, k, v, o, lse and the gradients need rows on 16-byte boundaries");
    if (!a->batch || !a->max_q) {        // no sequence: all rows belong to none
        const size_t row = (size_t)a->tokens * a->dim * 2;
        SPAMM_CUDA_TRY(cudaMemsetAsync(d_dq, 0, row * a->heads, (cudaStream_t)stream));
        SPAMM_CUDA_TRY(cudaMemsetAsync(d_dk, 0, row * a->kv_heads, (cudaStream_t)stream));
        SPAMM_CUDA_TRY(cudaMemsetAsync(d_dv, 0, row * a->kv_heads, (cudaStream_t)stream));
        return SPAMM_OK;
    }
    if (reinterpret_cast<uintptr_t>(a->d_o_low) & 15) return attn_refuse("d_o_low is not on a 16-byte boundary");
    if (!backward_fits(*a)) return attn_too_large();
    const BackwardPlan p = backward_plan(*a);
    if (!d_scratch || scratch_bytes < p.bytes || (reinterpret_cast<uintptr_t>(d_scratch) & 15))
        return attn_refuse("scratch too small or not on a 16-byte boundary");
    uint8_t *scratch = static_cast<uint8_t *>(d_scratch);
    cudaStream_t str = (cudaStream_t)stream;
#define SPAMM_BACKWARD(T, D)                                                                                            \
    backward_launch<T, D>(*a, p, static_cast<const T *>(d_do), do_token, do_head, static_cast<T *>(d_dq),               \
                          static_cast<T *>(d_dk), static_cast<T *>(d_dv), scratch, str)
    if (a->dtype == SPAMM_ATTN_BF16) return a->dim == 64 ? SPAMM_BACKWARD(__nv_bfloat16, 64) : SPAMM_BACKWARD(__nv_bfloat16, 128);
    return a->dim == 64 ? SPAMM_BACKWARD(__half, 64) : SPAMM_BACKWARD(__half, 128);
#undef SPAMM_BACKWARD
}
