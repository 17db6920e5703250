// Attention over listed blocks, forward.
//
//   o_i = sum_j p_ij v_j,  p_ij = exp(scale q_i.k_j - lse_i),  lse_i = log sum_j exp(scale q_i.k_j)
//
// over the keys j of the blocks on the list of query i's block that i may see.  One pass over the keys with a running
// maximum and sum (both float); p is rounded to the type of v for the product, as v itself is: the tensor cores take 16 bits,
// and half a step of p, as independent from key to key as those of v, about doubles the square of the error of the result's own
// rounding.
#include <stdio.h>
#include <string.h>
#include <atomic>
#include <cudaTypedefs.h>
#include "attn.cuh"
#include "attn_tc.cuh"

namespace spamm {

bool attn_rows_ok(const void *p, int64_t token, int64_t head)
{
    return p && !(reinterpret_cast<uintptr_t>(p) & 15) && !(token & 7) && !(head & 7);
}

int attn_refuse(const char *why)
{
    static thread_local char msg[160];
    snprintf(msg, sizeof(msg), "spamm_attn: %s", why);
    record_error_text(msg);
    return SPAMM_ERR_INVALID;
}

int attn_too_large()
{
    record_error_text("spamm_attn: more blocks of threads than a launch can have");
    return SPAMM_ERR_UNSUPPORTED;
}

int attn_check(const spamm_attn *a, bool need_lists)
{
    if (!a) return SPAMM_ERR_INVALID;
    if (a->dtype != SPAMM_ATTN_BF16 && a->dtype != SPAMM_ATTN_HALF) return attn_refuse("dtype is neither bf16 nor half");
    if (a->dim != 64 && a->dim != 128) return attn_refuse("dim is neither 64 nor 128");
    if (a->block != 16 && a->block != 32 && a->block != 64 && a->block != 128)
        return attn_refuse("block is none of 16, 32, 64, 128");
    if (a->batch < 0 || a->tokens < 0 || a->max_q < 0) return attn_refuse("negative size");
    if (a->kv_heads < 1 || a->heads < a->kv_heads || a->heads % a->kv_heads || a->heads / a->kv_heads > 128)
        return attn_refuse("heads is no multiple of kv_heads, or more than 128 times it");
    if (a->query_block < 1) return attn_refuse("query_block below 1");
    if (a->n_select < 0 || a->n_select > SPAMM_ATTN_MAX_SELECT) return attn_refuse("n_select outside 0..1024");
    if (a->n_pages < 0 || a->table_width < 0 || (int64_t)a->table_width * a->block > INT32_MAX)
        return attn_refuse("n_pages or table_width out of range");
    if (!a->d_cu) return attn_refuse("d_cu is null");
    if (a->n_pages && ((a->batch && !a->d_lengths) || (a->batch && a->table_width && !a->d_table) || a->table_stride < a->table_width || !a->d_status))
        return attn_refuse("paged keys need d_lengths, d_table, a table_stride and d_status");
    if (need_lists && a->n_select && a->batch && a->max_q && !a->d_lists) return attn_refuse("d_lists is null");
    return SPAMM_OK;
}

// The limit of dynamic shared memory, 48 KB less the kernel's fixed part at first, belongs to a kernel and a device, whatever
// thread sets it: it is raised to all that the device has beside the fixed part, once in the process, and never lowered, so
// that no call can undo another's.  (The call costs about as much as a launch.)  Two threads may both raise it: to the same
// value.
int attn_set_smem(const void *kernel)
{
    struct Raised { std::atomic<const void *> kernel; std::atomic<uint64_t> devices; };
    constexpr int ROOM = 64;
    static Raised raised[ROOM];
    int device = 0;
    SPAMM_CUDA_TRY(cudaGetDevice(&device));
    Raised *mine = nullptr;
    for (int i = 0; i < ROOM && !mine; i++) {
        const void *k = raised[i].kernel.load();
        if (!k && raised[i].kernel.compare_exchange_strong(k, kernel)) k = kernel;     // (on failure k is the other thread's)
        if (k == kernel) mine = &raised[i];
    }
    const uint64_t bit = device < 64 ? 1ull << device : 0;
    if (mine && mine->devices.load() & bit) return SPAMM_OK;
    cudaFuncAttributes have;
    int most = 0;
    SPAMM_CUDA_TRY(cudaFuncGetAttributes(&have, kernel));
    SPAMM_CUDA_TRY(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device));
    SPAMM_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)have.sharedSizeBytes));
    if (mine) mine->devices.fetch_or(bit);
    return SPAMM_OK;
}

// Output rows that belong to no sequence become zero: part `part` of `parts` of those that lie before, inside (beyond
// max_q) and, for the last sequence, behind sequence s, for the query heads of key head h.
template <typename T>
static __device__ void zero_tail(const spamm_attn &a, const Seq &sq, int s, int h, int part, int parts)
{
    const int G = a.heads / a.kv_heads, vecs = G * a.dim / 8;
    const int end_own = min(max(a.d_cu[s + 1], sq.row0), a.tokens);
    const int end = s == a.batch - 1 ? a.tokens : end_own;
    const int begin = sq.row0 + sq.nq;
    const int lead = s == 0 ? sq.row0 : 0;
    const int rows = lead + (end - begin);
    for (int i = part; i < rows; i += parts) {
        const int row = i < lead ? i : begin + (i - lead);
        for (int x = threadIdx.x; x < vecs; x += blockDim.x) {
            const int head = h * G + x / (a.dim / 8), d = x % (a.dim / 8) * 8;
            *reinterpret_cast<uint4 *>(static_cast<T *>(a.d_o) + row * a.o_token + head * a.o_head + d) = make_uint4(0, 0, 0, 0);
        }
        if (a.d_lse)
            for (int g = threadIdx.x; g < G; g += blockDim.x) a.d_lse[(int64_t)row * a.heads + h * G + g] = -CUDART_INF_F;
    }
}

// Eight values to o, and what their rounding left to `low` (when given).
template <typename T> static __device__ __forceinline__ void store8(T *dst, T *low, const float *y)
{
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = Pack<T>::two(y[2 * i], y[2 * i + 1]);
    *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<uint4 *>(x);
    if (low) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 back = Pack<T>::to2(x[i]);
            x[i] = Pack<T>::two(y[2 * i] - back.x, y[2 * i + 1] - back.y);
        }
        *reinterpret_cast<uint4 *>(low) = *reinterpret_cast<uint4 *>(x);
    }
}

// How a call is cut: tiles of rows over the (queries x heads of a key head) of a query block, and ranges of keys.
struct RowsPlan {
    int bq, nqb;            // queries per query block (all of them without lists), query blocks
    int tiles;              // tiles of a query block
    int n_split;            // ranges of keys
    int split_keys;         // keys of a range, a multiple of the block
    int max_entries;        // blocks of a range
    bool cluster;           // the ranges of 16 rows are a cluster's blocks of threads, which join them
    bool pairs;             // pairs of tiles of 128 rows to a block of threads
    TileShape shape;        // of a tile of 128 rows
};

constexpr int ROWS_STAGES = 3;
constexpr int ROWS_WARPS = 4;
constexpr int ROWS_CLUSTER = 8;

__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// Shared memory of block `rank` of the cluster, at this block's address `p`.
__device__ __forceinline__ uint32_t cluster_addr(const void *p, int rank)
{
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(smem_addr(p)), "r"(rank));
    return there;
}
__device__ __forceinline__ float cluster_load(uint32_t at)
{
    float x;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
    return x;
}
__device__ __forceinline__ float4 cluster_load4(uint32_t at)
{
    float4 x;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x.x), "=f"(x.y), "=f"(x.z), "=f"(x.w) : "r"(at) : "memory");
    return x;
}

// 16 rows (queries x heads) of one key head against one range of its keys.  Each of the four warps takes every fourth
// chunk of 16 keys with a ring of three chunks of its own, so that nothing but the end synchronises the block; the four
// results are joined in shared memory.  Bound by the reading of keys and values when rows are few: 32 sequences of up to 16384
// keys, 8 key heads of 128 (1.43 GB), take 243 us, 5.9 TB/s, and 6 us to join the ranges; 16 lists of 32 pages of 64, 4 key
// heads (68 MB), 23 us with the joining, 2.9 TB/s.  There every block of threads finds its list, then the pages, then the keys, one wait on
// memory after the other, and has 28 chunks of 16 keys to hide them behind.
template <typename T, int D>
__global__ __launch_bounds__(128) void attn_rows_kernel(const __grid_constant__ spamm_attn a, const RowsPlan p,
                                                        float *part_o, float *part_lse)
{
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int TILE16 = 16 * D * 2;
    uint8_t *ring = smem;                                              // [warp][stage][K | V]
    uint8_t *q_tile = ring + ROWS_WARPS * ROWS_STAGES * 2 * TILE16;
    int *blk = reinterpret_cast<int *>(q_tile + TILE16);               // the list; then this range's blocks
    int64_t *base = reinterpret_cast<int64_t *>(blk + max(a.n_select, p.max_entries) + (max(a.n_select, p.max_entries) & 1));
    __shared__ int shared_count;

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned idx = blockIdx.x;
    const int split = idx % p.n_split; idx /= p.n_split;
    const int tile = idx % p.tiles; idx /= p.tiles;
    const int qb = idx % p.nqb; idx /= p.nqb;
    const int h = idx % a.kv_heads;
    const int s = idx / a.kv_heads;
    const int G = a.heads / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    if (a.zero_tail && split == 0) zero_tail<T>(a, sq, s, h, qb * p.tiles + tile, p.nqb * p.tiles);
    const int n_tok = min(p.bq, sq.nq - qb * p.bq);                    // queries of this query block
    const int64_t n_rows = (int64_t)max(n_tok, 0) * G;
    if ((int64_t)tile * 16 >= n_rows) return;
    const int rows = (int)min((int64_t)16, n_rows - tile * 16);
    const int tok0 = tile * 16 / G;
    const int first_query = qb * p.bq + tok0, last_query = qb * p.bq + (tile * 16 + rows - 1) / G;
    const int limit_max = attn_limit(a, sq, sq.pos0 + last_query);
    const int limit_min = attn_limit(a, sq, sq.pos0 + first_query);

    // Q tile: row r is query (tile*16 + r) / G of the block, head (tile*16 + r) % G of the group
    for (int i = tid; i < 16 * D / 8; i += 128) {
        const int r = i / (D / 8), c = i % (D / 8);
        const int x = tile * 16 + r;
        const bool ok = r < rows;
        const int64_t off = (sq.row0 + qb * p.bq + (int64_t)(ok ? x / G : 0)) * a.q_token + (int64_t)(h * G + (ok ? x % G : 0)) * a.q_head;
        cp_async16(smem_addr(q_tile) + tile_off<D>(r, c), static_cast<const T *>(a.d_q) + off + c * 8, ok);
    }
    cp_commit();

    const int n_blocks = ceil_div(limit_max, a.block);
    int count = n_blocks;
    if (a.n_select) {
        if (warp == 0) {
            const int all_blocks = ceil_div(attn_limit(a, sq, sq.pos0 + qb * p.bq + n_tok - 1), a.block);
            const int n = attn_load_list(a, s, qb, p.nqb, h, all_blocks, n_blocks, blk, lane);
            if (lane == 0) shared_count = n;
        }
        __syncthreads();
        count = shared_count;
    }
    // the blocks of a cluster wait for one another and share the keys evenly
    const int per_split = p.cluster ? ceil_div(count, p.n_split) : p.split_keys / a.block;
    const int e0 = min(split * per_split, count), e1 = min(e0 + per_split, count);
    // where each block's rows begin: for k; for v they begin at the same place in pages
    for (int e = e0 + tid; e < e1; e += 128) {
        const int b = a.n_select ? blk[e] : e;
        base[e - e0] = attn_block_base(a, sq, s, h, b, a.k_token, a.k_head);
    }
    __syncthreads();

    const int chunks_per_block = a.block >> 4;
    const int n_chunks = (e1 - e0) * chunks_per_block;
    const int64_t k_tok = a.n_pages ? D : a.k_token, v_tok = a.n_pages ? D : a.v_token;
    const uint32_t my_ring = smem_addr(ring) + warp * ROWS_STAGES * 2 * TILE16;

    auto chunk_pos = [&](int c) {
        const int e = c / chunks_per_block;
        const int b = a.n_select ? blk[e0 + e] : e0 + e;
        return b * a.block + (c - e * chunks_per_block) * 16;
    };
    auto issue = [&](int c, int stage) {
        if (c < n_chunks) {
            const int e = c / chunks_per_block;
            const int b = a.n_select ? blk[e0 + e] : e0 + e;
            const int off = (c - e * chunks_per_block) * 16;
            const int64_t kb = base[e];
            const int64_t vb = a.n_pages ? kb : (int64_t)(sq.row0 + b * a.block) * a.v_token + h * a.v_head;
            const int n = min(16, limit_max - (b * a.block + off));            // rows that some query may see
            const T *kp = static_cast<const T *>(a.d_k) + (kb >= 0 ? kb + off * k_tok : 0);
            const T *vp = static_cast<const T *>(a.d_v) + (kb >= 0 ? vb + off * v_tok : 0);
            const uint32_t kt = my_ring + stage * 2 * TILE16, vt = kt + TILE16;
#pragma unroll
            for (int i = 0; i < 16 * D / 8 / 32; i++) {
                const int x = i * 32 + lane, r = x / (D / 8), c8 = x % (D / 8);
                const bool ok = kb >= 0 && r < n;
                cp_async16(kt + tile_off<D>(r, c8), kp + (ok ? r * k_tok : 0) + c8 * 8, ok);
                cp_async16(vt + tile_off<D>(r, c8), vp + (ok ? r * v_tok : 0) + c8 * 8, ok);
            }
        }
        cp_commit();
    };
    for (int i = 0; i < ROWS_STAGES - 1; i++) issue(warp + ROWS_WARPS * i, i);

    cp_wait<ROWS_STAGES - 1>();
    __syncthreads();                       // the Q tile, loaded by all threads
    uint32_t qf[D / 16][4];
#pragma unroll
    for (int ks = 0; ks < D / 16; ks++) a_frag<D>(smem_addr(q_tile), 0, ks, lane, qf[ks]);

    int limit[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const int r = (lane >> 2) + 8 * x;
        limit[x] = r < rows ? attn_limit(a, sq, sq.pos0 + qb * p.bq + (tile * 16 + r) / G) : limit_max;
    }
    const float scale2 = a.scale * LOG2E;
    float o[D / 8][4] = {};
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};

    int stage = 0;
    for (int c = warp; c < n_chunks; c += ROWS_WARPS) {
        issue(c + ROWS_WARPS * (ROWS_STAGES - 1), (stage + ROWS_STAGES - 1) % ROWS_STAGES);
        cp_wait<ROWS_STAGES - 1>();
        __syncwarp();
        const uint32_t kt = my_ring + stage * 2 * TILE16, vt = kt + TILE16;
        stage = stage + 1 == ROWS_STAGES ? 0 : stage + 1;
        float sc[2][4] = {};
#pragma unroll
        for (int ks = 0; ks < D / 16; ks++) {
            uint32_t b[4];
            b_frag2<D>(kt, 0, ks, lane, b);
            mma16816<T>(sc[0], qf[ks], b[0], b[1]);
            mma16816<T>(sc[1], qf[ks], b[2], b[3]);
        }
        const int p0 = base[c / chunks_per_block] < 0 ? INT32_MAX - 64 : chunk_pos(c);
        const bool masked = p0 > limit_min - 16;
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int nt = 0; nt < 2; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = sc[nt][i] * scale2;
                if (masked && p0 + nt * 8 + (lane & 3) * 2 + (i & 1) >= limit[i >> 1]) v = -CUDART_INF_F;
                sc[nt][i] = v;
                top[i >> 1] = fmaxf(top[i >> 1], v);
            }
#pragma unroll
        for (int x = 0; x < 2; x++) {
            top[x] = fmaxf(top[x], __shfl_xor_sync(~0u, top[x], 1));
            top[x] = fmaxf(top[x], __shfl_xor_sync(~0u, top[x], 2));
        }
        if (__any_sync(~0u, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const float f = m[x] == top[x] ? 1.f : fast_exp2(m[x] - top[x]);   // equal: also -inf against -inf
                l[x] *= f;
                m[x] = top[x];
#pragma unroll
                for (int n = 0; n < D / 8; n++) { o[n][2 * x] *= f; o[n][2 * x + 1] *= f; }
            }
        }
        const float m0 = m[0] == -CUDART_INF_F ? 0.f : m[0], m1 = m[1] == -CUDART_INF_F ? 0.f : m[1];
#pragma unroll
        for (int nt = 0; nt < 2; nt++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sc[nt][i] = fast_exp2(sc[nt][i] - (i < 2 ? m0 : m1));
                l[i >> 1] += sc[nt][i];
            }
        const uint32_t pf[4] = {Pack<T>::two(sc[0][0], sc[0][1]), Pack<T>::two(sc[0][2], sc[0][3]),
                                Pack<T>::two(sc[1][0], sc[1][1]), Pack<T>::two(sc[1][2], sc[1][3])};
#pragma unroll
        for (int n = 0; n < D / 16; n++) {
            uint32_t b[4];
            bt_frag2<D>(vt, 0, n * 16, lane, b);
            mma16816<T>(o[2 * n], pf, b[0], b[1]);
            mma16816<T>(o[2 * n + 1], pf, b[2], b[3]);
        }
        __syncwarp();
    }
    cp_wait<0>();
#pragma unroll
    for (int x = 0; x < 2; x++) {
        l[x] += __shfl_xor_sync(~0u, l[x], 1);
        l[x] += __shfl_xor_sync(~0u, l[x], 2);
    }
    __syncthreads();
    // join the four warps: [warp][16][D] sums, then maxima and sums of the rows
    float *so = reinterpret_cast<float *>(ring);
    float *sm = so + ROWS_WARPS * 16 * D, *sl = sm + ROWS_WARPS * 16;
    float *range_o = sl + ROWS_WARPS * 16, *range_lse = range_o + 16 * D;        // of the rows, for the cluster
#pragma unroll
    for (int n = 0; n < D / 8; n++)
#pragma unroll
        for (int x = 0; x < 2; x++)
            *reinterpret_cast<float2 *>(so + ((warp * 16 + (lane >> 2) + 8 * x) * D + n * 8 + (lane & 3) * 2)) =
                make_float2(o[n][2 * x], o[n][2 * x + 1]);
    if ((lane & 3) == 0)
#pragma unroll
        for (int x = 0; x < 2; x++) {
            sm[warp * 16 + (lane >> 2) + 8 * x] = m[x];
            sl[warp * 16 + (lane >> 2) + 8 * x] = l[x];
        }
    __syncthreads();
    const int r = tid >> 3, c0 = (tid & 7) * (D / 8);
    __shared__ unsigned odd_rows;
    if (tid == 0) odd_rows = 0;
    bool odd = false;
    if (r < rows) {
        float top = -CUDART_INF_F, f[ROWS_WARPS], total = 0.f;
#pragma unroll
        for (int w = 0; w < ROWS_WARPS; w++) top = fmaxf(top, sm[w * 16 + r]);
        const float t0 = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll
        for (int w = 0; w < ROWS_WARPS; w++) {
            f[w] = fast_exp2(sm[w * 16 + r] - t0);
            total += sl[w * 16 + r] * f[w];
        }
        // no visible key: no sum, output zero.  (A NaN among the scores stays: total is then NaN, not zero.)
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const float lse2 = total == 0.f ? -CUDART_INF_F : t0 + log2f(total);
        float y[D / 8] = {};
#pragma unroll
        for (int w = 0; w < ROWS_WARPS; w++)
#pragma unroll
            for (int i = 0; i < D / 8; i++) y[i] += so[(w * 16 + r) * D + c0 + i] * f[w];
#pragma unroll
        for (int i = 0; i < D / 8; i++) odd |= not_finite(__float_as_uint(y[i] * inv));
        odd = odd && total == total;
        const int x = tile * 16 + r;
        const int64_t row = sq.row0 + qb * p.bq + x / G;
        const int head = h * G + x % G;
        if (p.n_split == 1) {
#pragma unroll
            for (int i = 0; i < D / 8; i++) y[i] *= inv;
            T *dst = static_cast<T *>(a.d_o) + row * a.o_token + head * a.o_head + c0;
            T *low = a.d_o_low ? static_cast<T *>(a.d_o_low) + (row * a.heads + head) * D + c0 : nullptr;
#pragma unroll
            for (int i = 0; i < D / 64; i++) store8<T>(dst + 8 * i, low ? low + 8 * i : nullptr, y + 8 * i);
            if (a.d_lse && (tid & 7) == 0) a.d_lse[row * a.heads + head] = lse2 * LN2;
        } else {
            const int64_t at = (row * a.heads + head) * p.n_split + split;
            float *dst = p.cluster ? range_o + r * D : part_o + at * D;
#pragma unroll
            for (int i = 0; i < D / 8; i += 4)
                *reinterpret_cast<float4 *>(dst + c0 + i) = make_float4(y[i] * inv, y[i + 1] * inv, y[i + 2] * inv, y[i + 3] * inv);
            if ((tid & 7) == 0) *(p.cluster ? range_lse + r : part_lse + at) = lse2;
        }
    }
    const bool any_odd = __syncthreads_or(odd);
    // rows that are not finite once more, over their own keys alone (see row_keys)
    __shared__ uint32_t sure[D];
    if (any_odd) {
        if (odd) atomicOr(&odd_rows, 1u << r);
        if (tid < D) sure[tid] = 0;
        __syncthreads();
        sure_columns<T, D>(a, sq, s, h, static_cast<const T *>(a.d_v), a.v_token, a.v_head, e1 - e0, e0, nullptr,
                           a.n_select ? blk + e0 : nullptr, nullptr, limit_min, sure, tid, 128);
        __syncthreads();
    }
#pragma unroll 1
    for (int sr = warp; sr < rows && any_odd; sr += ROWS_WARPS) {
        if (!(odd_rows >> sr & 1)) continue;
        const int x = tile * 16 + sr, query = qb * p.bq + x / G, head = h * G + x % G;
        const int64_t row = sq.row0 + query;
        const int64_t at = (row * a.heads + head) * p.n_split + split;
        bool open = false;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) {
            const int d = lane * (D / 32) + i;
            const float2 got = p.n_split == 1 ? Pack<T>::to2(*reinterpret_cast<const uint32_t *>(static_cast<const T *>(a.d_o) + row * a.o_token + head * a.o_head + d))
                                              : *reinterpret_cast<const float2 *>((p.cluster ? range_o + sr * D : part_o + at * D) + d);
            open |= unsure(got, sure, d, ~0u);
        }
        if (!__any_sync(~0u, open)) continue;
        float q[D / 32], k[D / 32], v[D / 32], y[D / 32] = {}, top = -CUDART_INF_F, sum = 0.f;
        row_load<T, D>(static_cast<const T *>(a.d_q) + row * a.q_token + head * a.q_head, lane, q);
        row_keys<T>(a, sq, s, h, e1 - e0, attn_limit(a, sq, sq.pos0 + query), [&](int e) { return a.n_select ? blk[e0 + e] : e0 + e; },
                    [&](const T *kr, const T *vr) {
                        row_load<T, D>(kr, lane, k);
                        row_load<T, D>(vr, lane, v);
                        online_row<D>(row_dot<D>(q, k) * scale2, v, y, &top, &sum);
                    });
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
        for (int i = 0; i < D / 32; i += 2) {
            const int d = lane * (D / 32) + i;
            if (p.n_split == 1) {
                const uint32_t z = Pack<T>::two(y[i] * inv, y[i + 1] * inv);
                *reinterpret_cast<uint32_t *>(static_cast<T *>(a.d_o) + row * a.o_token + head * a.o_head + d) = z;
                const float2 back = Pack<T>::to2(z);
                if (a.d_o_low)
                    *reinterpret_cast<uint32_t *>(static_cast<T *>(a.d_o_low) + (row * a.heads + head) * D + d) =
                        Pack<T>::two(y[i] * inv - back.x, y[i + 1] * inv - back.y);
            } else {
                *reinterpret_cast<float2 *>((p.cluster ? range_o + sr * D : part_o + at * D) + d) = make_float2(y[i] * inv, y[i + 1] * inv);
            }
        }
    }
    if (!p.cluster) return;
    // the ranges joined as by attn_join_kernel, each block a share of the rows' pieces of eight values
    cluster_barrier();
    for (int i = split * 128 + tid; i < rows * (D / 8); i += p.n_split * 128) {
        const int jr = i / (D / 8), d = i % (D / 8) * 8;
        float lse[ROWS_CLUSTER], top = -CUDART_INF_F, total = 0.f, y[8] = {};
#pragma unroll
        for (int j = 0; j < ROWS_CLUSTER; j++) {
            lse[j] = j < p.n_split ? cluster_load(cluster_addr(range_lse + jr, j)) : -CUDART_INF_F;
            top = fmaxf(top, lse[j]);
        }
        const float t0 = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll
        for (int j = 0; j < ROWS_CLUSTER; j++) {
            if (lse[j] == -CUDART_INF_F) continue;
            const float f = fast_exp2(lse[j] - t0);
            const uint32_t from = cluster_addr(range_o + jr * D + d, j);
            const float4 u = cluster_load4(from), v = cluster_load4(from + 16);
            total += f;
            y[0] += f * u.x; y[1] += f * u.y; y[2] += f * u.z; y[3] += f * u.w;
            y[4] += f * v.x; y[5] += f * v.y; y[6] += f * v.z; y[7] += f * v.w;
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
        for (int k = 0; k < 8; k++) y[k] *= inv;
        const int x = tile * 16 + jr, head = h * G + x % G;
        const int64_t row = sq.row0 + qb * p.bq + x / G;
        store8<T>(static_cast<T *>(a.d_o) + row * a.o_token + head * a.o_head + d,
                  a.d_o_low ? static_cast<T *>(a.d_o_low) + (row * a.heads + head) * D + d : nullptr, y);
        if (a.d_lse && d == 0) a.d_lse[row * a.heads + head] = total == 0.f ? -CUDART_INF_F : (t0 + log2f(total)) * LN2;
    }
    cluster_barrier();                       // no block leaves while another reads its shared memory
}

// ---- pairs of tiles of 128 rows on the tensor memory path
//
// Per block of threads: two tiles of 128 rows (queries x heads of a key head) against a range of their keys, 128 keys (the
// blocks of the union of their lists one behind the other) at a time.  S = Q K^T goes to tensor memory; two threads for each
// row, half of the keys each, take the running maximum and write p over S in the type of v (one warp per scheduler and tile
// would not overlap its exponentials with its other instructions); O += P V takes p from tensor memory.  One warp issues the
// products of the two tiles in turn, so that one tile's exponentials run beside the other's products (two independent blocks
// per SM fall into step instead: both multiply, then both exponentiate).  K and V are shared by the pair and double
// buffered; one warp feeds them, a tensor copy for each block of keys and 64 values; the block in which the sequence ends is
// copied 16 bytes a time with zeros behind the last key (what lies there may be NaN).
//
// The running maximum is only raised when a row's scores exceed it by more than 2^8: until then p stays below 2^8, which
// both types and the float sums hold without loss, and O need not be rescaled in tensor memory.
//
// Where pairs would not fill the GPU, and wherever keys are listed, single tiles (TILES 1) with one buffer each for K and V:
// two blocks of threads per SM.
//
// A step of 128 keys and two tiles is 2 x 8 products of N = 128 for S and as many for O (about 66 clocks each, 2100 in all for
// D = 128), and 2 x 128 x 128 exponentials, 2048 clocks of the SM's special-function units if those took all of them, beside the
// multiplications, maxima, sums and conversions.  Bound by the chain of a step rather than by either: S has one buffer for a
// tile, p lies over it, and O += P V waits for all of p.  Two chunks of 1024 and 750 tokens over 32768 and 24006 keys, 32 heads
// of 128 (832 GFLOP): 870 to 882 us, 0.94 to 0.96 PFLOP/s.  Three of 16 pairs of exponentials by the polynomial: 853 us; none
// 860, six 863, eight 885, one per cent for a fifth of the unit's work.  Listed keys, 3 sequences of up to 8192, 16 blocks of 64 (276 GFLOP):
// 470 us, 0.59 PFLOP/s; a tile has 8 steps of 128 keys there, and its beginning and end weigh.
constexpr int TC_ROWS = 128, TC_KEYS = 128, TC_HALF = TC_KEYS / 2;
constexpr int TC_ENTRIES = 2048;        // blocks of a union, at most
constexpr int TC_POLY = 3;              // of 16 pairs of exponentials, those that the polynomial takes

struct TcCtrl {
    uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], pv_done[2];
    uint64_t met[8];                    // [tile][32 rows]: the two warps of the rows have left their maxima
    uint32_t tmem_base;
    uint32_t abort_flag;
    int32_t err;
    int32_t count;
    int32_t bad_page;
    uint32_t odd[2][4];                 // [tile]: rows whose result is not finite
    int32_t pad[3];
    float top[2][2][2][TC_ROWS];        // [tile][step & 1][half][row]
};

// The 256 threads of a tile meet.
static __device__ __forceinline__ void tile_barrier(int tile)
{
    asm volatile("bar.sync %0, 256;" ::"r"(tile + 1) : "memory");
}

template <typename T, int D, int TILES>
__global__ __launch_bounds__(TILES * 256 + 64, TILES == 1 ? 2 : 1) void attn_tc_kernel(const __grid_constant__ spamm_attn a, const __grid_constant__ RowsPlan p,
                                                                const __grid_constant__ RowMap k_map,
                                                                const __grid_constant__ RowMap v_map, float *part_o,
                                                                float *part_lse)
{
    extern __shared__ __align__(1024) uint8_t smem_tc[];
    constexpr int TILE = 128 * D * 2, STAGES = TILES, THREADS = TILES * 256 + 64, W_MMA = TILES * 8, W_LOAD = W_MMA + 1;
    constexpr int COLS = TILES * 256;                                  // S (P over it) of the tiles, then O
    uint8_t *const smem = smem_tc;
    const uint32_t q_tiles = smem_u32(smem), k_ring = q_tiles + TILES * TILE, v_ring = k_ring + STAGES * TILE;
    TcCtrl *ctrl = reinterpret_cast<TcCtrl *>(smem + 3 * TILES * TILE);
    const bool listed = TILES == 1 && a.n_select;
    uint32_t *bits = reinterpret_cast<uint32_t *>(ctrl + 1);           // [max_entries], with lists
    uint16_t *idx = reinterpret_cast<uint16_t *>(bits + (listed ? p.max_entries : 0));

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned where = blockIdx.x;
    // tiles that read the same keys run side by side, those with the longest causal rows first
    const int pair = p.tiles - 1 - where % p.tiles; where /= p.tiles;      // of tiles (or one tile)
    const int split = where % p.n_split; where /= p.n_split;
    const int h = where % a.kv_heads;
    const int s = where / a.kv_heads;
    const int G = a.heads / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    if (a.zero_tail && split == 0) zero_tail<T>(a, sq, s, h, pair, p.tiles);
    const TileRows tr[2] = {attn_tile(a, p.shape, sq, TILES * pair), TILES == 2 ? attn_tile(a, p.shape, sq, 2 * pair + 1) : TileRows{}};
    if (!tr[0].rows) return;
    const int limits[2] = {attn_limit(a, sq, sq.pos0 + tr[0].last), tr[1].rows ? attn_limit(a, sq, sq.pos0 + tr[1].last) : 0};
    const int limit_max = max(limits[0], limits[1]);

    if (warp < W_MMA) {
        // the queries of the warp's tile
        const int x0 = warp >> 3, t = tid & 255;
        const TileRows mine = x0 ? tr[1] : tr[0];
        constexpr int PASS = 256 / (D / 8);                            // rows at a time
        const int c = t % (D / 8);
        const T *src = static_cast<const T *>(a.d_q) + (int64_t)sq.row0 * a.q_token + (int64_t)h * G * a.q_head + c * 8;
#pragma unroll
        for (int qr = t / (D / 8); qr < TC_ROWS; qr += PASS) {
            const bool ok = qr < mine.rows;
            const int qy = mine.row0 + (ok ? qr : 0), tok = (int)p.shape.G.quotient(qy);
            cp_async16(q_tiles + x0 * TILE + panel_off(128, qr, c), src + tok * a.q_token + (qy - tok * G) * a.q_head, ok);
        }
        cp_commit();
    } else if (warp == W_MMA) {
        if (lane == 0) {
            for (int i = 0; i < 2; i++) {
                mbar_init(smem_u32(&ctrl->q_full[i]), 256);
                mbar_init(smem_u32(&ctrl->k_full[i]), 32);
                mbar_init(smem_u32(&ctrl->v_full[i]), 32);
                mbar_init(smem_u32(&ctrl->k_empty[i]), 1);
                mbar_init(smem_u32(&ctrl->v_empty[i]), 1);
                mbar_init(smem_u32(&ctrl->s_full[i]), 1);
                mbar_init(smem_u32(&ctrl->pv_done[i]), 1);
                mbar_init(smem_u32(&ctrl->p_full[i]), 256);
            }
            for (int i = 0; i < 8; i++) mbar_init(smem_u32(&ctrl->met[i]), 64);
            ctrl->abort_flag = 0;
            ctrl->err = 0;
            ctrl->bad_page = 0;
            for (int i = 0; i < 8; i++) ctrl->odd[i >> 2][i & 3] = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        tmem_alloc<COLS>(smem_u32(&ctrl->tmem_base));
        tc_fence_before();
    }
    const int log_block = 31 - __clz(a.block);
    const int b0 = min(split * (p.split_keys >> log_block), ceil_div(limit_max, a.block));
    const int b1 = min(b0 + (p.split_keys >> log_block), ceil_div(limit_max, a.block));
    int n_entries = b1 - b0;
    if (listed) {
        n_entries = attn_union<THREADS>(a, sq, s, h, tr[0], b0, b1, reinterpret_cast<uint32_t *>(smem + TILE), idx, bits, &ctrl->count);
    } else {
        __syncthreads();
        if (a.n_pages) {
            for (int e = tid; e < n_entries; e += THREADS) {
                const int page = a.d_table[(int64_t)s * a.table_stride + b0 + e];
                if (page < 0 || page >= a.n_pages) {
                    ctrl->bad_page = 1;
                    *a.d_status = SPAMM_ERR_INVALID;
                }
            }
            __syncthreads();
        }
    }
    tc_fence_after();
    // block of keys of entry e
    auto block_of = [&](int e) { return b0 + (listed ? (int)idx[e] : e); };
    auto page_of = [&](int b) { return a.d_table[(int64_t)s * a.table_stride + b]; };
    const int n_keys = n_entries << log_block, per_tile = TC_KEYS >> log_block;
    const int n_tiles = (n_keys + TC_KEYS - 1) / TC_KEYS;
    // whether some row of tile x reads keys of step j
    auto uses = [&](bool second, int j) {
        if (second && !tr[1].rows) return false;
        if (!listed) return (b0 << log_block) + j * TC_KEYS < (second ? limits[1] : limits[0]);
        bool any = false;
        for (int i = 0; i < per_tile; i++) {
            const int e = j * per_tile + i;
            any |= e < n_entries && bits[e] != 0;
        }
        return any;
    };
    const uint32_t tmem = ctrl->tmem_base, tmem_o = tmem + TILES * TC_KEYS;
    const WaitState ws{&ctrl->abort_flag, &ctrl->err};

    if (warp == W_LOAD) {
        // ---- K and V
        // lane's copies of a step: entry j * per_tile + my_i, values 64 * my_panel ..
        const int my_i = lane / (D / 64), my_panel = lane % (D / 64);
        // where they begin: the row of packed keys, or page * kv_heads + head; -1: not there, -2: to be copied by hand
        struct At { int row, pos; };
        auto look_up = [&](int j) {
            At at{-1, 0};
            const int e = j * per_tile + my_i;
            if (my_i < per_tile && e < n_entries) {
                const int b = block_of(e);
                at.pos = b * a.block;
                at.row = sq.row0 + at.pos;
                if (a.n_pages) {
                    const int page = page_of(b);
                    at.row = page < 0 || page >= a.n_pages ? -2 : page * a.kv_heads + h;
                }
                if (at.pos + a.block > sq.nk) at.row = -2;
            }
            return at;
        };
        // every lane takes part in the barrier's phase with the bytes of its tensor copy and one arrival
        auto load = [&](int j, const At &at, bool value, uint32_t dst, uint64_t *full) {
            const uint32_t bar = smem_u32(full);
            const RowMap &rm = value ? v_map : k_map;
            if (at.row >= 0 && rm.usable) {
                mbar_expect_tx(bar, a.block * 128);
                int y = 0, z = at.row;
                if (!a.n_pages) {
                    y = rm.swapped ? at.row : h;
                    z = rm.swapped ? h : at.row;
                }
                tma_box(dst + my_panel * (128 * 128) + (my_i << log_block) * 128, &rm.map, my_panel * 64, y, z, bar);
            }
            if (__any_sync(~0u, at.row == -2 || (at.row >= 0 && !rm.usable))) {
                const T *src0 = static_cast<const T *>(value ? a.d_v : a.d_k);
                const int64_t tok = a.n_pages ? D : value ? a.v_token : a.k_token;
                for (int i = 0; i < per_tile; i++) {
                    const int e = j * per_tile + i;
                    if (e >= n_entries) break;
                    const int b = block_of(e), pos = b * a.block;
                    int n = sq.nk - pos;                               // keys of the block that are there
                    int64_t from = (int64_t)(sq.row0 + pos) * tok + h * (value ? a.v_head : a.k_head);
                    bool page_ok = true;
                    if (a.n_pages) {
                        const int page = page_of(b);
                        page_ok = page >= 0 && page < a.n_pages;
                        from = ((int64_t)page * a.kv_heads + h) * a.block * D;
                    }
                    if (page_ok && rm.usable && n >= a.block) continue;
                    if (!page_ok) n = 0;
                    for (int x = lane; x < a.block * (D / 8); x += 32) {
                        const int r = x / (D / 8), c = x % (D / 8);
                        cp_async16(dst + panel_off(128, (i << log_block) + r, c), src0 + (r < n ? from + r * tok : 0) + c * 8, r < n);
                    }
                }
                cp_commit();
                cp_wait<0>();
                fence_async_smem();
            }
            mbar_arrive(bar);
        };
        bool fine = true;
        At at = look_up(0);
        for (int j = 0; j < n_tiles; j++) {
            const At next = look_up(j + 1);
            const int b = j % STAGES, round = j / STAGES;
            if (round) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->k_empty[b]), round - 1, 1));
            if (!fine) break;
            load(j, at, false, k_ring + b * TILE, &ctrl->k_full[b]);
            if (round) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->v_empty[b]), round - 1, 2));
            if (!fine) break;
            load(j, at, true, v_ring + b * TILE, &ctrl->v_full[b]);
            at = next;
        }
        __syncthreads();
    } else if (warp == W_MMA) {
        // ---- products: for each tile in turn, O of the step before, then S of this one.  They run in the order of their
        // issue: S may be written where p is still being read.
        if (n_tiles) {
            constexpr uint32_t s_desc = mma_desc<T>(128, TC_KEYS, false, false), o_desc = mma_desc<T>(128, D, false, true);
            const uint32_t base = __shfl_sync(~0u, tmem, 0);
            const uint64_t q_desc = desc_k_major(q_tiles), k_desc = desc_k_major(k_ring), v_desc = desc_mn_major(v_ring, 128);
            bool fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->q_full[0]), 0, 3) && (!tr[1].rows || ws.wait(smem_u32(&ctrl->q_full[1]), 0, 3)));
            int done[2] = {0, 0};                                      // steps whose O has been issued
            bool used[2] = {false, false};                             // by the step before
            for (int j = 0; j <= n_tiles && fine; j++) {
                const int kb = j % STAGES, vb = j ? (j - 1) % STAGES : 0;
                if (j) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->v_full[vb]), (j - 1) / STAGES, 5));
                // keys behind the last block of the range take no part: their rows of V were never written
                const int steps = min(TC_KEYS, n_keys - (j - 1) * TC_KEYS) / 16;
#pragma unroll
                for (int x = 0; x < TILES && fine; x++) {
                    const bool use = j < n_tiles && uses(x, j);
                    if (used[x]) {
                        fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->p_full[x]), done[x], 4));
                        if (!fine) break;
                        tc_fence_after();
                        const uint64_t vd = v_desc + vb * (TILE >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < TC_KEYS / 16; ks++)
                                if (ks < steps)
                                    mma_ts(base + (TILES * TC_KEYS + x * 128), base + x * TC_KEYS + (ks >> 2) * TC_HALF + (ks & 3) * 8,
                                           vd + step_mn_major(ks), o_desc, done[x] || ks);
                            umma_commit(smem_u32(&ctrl->pv_done[x]));
                        }
                        __syncwarp();
                        done[x]++;
                    }
                    if (x == 0 && j < n_tiles) fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->k_full[kb]), j / STAGES, 6));
                    if (!fine) break;
                    if (use) {
                        tc_fence_after();
                        const uint64_t qd = q_desc + x * (TILE >> 4), kd = k_desc + kb * (TILE >> 4);
                        if (elect_one()) {
#pragma unroll
                            for (int ks = 0; ks < D / 16; ks++)
                                mma_ss(base + x * TC_KEYS, qd + step_k_major(128, ks), kd + step_k_major(128, ks), s_desc, ks != 0);
                            umma_commit(smem_u32(&ctrl->s_full[x]));
                        }
                        __syncwarp();
                    }
                    used[x] = use;
                }
                if (fine && elect_one()) {
                    if (j) umma_commit(smem_u32(&ctrl->v_empty[vb]));
                    if (j < n_tiles) umma_commit(smem_u32(&ctrl->k_empty[kb]));
                }
                __syncwarp();
            }
        }
        __syncwarp();
        __syncthreads();
    } else {
        // ---- softmax: two threads for a row of the warp's tile, each half of the keys
        const int x0 = warp >> 3, half = warp >> 2 & 1, quad = warp & 3;
        const TileRows mine = x0 ? tr[1] : tr[0];
        const int rows = mine.rows;
        cp_wait<0>();
        fence_async_smem();
        mbar_arrive(smem_u32(&ctrl->q_full[x0]));
        const int r = tid & 127;
        const int y = mine.row0 + min(r, max(rows, 1) - 1), my_query = (int)p.shape.G.quotient(y);
        const int limit = attn_limit(a, sq, sq.pos0 + my_query), limit_min = attn_limit(a, sq, sq.pos0 + mine.first);
        const uint32_t my_bit = listed ? 1u << (my_query / a.query_block - mine.qb0) : 1u;
        const uint32_t all_bits = mine.n_qb == 32 ? ~0u : (1u << mine.n_qb) - 1;
        const float scale2 = a.scale * LOG2E;
        const uint32_t lane_s = tmem + ((uint32_t)(quad * 32) << 16) + x0 * TC_KEYS + half * TC_HALF;
        const uint32_t lane_o = tmem_o + ((uint32_t)(quad * 32) << 16) + x0 * 128 + half * (D / 2);
        const uint32_t met = smem_u32(&ctrl->met[x0 * 4 + quad]);
        float m = -CUDART_INF_F, l = 0.f;
        bool fine = true;
        int n_done = 0;
        for (int j = 0; j < n_tiles && rows; j++) {
            if (!uses(x0, j)) continue;
            // lanes 0..3: position and lists of this half's groups of 16 keys (far behind every limit: none there)
            int group_pos = INT32_MAX / 2;
            uint32_t group_bits = all_bits;
            if (lane < TC_HALF / 16) {
                const int key = j * TC_KEYS + half * TC_HALF + lane * 16, e = key >> log_block;
                if (e < n_entries) {
                    const int b = block_of(e);
                    group_pos = b * a.block + (key & (a.block - 1));
                    if (listed) group_bits = bits[e];
                    else if (ctrl->bad_page) {
                        const int page = page_of(b);
                        if (page < 0 || page >= a.n_pages) group_pos = INT32_MAX / 2;
                    }
                }
            }
            const bool masked = __any_sync(~0u, (lane < TC_HALF / 16 && group_pos > limit_min - 16) || group_bits != all_bits);
            fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->s_full[x0]), n_done, 7));
            if (!fine) break;
            tc_fence_after();
            uint32_t v[TC_HALF];
            tmem_ld32(lane_s, v);
            tmem_ld32(lane_s + 32, v + 32);
            tmem_wait_ld();
            tmem_landed<TC_HALF>(v);
            if (masked) {
#pragma unroll
                for (int g = 0; g < TC_HALF / 16; g++) {
                    const int pos = __shfl_sync(~0u, group_pos, g);
                    const int n = __shfl_sync(~0u, group_bits, g) & my_bit ? limit - pos : 0;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (i >= n) v[g * 16 + i] = 0xff800000u;
                }
            }
            float t0 = __uint_as_float(v[0]), t1 = __uint_as_float(v[1]);
#pragma unroll
            for (int i = 0; i < TC_HALF; i += 4) {
                t0 = fmaxf(t0, fmaxf(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
                t1 = fmaxf(t1, fmaxf(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])));
            }
            float top = fmaxf(t0, t1);
            ctrl->top[x0][n_done & 1][half][r] = top;
            mbar_arrive(met);
            fine = __all_sync(~0u, ws.wait(met, n_done, 10));
            if (!fine) break;
            top = fmaxf(top, ctrl->top[x0][n_done & 1][half ^ 1][r]) * scale2;
            const bool raise = top > m + 8.f || (m == -CUDART_INF_F && top > m);
            if (__any_sync(~0u, raise)) {
                const float f = raise ? fast_exp2(m - top) : 1.f;
                if (raise) { m = top; l *= f; }
                // the products before this S are complete, O is at rest; each thread takes half of its columns
                if (n_done) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t w[16];
                        tmem_ld16(lane_o + c * 16, w);
                        tmem_wait_ld();
                        tmem_landed<16>(w);
#pragma unroll
                        for (int i = 0; i < 16; i++) w[i] = __float_as_uint(__uint_as_float(w[i]) * f);
                        tmem_st16(lane_o + c * 16, w);
                    }
                }
            }
            const float m0 = m == -CUDART_INF_F ? 0.f : m;
            const float2 scale22 = make_float2(scale2, scale2), minus_m = make_float2(-m0, -m0);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int c = 0; c < TC_HALF / 32; c++) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float2 z = fma2(make_float2(__uint_as_float(v[c * 32 + 2 * i]), __uint_as_float(v[c * 32 + 2 * i + 1])), scale22, minus_m);
                    // spread evenly, so that both units are busy all the time
                    const float2 e = i * TC_POLY / 16 != (i + 1) * TC_POLY / 16 ? poly_exp2(z) : make_float2(fast_exp2(z.x), fast_exp2(z.y));
                    sum = add2(sum, e);
                    w[i] = Pack<T>::two(e.x, e.y);
                }
                tmem_st16(lane_s + c * 16, w);              // over this thread's S, which is in registers
            }
            l += sum.x + sum.y;
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(smem_u32(&ctrl->p_full[x0]));
            n_done++;
        }
        if (n_done && fine) {
            fine = __all_sync(~0u, ws.wait(smem_u32(&ctrl->pv_done[x0]), n_done - 1, 9));
            // the row's sum: both halves, in the same order for both threads
            ctrl->top[x0][n_done & 1][half][r] = l;
            mbar_arrive(met);
            fine = fine && __all_sync(~0u, ws.wait(met, n_done, 11));
            l = ctrl->top[x0][n_done & 1][0][r] + ctrl->top[x0][n_done & 1][1][r];
        }
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float lse2 = l == 0.f ? -CUDART_INF_F : (m == -CUDART_INF_F ? 0.f : m) + log2f(l);
        // every copy has landed and every product is done when all roles have come here: the tiles' room is free
        __syncthreads();
        uint8_t *const stage = smem + x0 * 3 * TILE;               // rows in the type (and their low parts behind), or in float
        const bool whole = p.n_split == 1;
        bool odd = false;
#pragma unroll 1
        for (int c = 0; c < D / 64 && rows; c++) {
            uint32_t v[32];
            const int d0 = half * (D / 2) + c * 32;
            if (n_done) {
                tmem_ld32(lane_o + c * 32, v);
                tmem_wait_ld();
                tmem_landed<32>(v);
            }
#pragma unroll
            for (int i = 0; i < 32; i++)
                v[i] = !fine ? 0x7fc00000u : n_done ? __float_as_uint(__uint_as_float(v[i]) * inv) : 0u;
#pragma unroll
            for (int i = 0; i < 32; i++) odd |= not_finite(v[i]);
            if (whole) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint8_t *at = stage + row_piece(D * 2, r, d0 / 8 + i);
                    store8<T>(reinterpret_cast<T *>(at), a.d_o_low ? reinterpret_cast<T *>(at + TILE) : nullptr, reinterpret_cast<float *>(v) + 8 * i);
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
                    *reinterpret_cast<uint4 *>(stage + row_piece(D * 4, r, d0 / 4 + i)) = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
        }
        if (r < rows && half == 0) {
            const int64_t row = sq.row0 + my_query;
            const int head = h * G + y - my_query * G;
            if (!whole) part_lse[(row * a.heads + head) * p.n_split + split] = fine ? lse2 : CUDART_NAN_F;
            else if (a.d_lse) a.d_lse[row * a.heads + head] = fine ? lse2 * LN2 : CUDART_NAN_F;
        }
        {
            const unsigned rows_odd = __ballot_sync(~0u, odd && l == l && fine && r < rows);
            if (rows_odd && lane == 0) atomicOr(&ctrl->odd[x0][quad], rows_odd);
        }
        tile_barrier(x0);
        if (ctrl->odd[x0][0] | ctrl->odd[x0][1] | ctrl->odd[x0][2] | ctrl->odd[x0][3]) {
            uint32_t *const sure = reinterpret_cast<uint32_t *>(stage + 2 * TILE);     // behind the rows
            if ((tid & 255) < D) sure[tid & 255] = 0;
            tile_barrier(x0);
            sure_columns<T, D>(a, sq, s, h, static_cast<const T *>(a.d_v), a.v_token, a.v_head, n_entries, b0, listed ? idx : nullptr, nullptr,
                               listed ? bits : nullptr, limit_min, sure, tid & 255, 256);
            tile_barrier(x0);
#pragma unroll 1
            for (int sr = warp & 7; sr < rows; sr += 8) {
                if (!(ctrl->odd[x0][sr >> 5] >> (sr & 31) & 1)) continue;
                const int sy = mine.row0 + sr, tok = (int)p.shape.G.quotient(sy), head = h * G + sy - tok * G;
                const int64_t row = sq.row0 + tok;
                const uint32_t bit = listed ? 1u << (tok / a.query_block - mine.qb0) : 1u;
                bool open = false;
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) {
                    const int d = lane * (D / 32) + i, piece = d * (whole ? 2 : 4);
                    const uint8_t *from = stage + row_piece(whole ? D * 2 : D * 4, sr, piece >> 4) + (piece & 15);
                    open |= unsure(whole ? Pack<T>::to2(*reinterpret_cast<const uint32_t *>(from)) : *reinterpret_cast<const float2 *>(from), sure, d, bit);
                }
                if (!__any_sync(~0u, open)) continue;
                float q[D / 32], k[D / 32], v[D / 32], o[D / 32] = {}, top = -CUDART_INF_F, sum = 0.f;
                row_load<T, D>(static_cast<const T *>(a.d_q) + row * a.q_token + head * a.q_head, lane, q);
                row_keys<T>(a, sq, s, h, n_entries, attn_limit(a, sq, sq.pos0 + tok),
                            [&](int e) { return !listed || bits[e] & bit ? block_of(e) : -1; },
                            [&](const T *kr, const T *vr) {
                                row_load<T, D>(kr, lane, k);
                                row_load<T, D>(vr, lane, v);
                                online_row<D>(row_dot<D>(q, k) * scale2, v, o, &top, &sum);
                            });
                const float scale_o = sum == 0.f ? 0.f : 1.f / sum;
                const int d0 = lane * (D / 32);
#pragma unroll
                for (int i = 0; i < D / 32; i += 2) {
                    const float y0 = o[i] * scale_o, y1 = o[i + 1] * scale_o;
                    const int piece = (d0 + i) * (whole ? 2 : 4);
                    uint8_t *at = stage + row_piece(whole ? D * 2 : D * 4, sr, piece >> 4) + (piece & 15);
                    if (whole) {
                        const uint32_t x = Pack<T>::two(y0, y1);
                        *reinterpret_cast<uint32_t *>(at) = x;
                        const float2 back = Pack<T>::to2(x);
                        if (a.d_o_low) *reinterpret_cast<uint32_t *>(at + TILE) = Pack<T>::two(y0 - back.x, y1 - back.y);
                    } else {
                        *reinterpret_cast<float2 *>(at) = make_float2(y0, y1);
                    }
                }
            }
            tile_barrier(x0);
        }
        if (whole) {
            const int c = (tid & 255) % (D / 8);
            for (int sr = (tid & 255) / (D / 8); sr < rows; sr += 256 / (D / 8)) {
                const int sy = mine.row0 + sr, tok = (int)p.shape.G.quotient(sy), head = h * G + sy - tok * G;
                const int64_t row = sq.row0 + tok;
                const uint8_t *from = stage + row_piece(D * 2, sr, c);
                *reinterpret_cast<uint4 *>(static_cast<T *>(a.d_o) + row * a.o_token + head * a.o_head + c * 8) = *reinterpret_cast<const uint4 *>(from);
                if (a.d_o_low)
                    *reinterpret_cast<uint4 *>(static_cast<T *>(a.d_o_low) + (row * a.heads + head) * D + c * 8) = *reinterpret_cast<const uint4 *>(from + TILE);
            }
        } else {
            const int c = (tid & 255) % (D / 4);
            for (int sr = (tid & 255) / (D / 4); sr < rows; sr += 256 / (D / 4)) {
                const int sy = mine.row0 + sr, tok = (int)p.shape.G.quotient(sy), head = h * G + sy - tok * G;
                const int64_t at = ((int64_t)(sq.row0 + tok) * a.heads + head) * p.n_split + split;
                *reinterpret_cast<uint4 *>(part_o + at * D + c * 4) = *reinterpret_cast<const uint4 *>(stage + row_piece(D * 4, sr, c));
            }
        }
        if (!fine && a.d_status) *a.d_status = SPAMM_ERR_DEVICE_WAIT;
        tc_fence_before();
    }
    __syncthreads();
    if (warp == W_MMA) {
        if (ctrl->abort_flag) drain_products();
        __syncwarp();
        tc_fence_after();
        tmem_free<COLS>(tmem);
    }
}

// Joins the ranges of keys of every row: o = sum_i 2^(lse_i - lse) o_i.  One warp for a row and head.  Bound by the reading of
// the ranges' floats: 1774 tokens of 32 heads of 128 in 3 ranges (102 MB) 28 us, 3.7 TB/s; one token for each of 32 sequences
// 6 us, a launch's own time.  (Few ranges of short rows are joined by a cluster instead, in attn_rows_kernel.)
template <typename T, int D>
__global__ __launch_bounds__(128) void attn_join_kernel(const __grid_constant__ spamm_attn a, int n_split,
                                                        const float *part_o, const float *part_lse)
{
    const int lane = threadIdx.x & 31;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int64_t per_seq = (int64_t)a.max_q * a.heads;
    if (w >= per_seq * a.batch) return;
    const int s = (int)(w / per_seq);
    const int i = (int)(w % per_seq / a.heads), head = (int)(w % a.heads);
    const Seq sq = attn_seq(a, s);
    if (i >= sq.nq) return;
    const int64_t row = sq.row0 + i, at = (row * a.heads + head) * n_split;
    float top = -CUDART_INF_F;
    for (int j = lane; j < n_split; j += 32) top = fmaxf(top, part_lse[at + j]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
    const float t0 = top == -CUDART_INF_F ? 0.f : top;
    float y[D / 32] = {}, total = 0.f;
    for (int j = 0; j < n_split; j++) {
        const float z = part_lse[at + j];
        if (z == -CUDART_INF_F) continue;
        const float f = fast_exp2(z - t0);
        total += f;
        const float *src = part_o + (at + j) * D + lane * (D / 32);
#pragma unroll
        for (int d = 0; d < D / 32; d++) y[d] += f * src[d];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    T *dst = static_cast<T *>(a.d_o) + row * a.o_token + head * a.o_head + lane * (D / 32);
    T *low = a.d_o_low ? static_cast<T *>(a.d_o_low) + (row * a.heads + head) * D + lane * (D / 32) : nullptr;
#pragma unroll
    for (int d = 0; d < D / 32; d += 2) {
        const uint32_t x = Pack<T>::two(y[d] * inv, y[d + 1] * inv);
        *reinterpret_cast<uint32_t *>(dst + d) = x;
        if (low) {
            const float2 back = Pack<T>::to2(x);
            *reinterpret_cast<uint32_t *>(low + d) = Pack<T>::two(y[d] * inv - back.x, y[d + 1] * inv - back.y);
        }
    }
    if (a.d_lse && lane == 0) a.d_lse[row * a.heads + head] = total == 0.f ? -CUDART_INF_F : (t0 + log2f(total)) * LN2;
}

// cuTensorMapEncodeTiled of the driver, looked up once through the runtime (the library does not link the driver).
static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder()
{
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

static bool encode_map(const spamm_attn &a, const void *p, const cuuint64_t *dims, const cuuint64_t *strides, const cuuint32_t *box,
                       RowMap *out)
{
    const auto encode = tensor_map_encoder();
    if (!encode) return false;
    const cuuint32_t step[3] = {1, 1, 1};
    const CUtensorMapDataType type = a.dtype == SPAMM_ATTN_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    return encode(&out->map, type, 3, const_cast<void *>(p), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

void attn_row_map(const spamm_attn &a, const void *p, int64_t token, int64_t head, int heads, int box_heads, int box_tokens,
                  RowMap *out)
{
    memset(out, 0, sizeof(*out));
    // the larger stride last, a multiple of the smaller; a dimension of one element has any stride
    if (heads == 1) head = a.dim;
    if (a.tokens == 1) token = head * heads;
    if (token <= 0 || head <= 0 || token >= (1ll << 38) || head >= (1ll << 38)) return;
    out->swapped = head > token;
    const int t = out->swapped ? 1 : 2, h = 3 - t;
    if ((out->swapped ? head % token : token % head) != 0) return;
    cuuint64_t dims[3] = {(cuuint64_t)a.dim}, strides[2];
    cuuint32_t box[3] = {64, 1, 1};
    dims[t] = a.tokens; dims[h] = heads;
    strides[t - 1] = (cuuint64_t)token * 2; strides[h - 1] = (cuuint64_t)head * 2;
    box[t] = box_tokens; box[h] = box_heads;
    out->usable = encode_map(a, p, dims, strides, box, out);
}

void attn_row_maps(const spamm_attn &a, int box_rows, RowMap *k, RowMap *v)
{
    if (!a.n_pages) {
        attn_row_map(a, a.d_k, a.k_token, a.k_head, a.kv_heads, 1, box_rows, k);
        attn_row_map(a, a.d_v, a.v_token, a.v_head, a.kv_heads, 1, box_rows, v);
        return;
    }
    memset(k, 0, sizeof(*k));
    memset(v, 0, sizeof(*v));
    if ((int64_t)a.n_pages * a.kv_heads > INT32_MAX) return;
    const cuuint64_t dims[3] = {(cuuint64_t)a.dim, (cuuint64_t)a.block, (cuuint64_t)a.n_pages * a.kv_heads};
    const cuuint64_t strides[2] = {(cuuint64_t)a.dim * 2, (cuuint64_t)a.block * a.dim * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    k->usable = encode_map(a, a.d_k, dims, strides, box, k);
    v->usable = encode_map(a, a.d_v, dims, strides, box, v);
}

static int64_t longest_list(const spamm_attn &a)
{
    return a.n_select ? min(a.n_select, attn_max_blocks(a)) : attn_max_blocks(a);
}

static bool use_tc(const spamm_attn &a) { return attn_big_tiles(a, longest_list(a) * a.block); }

static RowsPlan rows_plan(const spamm_attn &a)
{
    RowsPlan p{};
    const int G = a.heads / a.kv_heads;
    const bool tc = use_tc(a);
    if (tc) {
        p.bq = 0;
        p.nqb = 1;
        // Pairs of tiles where they fill the GPU without cutting the keys and the keys are not listed: two chunks of 1024 tokens
        // over 32768 keys take 898 us in pairs and 944 us in single tiles, but 8 chunks of 64 tokens over 8192 keys (two pairs
        // for each of 64 heads) 227 us and 186 us, and a training batch with lists of 1024 keys 497 us and 469 us: a pair is
        // alone on its SM, and nothing runs beside its beginning and its end.
        p.tiles = attn_tiles(a);
        p.pairs = !a.n_select && (int64_t)a.batch * a.kv_heads * ceil_div(p.tiles, 2) >= 148;
        if (p.pairs) p.tiles = ceil_div(p.tiles, 2);
        p.shape = attn_tile_shape(a);
    } else {
        p.bq = a.n_select ? min(a.query_block, a.max_q) : a.max_q;
        p.nqb = ceil_div(a.max_q, p.bq);
        p.tiles = (int)(((int64_t)p.bq * G + 15) / 16);
    }
    // tiles of 128 rows cut the sequence's blocks into ranges (they look through the lists for those in theirs), tiles of
    // 16 rows the list
    const int64_t blocks = max((int64_t)1, tc ? (int64_t)attn_max_blocks(a) : longest_list(a));
    const int64_t listed = (int64_t)attn_tile_lists(a) * a.n_select;       // blocks of a union
    const int64_t most = !tc ? SPAMM_ATTN_MAX_SELECT : !a.n_select ? blocks : listed <= TC_ENTRIES ? UNION_BLOCKS : TC_ENTRIES;
    const int64_t units = (int64_t)a.batch * a.kv_heads * p.nqb * p.tiles;
    // Tiles of 128 rows: enough blocks of threads to fill 148 SMs several times over (with lists the work is short as it is:
    // once), ranges of 1024 keys at the least.  Tiles of 16: two blocks per SM; lists are of one length, so one wave of equal
    // ranges does (296 blocks: 23 us against 37 us with 444 for 64 lists of 2048 keys), whole sequences are not, and two waves
    // even them out.
    int64_t want = (tc ? a.n_select ? 148 : 740 : a.n_select ? 296 : 600) / units + (tc || !a.n_select);
    want = max((int64_t)1, min(want, (blocks * a.block + (tc ? 1023 : 255)) / (tc ? 1024 : 256)));
    int64_t per = min(most, (blocks + want - 1) / want);
    p.n_split = (int)((blocks + per - 1) / per);
    // Ranges of tiles of 16 as a cluster, joined in its shared memory, where all of them run at once: 64 lists of 2048 keys 23 us
    // against 22 + 5.5 us with a kernel that joins.  In several waves the blocks of a cluster that are done hold room for which
    // others wait: 32 sequences of up to 16384 keys 265 us (more ranges 256 us and 277 us) against 243 + 6 us.
    p.cluster = !tc && p.n_split > 1 && p.n_split <= ROWS_CLUSTER && units * p.n_split <= 296;
    p.max_entries = (int)(tc && a.n_select ? min(per, listed) : per);
    p.split_keys = (int)(per * a.block);
    return p;
}

static size_t rows_smem(const spamm_attn &a, const RowsPlan &p)
{
    const int n = max(a.n_select, p.max_entries);
    return (size_t)ROWS_WARPS * ROWS_STAGES * 2 * 16 * a.dim * 2 + 16 * a.dim * 2 + 4 * (n + (n & 1)) + 8 * (size_t)p.max_entries;
}

template <typename T, int D>
static int forward_launch(const spamm_attn &a, float *scratch, cudaStream_t stream)
{
    const RowsPlan p = rows_plan(a);
    const int64_t grid = (int64_t)a.batch * a.kv_heads * p.nqb * p.tiles * p.n_split;
    const int64_t rows = (int64_t)a.batch * a.max_q * a.heads;
    if (grid > INT32_MAX || (rows + 3) / 4 > INT32_MAX || (use_tc(a) && !attn_tile_fits(a))) return attn_too_large();
    float *part_o = scratch;
    float *part_lse = scratch + (size_t)a.tokens * a.heads * p.n_split * D;
    if (use_tc(a)) {
        const int tiles = p.pairs ? 2 : 1;
        const size_t smem = tiles * 3 * TC_ROWS * D * 2 + sizeof(TcCtrl) + (a.n_select ? 6 * (size_t)p.max_entries : 0);
        const auto kernel = p.pairs ? attn_tc_kernel<T, D, 2> : attn_tc_kernel<T, D, 1>;
        int st = attn_set_smem((const void *)kernel);
        if (st) return st;
        RowMap k_map, v_map;
        attn_row_maps(a, a.block, &k_map, &v_map);
        kernel<<<(unsigned)grid, tiles * 256 + 64, smem, stream>>>(a, p, k_map, v_map, part_o, part_lse);
    } else {
        const size_t smem = rows_smem(a, p);
        int st = attn_set_smem((const void *)attn_rows_kernel<T, D>);
        if (st) return st;
        if (p.cluster) {
            cudaLaunchConfig_t how = {};
            cudaLaunchAttribute cluster = {};
            cluster.id = cudaLaunchAttributeClusterDimension;
            cluster.val.clusterDim.x = p.n_split;
            cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
            how.gridDim = dim3((unsigned)grid);
            how.blockDim = dim3(128);
            how.dynamicSmemBytes = smem;
            how.stream = stream;
            how.attrs = &cluster;
            how.numAttrs = 1;
            SPAMM_CUDA_TRY(cudaLaunchKernelEx(&how, attn_rows_kernel<T, D>, a, p, part_o, part_lse));
        } else {
            attn_rows_kernel<T, D><<<(unsigned)grid, 128, smem, stream>>>(a, p, part_o, part_lse);
        }
    }
    if (p.n_split > 1 && !p.cluster)
        attn_join_kernel<T, D><<<(unsigned)((rows + 3) / 4), 128, 0, stream>>>(a, p.n_split, part_o, part_lse);
    SPAMM_CUDA_TRY(cudaGetLastError());
    return SPAMM_OK;
}

}  // namespace spamm

using namespace spamm;

extern "C" size_t spamm_attn_forward_scratch_bytes(const spamm_attn *a)
{
    if (attn_check(a, false) || !a->batch || !a->max_q || !a->tokens) return 0;
    const RowsPlan p = rows_plan(*a);
    return p.n_split > 1 && !p.cluster ? (size_t)a->tokens * a->heads * p.n_split * (a->dim + 1) * sizeof(float) : 0;
}

extern "C" int spamm_attn_forward_dev(const spamm_attn *a, void *d_scratch, size_t scratch_bytes, void *stream)
{
    int st = attn_check(a, true);
    if (st) return st;
    if (!(a->scale > 0.f) || !(a->scale <= 3e38f)) return attn_refuse("scale is not a positive number");
    if (!a->tokens || !a->batch || !a->max_q) return SPAMM_OK;
    const bool k_ok = a->n_pages ? attn_rows_ok(a->d_k, 0, 0) && attn_rows_ok(a->d_v, 0, 0)
                                 : attn_rows_ok(a->d_k, a->k_token, a->k_head) && attn_rows_ok(a->d_v, a->v_token, a->v_head);
    if (reinterpret_cast<uintptr_t>(a->d_o_low) & 15) return attn_refuse("d_o_low is not on a 16-byte boundary");
    if (!k_ok || !attn_rows_ok(a->d_q, a->q_token, a->q_head) || !attn_rows_ok(a->d_o, a->o_token, a->o_head))
        return attn_refuse("q, k, v and o need rows on 16-byte boundaries");
    const size_t need = spamm_attn_forward_scratch_bytes(a);
    if (need && (!d_scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(d_scratch) & 15)))
        return attn_refuse("scratch too small or not on a 16-byte boundary");
    float *scratch = static_cast<float *>(d_scratch);
    if (a->dtype == SPAMM_ATTN_BF16)
        return a->dim == 64 ? forward_launch<__nv_bfloat16, 64>(*a, scratch, (cudaStream_t)stream)
                            : forward_launch<__nv_bfloat16, 128>(*a, scratch, (cudaStream_t)stream);
    return a->dim == 64 ? forward_launch<__half, 64>(*a, scratch, (cudaStream_t)stream)
                        : forward_launch<__half, 128>(*a, scratch, (cudaStream_t)stream);
}
