// New keys and values into the pages of a cache, keys and queries rotated by their positions on the way, the key sums of
// the touched pages brought up to date.
//
// A block of threads takes one page of one sequence and some of the key heads with their query heads.  The angles
// position * inv_freq are taken in double (a float angle of position 10^5 is off by 0.004), their sine and cosine are
// rounded to float and kept in shared memory for all heads.  A rotated pair is (a cos - b sin, b cos + a sin) with every
// product and sum rounded by itself, not fused: the stored keys are then the same bits wherever they are computed, and
// with them the key sums by which blocks are selected.  (But for about one cosine in 10^8, which lies so near the middle of two
// floats that the way its angle was put together decides.)
//
// Bound by reading and writing the tokens where they are many: 5 prompts of up to 4001 tokens, 32 heads and 4 key heads of 128,
// q with them (307 MB), 80 us, 3.8 TB/s: a block of threads turns, stores and sums one after the other.  One token for each of 64 sequences: 11 us,
// the chain of table, page, token and the sum over the page.
#include "attn.cuh"

namespace spamm {

constexpr int APPEND_THREADS = 256;

// Turns the pair of 8-value pieces (x, y) in place: element i by (cs[i].x, cs[i].y) = (cos, sin).
template <typename T> static __device__ __forceinline__ void turn_halves(uint4 &x, uint4 &y, const float2 *cs)
{
    uint32_t *xs = reinterpret_cast<uint32_t *>(&x), *ys = reinterpret_cast<uint32_t *>(&y);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 a = Pack<T>::to2(xs[i]), b = Pack<T>::to2(ys[i]);
        const float2 c0 = cs[2 * i], c1 = cs[2 * i + 1];
        xs[i] = Pack<T>::two(__fsub_rn(__fmul_rn(a.x, c0.x), __fmul_rn(b.x, c0.y)),
                             __fsub_rn(__fmul_rn(a.y, c1.x), __fmul_rn(b.y, c1.y)));
        ys[i] = Pack<T>::two(__fadd_rn(__fmul_rn(b.x, c0.x), __fmul_rn(a.x, c0.y)),
                             __fadd_rn(__fmul_rn(b.y, c1.x), __fmul_rn(a.y, c1.y)));
    }
}
// The same for four neighbouring pairs in one piece.
template <typename T> static __device__ __forceinline__ void turn_neighbours(uint4 &x, const float2 *cs)
{
    uint32_t *xs = reinterpret_cast<uint32_t *>(&x);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float2 a = Pack<T>::to2(xs[i]), c = cs[i];
        xs[i] = Pack<T>::two(__fsub_rn(__fmul_rn(a.x, c.x), __fmul_rn(a.y, c.y)),
                             __fadd_rn(__fmul_rn(a.y, c.x), __fmul_rn(a.x, c.y)));
    }
}

template <typename T, int D>
__global__ __launch_bounds__(APPEND_THREADS) void attn_append_kernel(const __grid_constant__ spamm_attn a, int pages_per_seq,
                                                                     int heads_per_cta, FastDiv div_k, FastDiv div_q, T *k_pages, T *v_pages,
                                                                     float *key_sums, const float *inv_freq, int n_freq,
                                                                     bool interleaved)
{
    extern __shared__ __align__(16) uint8_t smem[];
    float2 *turn = reinterpret_cast<float2 *>(smem);                  // [tokens of the page][n_freq]
    double *sums = reinterpret_cast<double *>(smem);                  // later: [threads][8]
    constexpr int V = D / 8;
    const int tid = threadIdx.x;
    const int s = blockIdx.x / pages_per_seq, j = blockIdx.x % pages_per_seq;
    const int h0 = blockIdx.y * heads_per_cta, hn = min(heads_per_cta, a.kv_heads - h0);
    const int G = a.heads / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    const int skip = max(0, -sq.pos0);                                // tokens that the cache's length leaves no place for
    if (skip && a.d_status) *a.d_status = SPAMM_ERR_INVALID;
    if (a.d_o && a.zero_tail) {
        // rows of q that belong to no sequence, or to no position
        const int end = s == a.batch - 1 ? a.tokens : min(max(a.d_cu[s + 1], sq.row0), a.tokens);
        const int lead = s == 0 ? sq.row0 : 0, head_rows = min(skip, sq.nq);
        const int begin = sq.row0 + min(sq.nq, max(sq.nk - sq.pos0, 0));
        const int rows = lead + head_rows + (end - begin), vecs = hn * G * V;
        for (int i = j; i < rows; i += pages_per_seq) {
            const int64_t row = i < lead ? i : i < lead + head_rows ? sq.row0 + i - lead : begin + (i - lead - head_rows);
            for (int x = tid; x < vecs; x += APPEND_THREADS)
                *reinterpret_cast<uint4 *>(static_cast<T *>(a.d_o) + row * a.o_token + (h0 * G + x / V) * a.o_head + x % V * 8) =
                    make_uint4(0, 0, 0, 0);
        }
    }
    const int first = max(sq.pos0, 0), end = min(sq.pos0 + sq.nq, sq.nk);    // positions that are written
    if (first >= end) return;
    const int b = first / a.block + j;
    const int lo = max(first, b * a.block), hi = min(end, (b + 1) * a.block);
    if (lo >= hi) return;
    const int n = hi - lo;
    int page = a.d_table[(int64_t)s * a.table_stride + b];
    if (page < 0 || page >= a.n_pages) {
        if (tid == 0) *a.d_status = SPAMM_ERR_INVALID;
        page = -1;
    }
    // Sines and cosines in double are the dearest part of a prompt's append, so that of position lo + 8 x + y is put together
    // from those of (lo + 8 x) and y by the sums' formula, in double (11 pairs instead of 32 for a page of 32; every angle is
    // exact, 24 bits of frequency times the position, and the formula's rounding is 2^-29 of the float's that follows).
    double2 *far = reinterpret_cast<double2 *>(smem + ((size_t)min(a.max_q, a.block) * n_freq * sizeof(float2) + 15) / 16 * 16);
    const int n_far = (n + 7) / 8, n_near = min(n, 8);
    for (int i = tid; i < (n_far + n_near - 1) * n_freq; i += APPEND_THREADS) {
        const int x = i / n_freq, f = i - x * n_freq;
        double sn, cs;
        sincos((double)(x < n_far ? lo + 8 * x : x - n_far + 1) * (double)inv_freq[f], &sn, &cs);
        far[i] = make_double2(cs, sn);
    }
    __syncthreads();
    for (int i = tid; i < n * n_freq; i += APPEND_THREADS) {
        const int t = i / n_freq, f = i - t * n_freq;
        double2 z = far[(t >> 3) * n_freq + f];
        if (t & 7) {
            const double2 w = far[(n_far + (t & 7) - 1) * n_freq + f];
            z = make_double2(z.x * w.x - z.y * w.y, z.y * w.x + z.x * w.y);
        }
        turn[i] = make_float2((float)z.x, (float)z.y);
    }
    __syncthreads();

    const int64_t row0 = sq.row0 + (lo - sq.pos0);                    // row of the page's first new token
    const int rv = n_freq / 8;                                        // 8-value pieces of half the turned part
    // Rows are (token, head), V neighbouring threads to a row; of keys and queries that are turned by halves a thread takes a
    // pair of pieces, and when that leaves no more than V / 2 of them, V / 2 threads a row.  (The last block of heads may hold
    // fewer than div_k.d: its rows beyond are skipped.)
    const int col = tid % V;
    const int64_t at0 = ((int64_t)page * a.kv_heads + h0) * a.block * D;
    if (page >= 0) {
        const T *src = static_cast<const T *>(a.d_v) + row0 * a.v_token + h0 * a.v_head + col * 8;
#pragma unroll 4
        for (int i = tid / V; i < n * (int)div_k.d; i += APPEND_THREADS / V) {
            const int t = (int)div_k.quotient(i), h = i - t * (int)div_k.d;
            if (h >= hn) continue;
            const uint4 x = *reinterpret_cast<const uint4 *>(src + t * a.v_token + h * a.v_head);
            *reinterpret_cast<uint4 *>(v_pages + at0 + (h * a.block + (lo + t) % a.block) * D + col * 8) = x;
        }
    }
    auto turn_rows = [&](const T *src, int64_t token, int64_t head, int rows, const FastDiv &div, int heads, auto to) {
        const int units = interleaved ? V : V - rv, lanes = units <= V / 2 ? V / 2 : V;
        const int u = tid % lanes, step = APPEND_THREADS / lanes;
        if (u >= units) return;
        const bool pair = !interleaved && u < rv, turned = interleaved ? u < 2 * rv : pair;
        const int p0 = (interleaved || pair ? u : u + rv) * 8;
#pragma unroll 4
        for (int i = tid / lanes; i < rows; i += step) {
            const int t = (int)div.quotient(i), h = i - t * (int)div.d;
            if (h >= heads) continue;
            const T *from = src + t * token + h * head;
            T *dst = to(t, h);
            const float2 *cs = turn + t * n_freq;
            uint4 x = *reinterpret_cast<const uint4 *>(from + p0);
            if (pair) {
                uint4 y = *reinterpret_cast<const uint4 *>(from + n_freq + p0);
                turn_halves<T>(x, y, cs + u * 8);
                *reinterpret_cast<uint4 *>(dst + n_freq + p0) = y;
            } else if (turned) {
                turn_neighbours<T>(x, cs + u * 4);
            }
            *reinterpret_cast<uint4 *>(dst + p0) = x;
        }
    };
    if (page >= 0)
        turn_rows(static_cast<const T *>(a.d_k) + row0 * a.k_token + h0 * a.k_head, a.k_token, a.k_head, n * (int)div_k.d, div_k, hn,
                  [&](int t, int h) { return k_pages + at0 + (h * a.block + (lo + t) % a.block) * D; });
    if (a.d_o) {
        T *out = static_cast<T *>(a.d_o) + row0 * a.o_token + (int64_t)h0 * G * a.o_head;
        turn_rows(static_cast<const T *>(a.d_q) + row0 * a.q_token + (int64_t)h0 * G * a.q_head, a.q_token, a.q_head, n * (int)div_q.d, div_q,
                  hn * G, [&](int t, int h) { return out + t * a.o_token + h * a.o_head; });
    }
    if (page < 0 || !key_sums) return;
    // the sum of all keys that the page holds: columns of 8 values, the rows dealt out to groups of threads
    const int held = hi - b * a.block;
    for (int c0 = 0; c0 < hn * V; c0 += APPEND_THREADS) {
        const int cols = min(APPEND_THREADS, hn * V - c0), groups = APPEND_THREADS / cols;
        const int col = tid % cols, g = tid / cols;
        const int h = h0 + (c0 + col) / V, c = (c0 + col) % V;
        const T *src = k_pages + ((int64_t)page * a.kv_heads + h) * a.block * D + c * 8;
        double y[8] = {};
        __syncthreads();                                              // keys are stored; `turn` and `sums` are free
        if (g < groups)
#pragma unroll 4
            for (int r = g; r < held; r += groups) {
                const uint4 x = __ldcg(reinterpret_cast<const uint4 *>(src + r * D));
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = Pack<T>::to2(xs[i]);
                    y[2 * i] += (double)f.x;
                    y[2 * i + 1] += (double)f.y;
                }
            }
#pragma unroll
        for (int i = 0; i < 8; i++) sums[tid * 8 + i] = y[i];
        __syncthreads();
        for (int i = tid; i < cols * 8; i += APPEND_THREADS) {
            double z = 0.0;
            for (int k = 0; k < groups; k++) z += sums[(k * cols + i / 8) * 8 + i % 8];
            const int hh = h0 + (c0 + i / 8) / V, d = (c0 + i / 8) % V * 8 + i % 8;
            key_sums[((int64_t)page * a.kv_heads + hh) * D + d] = (float)z;
        }
    }
}

template <typename T, int D>
static int append_launch(const spamm_attn &a, void *k_pages, void *v_pages, float *key_sums, const float *inv_freq, int n_freq,
                         int interleaved, cudaStream_t stream)
{
    const int64_t per = ((int64_t)a.max_q + 2 * a.block - 2) / a.block;   // pages that max_q tokens may touch
    const int64_t grid = per * a.batch;
    if (grid > INT32_MAX) return attn_too_large();
    // a block of threads for each page and key head where pages are few, several heads where they fill the GPU (the sines of a
    // page are then taken once for them); 600 blocks are one wave of four to an SM
    int split = (int)max((int64_t)1, min((int64_t)a.kv_heads, (600 + grid - 1) / grid));
    const int heads_per_cta = ceil_div(a.kv_heads, split);
    split = ceil_div(a.kv_heads, heads_per_cta);
    const int tokens = min(a.max_q, a.block);
    const size_t turns = ((size_t)tokens * n_freq * sizeof(float2) + 15) / 16 * 16 + (size_t)(ceil_div(tokens, 8) + 7) * n_freq * sizeof(double2);
    const size_t smem = max(turns, (size_t)APPEND_THREADS * 8 * sizeof(double));
    int st = attn_set_smem((const void *)attn_append_kernel<T, D>);
    if (st) return st;
    attn_append_kernel<T, D><<<dim3((unsigned)grid, split), APPEND_THREADS, smem, stream>>>(
        a, (int)per, heads_per_cta, fast_div(heads_per_cta), fast_div(heads_per_cta * (a.heads / a.kv_heads)), static_cast<T *>(k_pages), static_cast<T *>(v_pages), key_sums, inv_freq, n_freq, interleaved != 0);
    SPAMM_CUDA_TRY(cudaGetLastError());
    return SPAMM_OK;
}

}  // namespace spamm

using namespace spamm;

extern "C" int spamm_attn_append_dev(const spamm_attn *a, void *d_k_pages, void *d_v_pages, float *d_key_sums,
                                     const float *d_inv_freq, int n_freq, int interleaved, void *stream)
{
    int st = attn_check(a, false);
    if (st) return st;
    if (!a->n_pages)
        return attn_refuse("append needs pages");
    if (!d_inv_freq) n_freq = 0;
    if (n_freq < 0 || 2 * (int64_t)n_freq > a->dim || n_freq % 8)
        return attn_refuse("n_freq is no multiple of 8 up to dim / 2");
    if (a->kv_heads > 65535) return attn_too_large();
    if (!a->batch || !a->max_q || !a->tokens) return SPAMM_OK;
    if (!attn_rows_ok(a->d_k, a->k_token, a->k_head) || !attn_rows_ok(a->d_v, a->v_token, a->v_head) ||
        !attn_rows_ok(d_k_pages, 0, 0) || !attn_rows_ok(d_v_pages, 0, 0) ||
        (a->d_o && (!attn_rows_ok(a->d_q, a->q_token, a->q_head) || !attn_rows_ok(a->d_o, a->o_token, a->o_head))))
        return attn_refuse("q, k, v, o and the pages need rows on 16-byte boundaries");
    cudaStream_t str = (cudaStream_t)stream;
    if (a->dtype == SPAMM_ATTN_BF16)
        return a->dim == 64 ? append_launch<__nv_bfloat16, 64>(*a, d_k_pages, d_v_pages, d_key_sums, d_inv_freq, n_freq, interleaved, str)
                            : append_launch<__nv_bfloat16, 128>(*a, d_k_pages, d_v_pages, d_key_sums, d_inv_freq, n_freq, interleaved, str);
    return a->dim == 64 ? append_launch<__half, 64>(*a, d_k_pages, d_v_pages, d_key_sums, d_inv_freq, n_freq, interleaved, str)
                        : append_launch<__half, 128>(*a, d_k_pages, d_v_pages, d_key_sums, d_inv_freq, n_freq, interleaved, str);
}
