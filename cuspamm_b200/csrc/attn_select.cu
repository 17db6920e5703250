// The blocks of keys that every query block reads: the n_select largest of
//
//   score(b) = (sum of the query block's queries over the G heads) . (sum of the keys of b) / (keys held by b)
//
// The choice is discrete, so a rounding that depends on an order of summation would change whole blocks of the result
// now and then.  Sums and products are therefore taken in double: bf16 and half values add up without any rounding
// there (short of wildly different magnitudes), and the double rate of this GPU is half its float rate.  Only the key
// sums, which a cache keeps, are rounded to float.
#include "attn.cuh"

namespace spamm {

// Key sums of packed keys: block b of sequence s at row cu[s] / block + s + b (no two sequences share a row).
__device__ __forceinline__ int64_t sums_row(const spamm_attn &a, const Seq &sq, int s, int b)
{
    return (int64_t)sq.row0 / a.block + s + b;
}

template <typename T, int D>
__global__ __launch_bounds__(256) void attn_key_sums_kernel(const __grid_constant__ spamm_attn a, int nkb, float *key_sums)
{
    constexpr int V = D / 8;
    __shared__ double sums[256 * 8];
    const int tid = threadIdx.x, s = blockIdx.x / nkb, b = blockIdx.x % nkb;
    const Seq sq = attn_seq(a, s);
    const int held = min(a.block, sq.nk - b * a.block);
    if (held <= 0) return;
    float *out = key_sums + sums_row(a, sq, s, b) * a.kv_heads * D;
    for (int c0 = 0; c0 < a.kv_heads * V; c0 += 256) {
        const int cols = min(256, a.kv_heads * V - c0), groups = 256 / cols;
        const int col = tid % cols, g = tid / cols, h = (c0 + col) / V, c = (c0 + col) % V;
        const T *src = static_cast<const T *>(a.d_k) + (int64_t)(sq.row0 + b * a.block) * a.k_token + h * a.k_head + c * 8;
        double y[8] = {};
        if (g < groups)
#pragma unroll 4
            for (int r = g; r < held; r += groups) {
                const uint4 x = *reinterpret_cast<const uint4 *>(src + r * a.k_token);
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float2 f = Pack<T>::to2(xs[i]);
                    y[2 * i] += (double)f.x;
                    y[2 * i + 1] += (double)f.y;
                }
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) sums[tid * 8 + i] = y[i];
        __syncthreads();
        for (int i = tid; i < cols * 8; i += 256) {
            double z = 0.0;
            for (int k = 0; k < groups; k++) z += sums[(k * cols + i / 8) * 8 + i % 8];
            out[(int64_t)c0 * 8 + i] = (float)z;
        }
    }
}

// Doubles as unsigned integers in the same order; NaN lowest, both zeros alike, 0 kept for "no candidate".
__device__ __forceinline__ unsigned long long order_key(double x)
{
    if (x != x) return 1ull;
    const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | (1ull << 63);
}

// One query block and key head per block of threads.
template <typename T, int D>
__global__ __launch_bounds__(128) void attn_select_kernel(const __grid_constant__ spamm_attn a, int nqb, int n_first, int n_local,
                                                          const float *key_sums, int32_t *lists)
{
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int V = D / 8;
    unsigned long long *keys = reinterpret_cast<unsigned long long *>(smem);
    __shared__ double part[128 * 8];
    __shared__ double qsum[D];
    __shared__ int hist[256];
    __shared__ unsigned long long s_prefix;
    __shared__ int s_left;
    const int tid = threadIdx.x, lane = tid & 31;
    unsigned idx = blockIdx.x;
    const int h = idx % a.kv_heads; idx /= a.kv_heads;
    const int qb = idx % nqb;
    const int s = idx / nqb;
    const int G = a.heads / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    int32_t *out = lists + (((int64_t)s * nqb + qb) * a.kv_heads + h) * a.n_select;
    const int64_t q0 = (int64_t)qb * a.query_block;
    const int n_tok = (int)min((int64_t)a.query_block, sq.nq - q0);
    const int first = sq.pos0 + (int)min(q0, (int64_t)sq.nq), last = first + max(n_tok, 0) - 1;
    const int n_blocks = n_tok > 0 ? ceil_div(attn_limit(a, sq, last), a.block) : 0;
    if (n_blocks <= 0) {
        for (int i = tid; i < a.n_select; i += 128) out[i] = -1;
        return;
    }
    // sum of the queries
    {
        const int c = tid % V, g = tid / V;
        double y[8] = {};
        const T *src = static_cast<const T *>(a.d_q) + (sq.row0 + q0) * a.q_token + (int64_t)h * G * a.q_head + c * 8;
        for (int r = g; r < n_tok * G; r += 128 / V) {
            const uint4 x = *reinterpret_cast<const uint4 *>(src + r / G * a.q_token + r % G * a.q_head);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = Pack<T>::to2(xs[i]);
                y[2 * i] += (double)f.x;
                y[2 * i + 1] += (double)f.y;
            }
        }
#pragma unroll
        for (int i = 0; i < 8; i++) part[(g * V + c) * 8 + i] = y[i];
    }
    __syncthreads();
    for (int d = tid; d < D; d += 128) {
        double z = 0.0;
        for (int g = 0; g < 128 / V; g++) z += part[g * D + d];
        qsum[d] = z;
    }
    __syncthreads();
    // scores as ordered integers
    const int first_block = first >= 0 ? first / a.block : -1, last_block = last >= 0 ? last / a.block : -1;
    for (int b = tid; b < n_blocks; b += 128) {
        const bool forced = b < n_first || (b > first_block - n_local && b <= last_block && n_local > 0);
        unsigned long long key = ~0ull;
        const int64_t row = a.n_pages ? (int64_t)a.d_table[(int64_t)s * a.table_stride + b] : sums_row(a, sq, s, b);
        if (a.n_pages && (row < 0 || row >= a.n_pages)) {
            *a.d_status = SPAMM_ERR_INVALID;
            key = 0;
        } else if (!forced) {
            const float4 *ks = reinterpret_cast<const float4 *>(key_sums + (row * a.kv_heads + h) * D);
            double z = 0.0;
#pragma unroll 8
            for (int d = 0; d < D / 4; d++) {
                const float4 k = ks[d];
                z = fma(qsum[4 * d], (double)k.x, z);
                z = fma(qsum[4 * d + 1], (double)k.y, z);
                z = fma(qsum[4 * d + 2], (double)k.z, z);
                z = fma(qsum[4 * d + 3], (double)k.w, z);
            }
            key = order_key(z / (double)min(a.block, sq.nk - b * a.block));
        }
        keys[b] = key;
    }
    if (tid == 0) { s_prefix = 0; s_left = a.n_select; }
    __syncthreads();
    // the n_select-th largest key, eight bits at a time; all candidates when there are no more than n_select blocks
    unsigned long long mask = 0;
    if (n_blocks > a.n_select) {
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += 128) hist[i] = 0;
            __syncthreads();
            const unsigned long long prefix = s_prefix;
            for (int b = tid; b < n_blocks; b += 128)
                if ((keys[b] & mask) == prefix) atomicAdd(&hist[(int)(keys[b] >> shift) & 255], 1);
            __syncthreads();
            if (tid < 32) {
                // lane's eight bins from the top: where the running count reaches s_left
                const int left = s_left;
                int mine = 0;
                for (int i = 0; i < 8; i++) mine += hist[255 - lane * 8 - i];
                int run = mine;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const int u = __shfl_up_sync(~0u, run, d);
                    if (lane >= d) run += u;
                }
                const int before = run - mine;
                if (before < left && run >= left) {
                    int rest = left - before, bin = 255 - lane * 8;
                    while (hist[bin] < rest) rest -= hist[bin--];
                    s_prefix = prefix | ((unsigned long long)bin << shift);
                    s_left = rest;
                }
            }
            mask |= 255ull << shift;
            __syncthreads();
        }
    }
    // keep what is above the threshold, and of its equals the first s_left
    if (tid < 32) {
        const unsigned long long threshold = s_prefix;
        int left = n_blocks > a.n_select ? s_left : INT32_MAX, count = 0;
        for (int b0 = 0; b0 < n_blocks; b0 += 32) {
            const int b = b0 + lane;
            const unsigned long long key = b < n_blocks ? keys[b] : 0;
            const unsigned eq = __ballot_sync(~0u, key == threshold && key != 0);
            const bool tie = key == threshold && key != 0 && __popc(eq & ((1u << lane) - 1)) < left;
            const bool keep = key > threshold || tie;
            const unsigned m = __ballot_sync(~0u, keep);
            const int at = count + __popc(m & ((1u << lane) - 1));
            if (keep && at < a.n_select) out[at] = b;
            count += __popc(m);
            left -= min(left, __popc(eq));
        }
        for (int i = min(count, a.n_select) + lane; i < a.n_select; i += 32) out[i] = -1;
    }
}

template <typename T, int D>
static int select_launch(const spamm_attn &a, const float *key_sums, int n_first, int n_local, int32_t *lists, float *scratch,
                         cudaStream_t stream)
{
    const int nkb = attn_max_blocks(a), nqb = attn_query_blocks(a);
    const int64_t grid = (int64_t)a.batch * nqb * a.kv_heads, sums_grid = (int64_t)a.batch * nkb;
    if (grid > INT32_MAX || sums_grid > INT32_MAX) return attn_too_large();
    if (!a.n_pages) {
        attn_key_sums_kernel<T, D><<<(unsigned)sums_grid, 256, 0, stream>>>(a, nkb, scratch);
        key_sums = scratch;
    }
    const size_t smem = (size_t)nkb * 8;
    int st = attn_set_smem((const void *)attn_select_kernel<T, D>, smem);
    if (st) return st;
    attn_select_kernel<T, D><<<(unsigned)grid, 128, smem, stream>>>(a, nqb, n_first, n_local, key_sums, lists);
    SPAMM_CUDA_TRY(cudaGetLastError());
    return SPAMM_OK;
}

}  // namespace spamm

using namespace spamm;

extern "C" size_t spamm_attn_select_scratch_bytes(const spamm_attn *a)
{
    if (attn_check(a, false) || a->n_pages || !a->batch || !a->max_q || !a->tokens) return 0;
    return ((size_t)a->tokens / a->block + a->batch + 1) * a->kv_heads * a->dim * sizeof(float);
}

extern "C" int spamm_attn_select_dev(const spamm_attn *a, const float *d_key_sums, int n_first, int n_local,
                                     int32_t *d_lists_out, void *d_scratch, size_t scratch_bytes, void *stream)
{
    int st = attn_check(a, false);
    if (st) return st;
    const int64_t forced = (int64_t)n_first + (n_local > 0 ? n_local + ((int64_t)a->query_block + a->block - 2) / a->block : 0);
    if (n_first < 0 || n_local < 0 || a->n_select < 1 || (int64_t)a->n_select < forced)
        return attn_refuse("n_select is below 1 or leaves no room for the first and the local blocks");
    if (!a->batch || !a->max_q) return SPAMM_OK;
    if (attn_max_blocks(*a) > SPAMM_ATTN_MAX_BLOCKS) {
        record_error_text("spamm_attn: more than 16384 blocks to rank");
        return SPAMM_ERR_UNSUPPORTED;
    }
    if (!d_lists_out || (a->tokens && (!attn_rows_ok(a->d_q, a->q_token, a->q_head) ||
        (a->n_pages ? !attn_rows_ok(d_key_sums, 0, 0) : !attn_rows_ok(a->d_k, a->k_token, a->k_head)))))
        return attn_refuse("q, k and the key sums need rows on 16-byte boundaries");
    const size_t need = spamm_attn_select_scratch_bytes(a);
    if (need && (!d_scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(d_scratch) & 15)))
        return attn_refuse("scratch too small or not on a 16-byte boundary");
    cudaStream_t str = (cudaStream_t)stream;
    float *scratch = static_cast<float *>(d_scratch);
    if (a->dtype == SPAMM_ATTN_BF16)
        return a->dim == 64 ? select_launch<__nv_bfloat16, 64>(*a, d_key_sums, n_first, n_local, d_lists_out, scratch, str)
                            : select_launch<__nv_bfloat16, 128>(*a, d_key_sums, n_first, n_local, d_lists_out, scratch, str);
    return a->dim == 64 ? select_launch<__half, 64>(*a, d_key_sums, n_first, n_local, d_lists_out, scratch, str)
                        : select_launch<__half, 128>(*a, d_key_sums, n_first, n_local, d_lists_out, scratch, str);
}
