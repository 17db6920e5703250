// The blocks of keys that every query block reads: the n_select largest of
//
//   score(b) = (sum of the query block's queries over the G heads) . (sum of the keys of b) / (keys held by b)
//
// The choice is discrete, so a rounding that depends on an order of summation would change whole blocks of the result
// now and then.  Sums and products are therefore taken in double: bf16 and half values add up without any rounding
// there (short of wildly different magnitudes), and the double rate of this GPU is half its float rate.  Only the key
// sums, which a cache keeps, are rounded to float.
#include <type_traits>
#include "attn.cuh"

namespace spamm {

// Key sums of packed keys: block b of sequence s at row cu[s] / block + s + b (no two sequences share a row).
__device__ __forceinline__ int64_t sums_row(const spamm_attn &a, const Seq &sq, int s, int b)
{
    return (int64_t)sq.row0 / a.block + s + b;
}

// Eight double sums of values that come 16 bytes at a time.  The conversion to double is slow (8 values a clock and SM), so
// the bits of the float are put where the double has them instead: read as a double they stand for the value times 2^-896,
// zeros and subnormals included, and sums of them are scaled back once at the end.  Infinities and NaN alone would be read as
// finite; `odd` notices them and the sums are then taken again with conversions.
template <typename T> struct Sum8 {
    double y[8];
    uint32_t odd;
    __device__ __forceinline__ Sum8() : odd(0)
    {
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = 0.0;
    }
    static __device__ __forceinline__ double moved(float f)
    {
        const uint32_t x = __float_as_uint(f);
        return __hiloint2double((int)((x & 0x80000000u) | ((x & 0x7fffffffu) >> 3)), 0);   // the low 13 bits are zero
    }
    __device__ __forceinline__ void add(uint4 x)
    {
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            // an exponent of all ones carries into the sign's place
            odd |= (xs[i] & 0x7fff7fffu) + (std::is_same<T, __nv_bfloat16>::value ? 0x00800080u : 0x04000400u);
            const float2 f = Pack<T>::to2(xs[i]);
            y[2 * i] += moved(f.x);
            y[2 * i + 1] += moved(f.y);
        }
    }
    __device__ __forceinline__ void add_slowly(uint4 x)
    {
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = Pack<T>::to2(xs[i]);
            y[2 * i] += (double)f.x;
            y[2 * i + 1] += (double)f.y;
        }
    }
    // Sums what `at(r)` points to for r = first, first + step, ... below n.
    template <typename At> __device__ __forceinline__ void all(int first, int step, int n, At at)
    {
#pragma unroll 8
        for (int r = first; r < n; r += step) add(*reinterpret_cast<const uint4 *>(at(r)));
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] *= 0x1p896;
        if (odd & 0x80008000u) {
#pragma unroll
            for (int i = 0; i < 8; i++) y[i] = 0.0;
            for (int r = first; r < n; r += step) add_slowly(*reinterpret_cast<const uint4 *>(at(r)));
        }
    }
};

template <typename T, int D>
static __device__ void key_sums_of(const spamm_attn &a, int block, int nkb, double *sums, float *key_sums)
{
    constexpr int V = D / 8;
    const int tid = threadIdx.x, s = block / nkb, b = block % nkb;
    const Seq sq = attn_seq(a, s);
    const int held = min(a.block, sq.nk - b * a.block);
    if (held <= 0) return;
    float *out = key_sums + sums_row(a, sq, s, b) * a.kv_heads * D;
    for (int c0 = 0; c0 < a.kv_heads * V; c0 += 256) {
        const int cols = min(256, a.kv_heads * V - c0), groups = 256 / cols;
        const int col = tid % cols, g = tid / cols, h = (c0 + col) / V, c = (c0 + col) % V;
        const T *src = static_cast<const T *>(a.d_k) + (int64_t)(sq.row0 + b * a.block) * a.k_token + h * a.k_head + c * 8;
        Sum8<T> sum;
        if (g < groups) sum.all(g, groups, held, [&](int r) { return src + r * a.k_token; });
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; i++) sums[tid * 8 + i] = sum.y[i];
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

// What a query block may and must read: blocks [0, n) are candidates, those below n_first and in (lo, hi] are taken.
struct Reach { int n, lo, hi; };
__device__ __forceinline__ Reach reach_of(const spamm_attn &a, const Seq &sq, int64_t q0, int n_tok, int n_local)
{
    Reach r{0, 0, -1};
    if (n_tok <= 0) return r;
    const int first = sq.pos0 + (int)q0, last = first + n_tok - 1;
    r.n = ceil_div(attn_limit(a, sq, last), a.block);
    if (n_local > 0) {
        r.lo = (first >= 0 ? first / a.block : -1) - n_local;
        r.hi = last >= 0 ? last / a.block : -1;
    }
    return r;
}
__device__ __forceinline__ bool taken(const Reach &r, int b, int n_first) { return b < n_first || (b > r.lo && b <= r.hi); }

// The ordered key of the score z of candidate b.  Every block but the last is full, and 1 / block a power of two.
__device__ __forceinline__ unsigned long long score_key(const spamm_attn &a, const Seq &sq, const Reach &r, int b, int n_first, double z,
                                                        double per_key)
{
    if (taken(r, b, n_first)) return ~0ull;
    const int held = sq.nk - b * a.block;
    return order_key(held < a.block ? z / (double)held : z * per_key);
}

// Row of the key sums of block b; -1 for a page that does not exist.
__device__ __forceinline__ int64_t key_sum_row(const spamm_attn &a, const Seq &sq, int s, int b)
{
    if (!a.n_pages) return sums_row(a, sq, s, b);
    const int page = a.d_table[(int64_t)s * a.table_stride + b];
    if (page < 0 || page >= a.n_pages) {
        *a.d_status = SPAMM_ERR_INVALID;
        return -1;
    }
    return page;
}

// The sums of every query block's queries over the heads of a key head, double [lists][D].  WIDE: a block of threads for a
// list (from 64 rows on: four loads for each thread), else a group of D / 8 threads, whose sums need no joining.
template <typename T, int D, bool WIDE>
static __device__ void query_sums_of(const spamm_attn &a, int block, int nqb, const FastDiv &div_g, double *part, double *query_sums)
{
    constexpr int V = D / 8, GROUPS = 256 / V;
    const int tid = threadIdx.x, c = tid % V, g = tid / V, G = a.heads / a.kv_heads;
    const int64_t list = WIDE ? block : (int64_t)block * GROUPS + g;
    const int64_t lists = (int64_t)a.batch * nqb * a.kv_heads;
    if (list >= lists) return;
    const int h = (int)(list % a.kv_heads), qb = (int)(list / a.kv_heads % nqb), s = (int)(list / a.kv_heads / nqb);
    const Seq sq = attn_seq(a, s);
    const int64_t q0 = (int64_t)qb * a.query_block;
    const int n_tok = (int)min((int64_t)a.query_block, sq.nq - q0);
    if (n_tok <= 0) return;
    const T *src = static_cast<const T *>(a.d_q) + (sq.row0 + q0) * a.q_token + (int64_t)h * G * a.q_head + c * 8;
    Sum8<T> sum;
    sum.all(WIDE ? g : 0, WIDE ? GROUPS : 1, n_tok * G, [&](int r) {
        const int tok = (int)div_g.quotient(r);
        return src + tok * a.q_token + (r - tok * G) * a.q_head;
    });
    double *out = query_sums + list * D;
    if constexpr (!WIDE) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            reinterpret_cast<double2 *>(out + c * 8)[i] = make_double2(sum.y[2 * i], sum.y[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) part[(g * V + c) * 8 + i] = sum.y[i];
        __syncthreads();
        for (int d = tid; d < D; d += 256) {
            double z = 0.0;
            for (int k = 0; k < GROUPS; k++) z += part[k * D + d];
            out[d] = z;
        }
    }
}

// Both kinds of sums in one launch: the first key_blocks blocks of threads take those of the keys.  Bound by the reading of q
// and k: 3 sequences of up to 16384, 32 heads of 128 and 8 key heads (369 MB), 79 us, 4.7 TB/s; 32768 lists
// of 16 rows (143 MB) 36 us, 4.0 TB/s.
template <typename T, int D, bool WIDE>
__global__ __launch_bounds__(256, 4) void attn_sums_kernel(const __grid_constant__ spamm_attn a, int key_blocks, int nkb, int nqb,
                                                           FastDiv div_g, float *key_sums, double *query_sums)
{
    __shared__ double part[256 * 8];
    if ((int)blockIdx.x < key_blocks) key_sums_of<T, D>(a, blockIdx.x, nkb, part, key_sums);
    else query_sums_of<T, D, WIDE>(a, blockIdx.x - key_blocks, nqb, div_g, part, query_sums);
}

// The number that an ordered key stands for.
__device__ __forceinline__ double key_value(unsigned long long key)
{
    return __longlong_as_double((long long)(key >> 63 ? key & 0x7fffffffffffffffull : ~key));
}
// The next key to try between low and high (low < result < high; high - low > 1): halfway between the values for the first
// rounds, which comes near a rank in few of them, halfway between the keys from then on, which always ends.
__device__ __forceinline__ unsigned long long key_between(unsigned long long low, unsigned long long high, int round)
{
    if (round < 16) {
        const double x = 0.5 * key_value(low) + 0.5 * key_value(high);
        const unsigned long long key = order_key(x);
        if (key > low && key < high) return key;
    }
    return low + ((high - low) >> 1);
}

// One warp writes the keys above the threshold, and of its equals the first `left`, as an ascending list.
static __device__ __forceinline__ void write_list(const unsigned long long *keys, int n, unsigned long long threshold, int left, int n_select,
                                  int32_t *out, int lane)
{
    int count = 0;
    for (int b0 = 0; b0 < n; b0 += 32) {
        const int b = b0 + lane;
        const unsigned long long key = b < n ? keys[b] : 0;
        const unsigned eq = __ballot_sync(~0u, key == threshold && key != 0);
        const bool tie = key == threshold && key != 0 && __popc(eq & ((1u << lane) - 1)) < left;
        const unsigned m = __ballot_sync(~0u, key > threshold || tie);
        const int at = count + __popc(m & ((1u << lane) - 1));
        if ((m >> lane & 1) && at < n_select) out[at] = b;
        count += __popc(m);
        left -= min(left, __popc(eq));
    }
    for (int i = min(count, n_select) + lane; i < n_select; i += 32) out[i] = -1;
}

// Writes the n_select largest of keys[0, n) in shared memory (0: no candidate) as an ascending list, by all threads.  The
// threshold is searched between the smallest and the largest key, until exactly n_select keys are at or above it or it is
// the n_select-th largest key itself.
template <int THREADS>
static __device__ void write_largest(const unsigned long long *keys, int n, int n_select, int32_t *out)
{
    __shared__ int counts[3];                    // taken in turn, each cleared two rounds ahead
    __shared__ unsigned long long ends[2];
    const int tid = threadIdx.x, lane = tid & 31;
    if (tid < 3) counts[tid] = 0;
    if (tid == 0) { ends[0] = ~0ull; ends[1] = 0; }
    __syncthreads();
    int round = 0;
    auto count = [&](auto pred) {
        int c = 0;
        for (int b = tid; b < n; b += THREADS) c += pred(keys[b]);
        c = __reduce_add_sync(~0u, c);
        if (lane == 0 && c) atomicAdd(&counts[round % 3], c);
        __syncthreads();
        c = counts[round % 3];
        if (tid == 0) counts[(round + 2) % 3] = 0;
        round++;
        return c;
    };
    unsigned long long threshold = 1;
    int left = INT32_MAX;
    if (n > n_select) {
        // blocks that are taken in any case have the key ~0 and are left out of the range of the search
        unsigned long long low = ~0ull, high = 0;
        for (int b = tid; b < n; b += THREADS) {
            low = min(low, keys[b]);
            if (keys[b] != ~0ull) high = max(high, keys[b]);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            low = min(low, __shfl_xor_sync(~0u, low, d));
            high = max(high, __shfl_xor_sync(~0u, high, d));
        }
        if (lane == 0) {
            atomicMin(&ends[0], low);
            atomicMax(&ends[1], high);
        }
        __syncthreads();
        low = ends[0];
        high = ends[1] + 1;                      // all keys are at or above low, fewer than n_select at or above high
        bool exact = false;
        while (low < high && high - low > 1 && !exact) {
            const unsigned long long want = key_between(low, high, round);
            const int c = count([&](unsigned long long k) { return k >= want; });
            exact = c == n_select;
            if (c >= n_select) low = want;
            else high = want;
        }
        threshold = low;
        if (!exact) left = n_select - count([&](unsigned long long k) { return k > threshold; });
    }
    // every warp writes the part of the list that lies in its share of the blocks
    __shared__ int2 shares[THREADS / 32];
    const int warp = tid >> 5, share = (n + THREADS - 1) / THREADS * 32;
    const int from = min(warp * share, n), to = min(from + share, n);
    int above = 0, equal = 0;
    for (int b = from + lane; b < to; b += 32) {
        above += keys[b] > threshold;
        equal += keys[b] == threshold && threshold != 0;
    }
    above = __reduce_add_sync(~0u, above);
    equal = __reduce_add_sync(~0u, equal);
    if (lane == 0) shares[warp] = make_int2(above, equal);
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < THREADS / 32; w++) {
        const int2 x = shares[w];
        const int ties = min(x.y, left);
        if (w < warp) at += x.x + ties;
        else if (w == warp) equal = ties;                    // of this share's equals, the first so many
        left -= ties;
        all += x.x + ties;
    }
    for (int b0 = from; b0 < to; b0 += 32) {
        const int b = b0 + lane;
        const unsigned long long key = b < to ? keys[b] : 0;
        const unsigned eq = __ballot_sync(~0u, key == threshold && key != 0);
        const bool tie = key == threshold && key != 0 && __popc(eq & ((1u << lane) - 1)) < equal;
        const unsigned m = __ballot_sync(~0u, key > threshold || tie);
        const int to_at = at + __popc(m & ((1u << lane) - 1));
        if ((m >> lane & 1) && to_at < n_select) out[to_at] = b;
        at += __popc(m);
        equal -= min(equal, __popc(eq));
    }
    for (int i = min(all, n_select) + tid; i < n_select; i += THREADS) out[i] = -1;
}

// write_largest by one warp.
static __device__ __noinline__ void pick_by_whole_keys(const unsigned long long *mine, int n, int n_select, int32_t *out, int lane)
{
    unsigned long long threshold = 1;
    int left = INT32_MAX;
    if (n > n_select) {
        unsigned long long low = ~0ull, high = 0;
        for (int b = lane; b < n; b += 32) {
            low = min(low, mine[b]);
            if (mine[b] != ~0ull) high = max(high, mine[b]);
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) {
            low = min(low, __shfl_xor_sync(~0u, low, d));
            high = max(high, __shfl_xor_sync(~0u, high, d));
        }
        high++;
        bool exact = false;
        for (int round = 0; low < high && high - low > 1 && !exact; round++) {
            const unsigned long long want = key_between(low, high, round);
            int c = 0;
            for (int b = lane; b < n; b += 32) c += mine[b] >= want;
            c = __reduce_add_sync(~0u, c);
            exact = c == n_select;
            if (c >= n_select) low = want;
            else high = want;
        }
        threshold = low;
        if (!exact) {
            int above = 0;
            for (int b = lane; b < n; b += 32) above += mine[b] > threshold;
            left = n_select - __reduce_add_sync(~0u, above);
        }
    }
    write_list(mine, n, threshold, left, n_select, out, lane);
}

// The same by the upper halves of the keys alone, which nearly always suffice: held in registers, R for each of the LANES lanes
// of a list, 32 / LANES lists to a warp, whose searches are then under way together.  n_most: the warp's largest n, at most
// LANES * R.  False, and nothing written, where upper halves are alike at the border.
template <int LANES, int R>
static __device__ __forceinline__ bool pick_by_upper_halves(const unsigned long long *mine, int n, int n_most, int n_select, bool wanted,
                                                            int32_t *out, int lane)
{
    const int l = lane % LANES, group = lane - l;
    constexpr unsigned MASK = LANES == 32 ? ~0u : (1u << (LANES % 32)) - 1;
    uint32_t k[R], low = ~0u, high = 0;
#pragma unroll
    for (int x = 0; x < R; x++) {
        const int b = x * LANES + l;
        k[x] = b < n ? reinterpret_cast<const uint32_t *>(mine)[2 * b + 1] : 0;      // no branch: all are requested at once
    }
    // (groups of eight: a branch for each would cost more than what it skips)
#pragma unroll
    for (int x0 = 0; x0 < R; x0 += 8) {
        if (x0 * LANES >= n_most) break;
#pragma unroll
        for (int x = x0; x < x0 + 8; x++) {
            low = min(low, x * LANES + l < n ? k[x] : ~0u);
            high = max(high, k[x] != ~0u ? k[x] : 0);
        }
    }
#pragma unroll
    for (int d = 1; d < LANES; d <<= 1) {
        low = min(low, __shfl_xor_sync(~0u, low, d));
        high = max(high, __shfl_xor_sync(~0u, high, d));
    }
    high++;
    const bool all = n <= n_select;                          // every candidate is taken
    bool exact = all;
    for (int round = 0; __any_sync(~0u, !exact && low < high && high - low > 1); round++) {
        uint32_t want = (uint32_t)(key_between((unsigned long long)low << 32, (unsigned long long)high << 32, round) >> 32);
        if (want == low) want++;
        int c = 0, c1 = 0;
#pragma unroll
        for (int x0 = 0; x0 < R; x0 += 8) {
            if (x0 * LANES >= n_most) break;
#pragma unroll
            for (int x = x0; x < x0 + 8; x += 2) {
                c += k[x] >= want;
                c1 += k[x + 1] >= want;
            }
        }
        c += c1;
        if (LANES == 32) {
            c = __reduce_add_sync(~0u, c);
        } else {
#pragma unroll
            for (int d = 1; d < LANES; d <<= 1) c += __shfl_xor_sync(~0u, c, d);
        }
        if (!exact && low < high && high - low > 1) {
            exact = c == n_select;
            if (c >= n_select) low = want;
            else high = want;
        }
    }
    int count = 0;
#pragma unroll
    for (int x = 0; x < R; x++) {
        if (x * LANES >= n_most) break;
        const int b = x * LANES + l;
        const bool keep = exact && b < n && (all ? mine[b] != 0 : k[x] >= low);
        const unsigned m = __ballot_sync(~0u, keep) >> group & MASK;
        if (keep && wanted) out[count + __popc(m & ((1u << l) - 1))] = b;
        count += __popc(m);
    }
    if (exact && wanted)
        for (int x = count + l; x < n_select; x += LANES) out[x] = -1;
    return exact;
}

constexpr int SELECT_TILE32_BLOCKS = 256;      // blocks of a sequence up to which tiles of 32 query blocks are used

// ---- many query blocks: QT of them and one key head per block of threads, scores as double products on the tensor cores
// (m8n8k4), the lists picked from shared memory
__device__ __forceinline__ void mma_double(double *c, double a, double b)
{
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                 : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

// Bound by the double products for long sequences and by the searches for the lists: 32768 lists over up to 128 blocks 66 us, of
// which the products (1.1 GFLOP in double, half of them masked) are less than half; 4512 lists over up to 256 blocks 33 us.
template <int D, int QT>
__global__ __launch_bounds__(256) void attn_select_tile_kernel(const __grid_constant__ spamm_attn a, int nqb, int nkb, int n_first,
                                                               int n_local, const float *key_sums, const double *query_sums,
                                                               int32_t *lists)
{
    constexpr int LD = D + 4;                               // rows 4 doubles apart from a multiple of the banks
    constexpr int MG = QT / 8, NG = 8 / MG, KT = QT == 8 ? 64 : 32, NT = KT / NG / 8;
    extern __shared__ __align__(16) uint8_t smem[];
    double *qs = reinterpret_cast<double *>(smem);          // [QT][LD]
    double *ks = qs + QT * LD;                              // [KT][LD]
    unsigned long long *keys = reinterpret_cast<unsigned long long *>(ks + KT * LD);    // [QT][nkb]
    __shared__ Reach reach[QT];
    __shared__ bool there[KT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int q_tiles = ceil_div(nqb, QT);
    unsigned idx = blockIdx.x;
    const int qt = q_tiles - 1 - idx % q_tiles; idx /= q_tiles;
    const int h = idx % a.kv_heads, s = idx / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    if (tid < QT) {
        const int64_t q0 = (int64_t)(qt * QT + tid) * a.query_block;
        reach[tid] = reach_of(a, sq, q0, qt * QT + tid < nqb ? (int)min((int64_t)a.query_block, sq.nq - q0) : 0, n_local);
    }
    // (loads in batches: the compiler may not move one above a store to shared memory)
    {
        constexpr int N = QT * (D / 2) / 256;
        double2 x[N];
        const int c = tid % (D / 2) * 2, r0 = tid / (D / 2);
        const double *src = query_sums + (((int64_t)s * nqb + qt * QT) * a.kv_heads + h) * D + c;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = r0 + i * (512 / D);
            x[i] = make_double2(0.0, 0.0);
            if ((int64_t)(qt * QT + r) * a.query_block < sq.nq) x[i] = *reinterpret_cast<const double2 *>(src + (int64_t)r * a.kv_heads * D);
        }
#pragma unroll
        for (int i = 0; i < N; i++) *reinterpret_cast<double2 *>(qs + (r0 + i * (512 / D)) * LD + c) = x[i];
    }
    __syncthreads();
    int n_most = 0;
#pragma unroll 1
    for (int i = 0; i < QT; i++) n_most = max(n_most, reach[i].n);
    const int mg = warp % MG, ng = warp / MG;
    const double per_key = 1.0 / (double)a.block;
    constexpr int PER_ROW = 256 / KT;                       // threads of a row of key sums
    const int my_row = tid / PER_ROW, my_col = tid % PER_ROW;
    constexpr int KN = D / 4 / PER_ROW;
    float4 k[KN];
    int64_t row = -1;
    auto fetch = [&](int b0) {
        row = b0 + my_row < n_most ? key_sum_row(a, sq, s, b0 + my_row) : -1;
        const float4 *src = reinterpret_cast<const float4 *>(key_sums + (max(row, (int64_t)0) * a.kv_heads + h) * D);
#pragma unroll
        for (int i = 0; i < KN; i++) k[i] = row >= 0 ? src[i * PER_ROW + my_col] : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    fetch(0);
    for (int b0 = 0; b0 < n_most; b0 += KT) {
        // this step's key sums are in registers already; the next step's are requested before the products
        if (my_col == 0) there[my_row] = row >= 0;
#pragma unroll
        for (int i = 0; i < KN; i++) {
            double *dst = ks + my_row * LD + (i * PER_ROW + my_col) * 4;
            *reinterpret_cast<double2 *>(dst) = make_double2((double)k[i].x, (double)k[i].y);
            *reinterpret_cast<double2 *>(dst + 2) = make_double2((double)k[i].z, (double)k[i].w);
        }
        fetch(b0 + KT);
        __syncthreads();
        double acc[NT][2] = {};
        const double *qa = qs + (mg * 8 + (lane >> 2)) * LD + (lane & 3);
        const double *kb = ks + (ng * NT * 8 + (lane >> 2)) * LD + (lane & 3);
#pragma unroll 16
        for (int k = 0; k < D; k += 4) {
            const double x = qa[k];
#pragma unroll
            for (int n = 0; n < NT; n++) mma_double(acc[n], x, kb[n * 8 * LD + k]);
        }
        const int i = mg * 8 + (lane >> 2);
        const Reach rr = reach[i];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int at = (ng * NT + n) * 8 + (lane & 3) * 2 + e, b = b0 + at;
                if (b < nkb) keys[i * nkb + b] = b < rr.n && there[at] ? score_key(a, sq, rr, b, n_first, acc[n][e], per_key) : 0;
            }
        __syncthreads();
    }
    if constexpr (QT == 32) {
        // four lists to a warp
        const int i = warp * 4 + lane / 8, qb = qt * QT + i;
        const bool exact = pick_by_upper_halves<8, SELECT_TILE32_BLOCKS / 8>(keys + i * nkb, reach[i].n, n_most, a.n_select, qb < nqb,
                                                                             lists + (((int64_t)s * nqb + qb) * a.kv_heads + h) * a.n_select, lane);
        // the rest, where upper halves are alike at the border
        unsigned rest = __ballot_sync(~0u, !exact && lane % 8 == 0 && qb < nqb);
        while (rest) {
            const int slow = warp * 4 + (__ffs(rest) - 1) / 8;
            rest &= rest - 1;
            pick_by_whole_keys(keys + slow * nkb, reach[slow].n, a.n_select,
                               lists + (((int64_t)s * nqb + qt * QT + slow) * a.kv_heads + h) * a.n_select, lane);
        }
    } else {
        for (int i = warp; i < QT; i += 8) {
            const int qb = qt * QT + i;
            if (qb >= nqb) break;
            pick_by_whole_keys(keys + i * nkb, reach[i].n, a.n_select, lists + (((int64_t)s * nqb + qb) * a.kv_heads + h) * a.n_select, lane);
        }
    }
}

// ---- few query blocks (decoding): SPREAD_BLOCKS blocks of keys to a warp, so that the reading of the key sums, which bounds
// it, spreads over the GPU; up to eight query blocks of a sequence at once.  The key sums go from global memory straight into
// registers, eight blocks at a time and the next eight under way: a lane has every fourth group of four values of one block.
// One query block (the newest token): plain products, joined by two shuffles.  Several: m8n8k4, where a lane's four values
// enter four products in turn (the sum then takes the values in another order, for both operands alike).  Sums of up to 16 rows
// are taken here, by every block of threads for itself: one launch less, for a few kilobytes of q.  16 sequences of up to 65537
// keys in pages of 64, 8 key heads of 128 (44 MB of key sums): 16 us, 2.8 TB/s.
constexpr int SPREAD_ROWS = 16;          // rows of a query block up to which their sums are taken here
constexpr int SPREAD_BLOCKS = 32, SPREAD_WARPS = 4;

template <typename T, int D>
__global__ __launch_bounds__(SPREAD_WARPS * 32, 6) void attn_spread_scores_kernel(const __grid_constant__ spamm_attn a, int nqb, int spans,
                                                                                 int nkb, int n_first, int n_local,
                                                                                 const float *key_sums, const double *query_sums,
                                                                                 unsigned long long *keys)
{
    constexpr int N = D / 16;            // groups of four values of a lane
    __shared__ __align__(16) double qs[8][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = lane >> 2, kk = lane & 3;
    const int groups = ceil_div(nqb, 8);
    unsigned idx = blockIdx.x;
    const int span = idx % spans; idx /= spans;
    const int qg = idx % groups; idx /= groups;
    const int h = idx % a.kv_heads, s = idx / a.kv_heads;
    const Seq sq = attn_seq(a, s);
    const int G = a.heads / a.kv_heads;
    const int n_lists = min(8, ceil_div(sq.nq, a.query_block) - qg * 8);      // of this group
    if (n_lists <= 0) return;
    {
        // the last query block reaches furthest
        const int64_t q0 = (int64_t)(qg * 8 + n_lists - 1) * a.query_block;
        const Reach last = reach_of(a, sq, q0, (int)min((int64_t)a.query_block, sq.nq - q0), 0);
        if (span * SPREAD_WARPS * SPREAD_BLOCKS >= last.n) return;
    }
    const int first_b = (span * SPREAD_WARPS + warp) * SPREAD_BLOCKS;
    // this lane's block of the warp's 32: the row of its key sums
    int64_t my_row = -1;
    if (first_b + lane < ceil_div(sq.nk, a.block)) my_row = key_sum_row(a, sq, s, first_b + lane);
    const unsigned ok = __ballot_sync(~0u, my_row >= 0);
    auto fetch = [&](int x, float4 *k) {
        const int64_t at = __shfl_sync(~0u, my_row, 8 * x + row);
        const float4 *ks = reinterpret_cast<const float4 *>(key_sums + (max(at, (int64_t)0) * a.kv_heads + h) * D) + kk;
#pragma unroll
        for (int i = 0; i < N; i++) k[i] = at >= 0 ? ks[4 * i] : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    float4 k[N], next[N];
    fetch(0, k);
    for (int i = tid; i < n_lists * D; i += SPREAD_WARPS * 32) {
        const int l = i / D, d = i % D;
        const int64_t q0 = (int64_t)(qg * 8 + l) * a.query_block;
        double z = 0.0;
        if (query_sums) {
            z = query_sums[(((int64_t)s * nqb + qg * 8 + l) * a.kv_heads + h) * D + d];
        } else {
            const int rows = (int)min((int64_t)a.query_block, sq.nq - q0) * G;
            const T *src = static_cast<const T *>(a.d_q) + (sq.row0 + q0) * a.q_token + (int64_t)h * G * a.q_head + d;
#pragma unroll 4
            for (int r = 0; r < rows; r++) z += (double)(float)src[r / G * a.q_token + r % G * a.q_head];
        }
        qs[l][d] = z;
    }
    __syncthreads();
    const double per_key = 1.0 / (double)a.block;
    auto store = [&](int l, int b, bool there, double z) {
        const int64_t q0 = (int64_t)(qg * 8 + l) * a.query_block;
        const Reach reach = reach_of(a, sq, q0, (int)min((int64_t)a.query_block, sq.nq - q0), n_local);
        if (b < reach.n)
            keys[(((int64_t)s * nqb + qg * 8 + l) * a.kv_heads + h) * nkb + b] = there ? score_key(a, sq, reach, b, n_first, z, per_key) : 0;
    };
    // the list whose sums this lane reads (lanes of rows without one: any, their results are not used)
    const double *q = qs[n_lists == 1 ? 0 : min(row, n_lists - 1)] + 4 * kk;
#pragma unroll 1
    for (int x = 0; x < SPREAD_BLOCKS / 8; x++) {
        if (!(ok >> (8 * x))) {
            // nothing but blocks that are not there: their keys are written all the same
            if (first_b + 8 * x >= ceil_div(sq.nk, a.block)) break;
        }
        if (x + 1 < SPREAD_BLOCKS / 8) fetch(x + 1, next);
        if (n_lists == 1) {
            double z0 = 0.0, z1 = 0.0;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const double2 u = *reinterpret_cast<const double2 *>(q + 16 * i), v = *reinterpret_cast<const double2 *>(q + 16 * i + 2);
                z0 = fma(u.x, (double)k[i].x, z0);
                z1 = fma(u.y, (double)k[i].y, z1);
                z0 = fma(v.x, (double)k[i].z, z0);
                z1 = fma(v.y, (double)k[i].w, z1);
            }
            z0 += z1;
            z0 += __shfl_xor_sync(~0u, z0, 1);
            z0 += __shfl_xor_sync(~0u, z0, 2);
            if (kk == 0) store(0, first_b + 8 * x + row, ok >> (8 * x + row) & 1, z0);
        } else {
            double acc[2][2] = {};
#pragma unroll
            for (int i = 0; i < N; i++) {
                const double2 u = *reinterpret_cast<const double2 *>(q + 16 * i), v = *reinterpret_cast<const double2 *>(q + 16 * i + 2);
                mma_double(acc[0], u.x, (double)k[i].x);
                mma_double(acc[1], u.y, (double)k[i].y);
                mma_double(acc[0], v.x, (double)k[i].z);
                mma_double(acc[1], v.y, (double)k[i].w);
            }
            if (row < n_lists)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    store(row, first_b + 8 * x + 2 * kk + e, ok >> (8 * x + 2 * kk + e) & 1, acc[0][e] + acc[1][e]);
        }
#pragma unroll
        for (int i = 0; i < N; i++) k[i] = next[i];
    }
}

// The lists of spread scores: by one warp each up to LARGEST_WARP blocks (128 lists over up to 1025: 10 us, the
// latency of its rounds), by a block of threads beyond (14 us).
constexpr int LARGEST_WARP = 2048;

static __device__ __forceinline__ int candidates(const spamm_attn &a, int nqb, int list)
{
    const int s = list / a.kv_heads / nqb, qb = list / a.kv_heads % nqb;
    const Seq sq = attn_seq(a, s);
    const int64_t q0 = (int64_t)qb * a.query_block;
    return reach_of(a, sq, q0, (int)min((int64_t)a.query_block, sq.nq - q0), 0).n;
}
template <int R>
__global__ __launch_bounds__(32) void attn_largest_warp_kernel(const __grid_constant__ spamm_attn a, int nqb, int nkb,
                                                               const unsigned long long *keys, int32_t *lists)
{
    const int n = candidates(a, nqb, blockIdx.x);
    const unsigned long long *mine = keys + (int64_t)blockIdx.x * nkb;
    int32_t *out = lists + (int64_t)blockIdx.x * a.n_select;
    if (!pick_by_upper_halves<32, R>(mine, n, n, a.n_select, true, out, threadIdx.x)) pick_by_whole_keys(mine, n, a.n_select, out, threadIdx.x);
}
template <int THREADS>
__global__ __launch_bounds__(THREADS) void attn_largest_kernel(const __grid_constant__ spamm_attn a, int nqb, int nkb,
                                                               const unsigned long long *keys, int32_t *lists)
{
    extern __shared__ __align__(16) unsigned long long copy[];
    const int n = candidates(a, nqb, blockIdx.x);
    for (int i = threadIdx.x; i < n; i += THREADS) copy[i] = keys[(int64_t)blockIdx.x * nkb + i];
    write_largest<THREADS>(copy, n, a.n_select, lists + (int64_t)blockIdx.x * a.n_select);
}

// ---- many query blocks of sequences too long for that: one list per block of threads
template <typename T, int D>
__global__ __launch_bounds__(128) void attn_select_kernel(const __grid_constant__ spamm_attn a, int nqb, int n_first, int n_local,
                                                          const float *key_sums, const double *query_sums, int32_t *lists)
{
    extern __shared__ __align__(16) uint8_t smem[];
    unsigned long long *keys = reinterpret_cast<unsigned long long *>(smem);
    __shared__ double qsum[D];
    const int tid = threadIdx.x;
    unsigned idx = blockIdx.x;
    const int h = idx % a.kv_heads; idx /= a.kv_heads;
    const int qb = idx % nqb, s = idx / nqb;
    const Seq sq = attn_seq(a, s);
    const int64_t q0 = (int64_t)qb * a.query_block;
    const int n_tok = (int)min((int64_t)a.query_block, sq.nq - q0);
    const Reach reach = reach_of(a, sq, q0, n_tok, n_local);
    if (n_tok > 0)
        for (int d = tid; d < D; d += 128) qsum[d] = query_sums[(int64_t)blockIdx.x * D + d];
    __syncthreads();
    for (int b = tid; b < reach.n; b += 128) {
        unsigned long long key = ~0ull;
        const int64_t row = key_sum_row(a, sq, s, b);
        if (row < 0) {
            key = 0;
        } else if (!taken(reach, b, n_first)) {
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
    write_largest<128>(keys, reach.n, a.n_select, lists + (((int64_t)s * nqb + qb) * a.kv_heads + h) * a.n_select);
}

// Which of the four (times with the sums, 8 key heads of 128 unless noted).  A tile of eight query blocks wants eight in a
// sequence, and tiles enough to fill the GPU when the blocks of keys are many: else the scores are spread (16 sequences of one
// token over up to 1025 blocks: 16 us and 10 us for the lists; as tiles of one list each seven eighths of the products would be
// empty).  1024 lists over 32 blocks: tiles of 8 15 us, spread 24 us, one by one 19 us.  Tiles of 32 need 4096 lists: 2048
// lists over 64 blocks 19 us against 17 us in tiles of 8, 8192 lists 30 us against 42 us (one by one 79 us, spread 103 us).
// Beyond 1024 blocks the scores of eight query blocks do not fit shared memory.
enum SelectWay { SELECT_SPREAD, SELECT_TILE32, SELECT_TILE8, SELECT_ONE };
static SelectWay select_way(const spamm_attn &a)
{
    const int64_t groups = (int64_t)a.batch * a.kv_heads, nqb = attn_query_blocks(a), blocks = attn_max_blocks(a);
    if (nqb < 8 || (blocks > 128 && groups * ((nqb + 7) / 8) < 148) || (blocks > 1024 && groups * nqb < 1184)) return SELECT_SPREAD;
    if (blocks <= SELECT_TILE32_BLOCKS && groups * nqb >= 4096) return SELECT_TILE32;
    return blocks <= 1024 ? SELECT_TILE8 : SELECT_ONE;
}

template <int D, int QT>
static int select_tile_launch(const spamm_attn &a, int nqb, int nkb, int n_first, int n_local, const float *key_sums,
                              const double *query_sums, int32_t *lists, cudaStream_t stream)
{
    const size_t smem = (size_t)(QT + (QT == 8 ? 64 : 32)) * (D + 4) * 8 + (size_t)QT * nkb * 8;
    const int64_t grid = (int64_t)a.batch * a.kv_heads * ceil_div(nqb, QT);
    int st = attn_set_smem((const void *)attn_select_tile_kernel<D, QT>);
    if (st) return st;
    attn_select_tile_kernel<D, QT><<<(unsigned)grid, 256, smem, stream>>>(a, nqb, nkb, n_first, n_local, key_sums, query_sums, lists);
    return SPAMM_OK;
}

// No page table: nothing to list.
static int clear_lists(const spamm_attn &a, int32_t *lists, cudaStream_t stream)
{
    SPAMM_CUDA_TRY(cudaMemsetAsync(lists, 0xff, (size_t)a.batch * attn_query_blocks(a) * a.kv_heads * a.n_select * 4, stream));
    return SPAMM_OK;
}

static size_t key_sums_bytes(const spamm_attn &a)
{
    if (a.n_pages) return 0;
    return (((size_t)a.tokens / a.block + a.batch + 1) * a.kv_heads * a.dim * sizeof(float) + 15) / 16 * 16;
}

template <typename T, int D>
static int select_launch(const spamm_attn &a, const float *key_sums, int n_first, int n_local, int32_t *lists, float *scratch,
                         cudaStream_t stream)
{
    const int nkb = attn_max_blocks(a), nqb = attn_query_blocks(a);
    const int64_t grid = (int64_t)a.batch * nqb * a.kv_heads, sums_grid = (int64_t)a.batch * nkb;
    if (grid > INT32_MAX || sums_grid > INT32_MAX) return attn_too_large();
    const int key_blocks = !a.n_pages && a.tokens ? (int)sums_grid : 0;
    if (!a.n_pages) key_sums = scratch;
    const int G = a.heads / a.kv_heads;
    double *query_sums = reinterpret_cast<double *>(reinterpret_cast<uint8_t *>(scratch) + key_sums_bytes(a));
    if ((int64_t)min(a.query_block, a.max_q) * G > INT32_MAX / 2) return attn_too_large();
    const SelectWay way = select_way(a);
    const int rows = min(a.query_block, a.max_q) * G;
    // the queries' sums: a block of threads for a list of many rows, 2048 / D lists to a block of few, none where the scores'
    // kernel takes them itself
    const bool wide = rows >= 64;
    const int64_t query_blocks = wide ? grid : way != SELECT_SPREAD || rows > SPREAD_ROWS ? (grid + 2048 / D - 1) / (2048 / D) : 0;
    if (key_blocks + query_blocks > INT32_MAX) return attn_too_large();
    if (key_blocks + query_blocks) {
        const auto sums = wide ? attn_sums_kernel<T, D, true> : attn_sums_kernel<T, D, false>;
        sums<<<(unsigned)(key_blocks + query_blocks), 256, 0, stream>>>(a, key_blocks, nkb, nqb, fast_div(G), scratch, query_sums);
    }
    int st = SPAMM_OK;
    switch (way) {
    case SELECT_SPREAD: {
        if (!nkb) return clear_lists(a, lists, stream);
        unsigned long long *keys = reinterpret_cast<unsigned long long *>(query_sums + grid * D);
        const int spans = ceil_div(nkb, SPREAD_BLOCKS * SPREAD_WARPS);
        const int64_t blocks = (int64_t)a.batch * a.kv_heads * ceil_div(nqb, 8) * spans;
        if (blocks > INT32_MAX) return attn_too_large();
        attn_spread_scores_kernel<T, D><<<(unsigned)blocks, SPREAD_WARPS * 32, 0, stream>>>(a, nqb, spans, nkb, n_first, n_local, key_sums,
                                                                              rows > SPREAD_ROWS ? query_sums : nullptr, keys);
        if (nkb <= LARGEST_WARP / 4) {
            attn_largest_warp_kernel<LARGEST_WARP / 128><<<(unsigned)grid, 32, 0, stream>>>(a, nqb, nkb, keys, lists);
        } else if (nkb <= LARGEST_WARP) {
            attn_largest_warp_kernel<LARGEST_WARP / 32><<<(unsigned)grid, 32, 0, stream>>>(a, nqb, nkb, keys, lists);
        } else {
            st = attn_set_smem((const void *)attn_largest_kernel<256>);
            if (st) return st;
            attn_largest_kernel<256><<<(unsigned)grid, 256, (size_t)nkb * 8, stream>>>(a, nqb, nkb, keys, lists);
        }
        break;
    }
    case SELECT_TILE32: st = select_tile_launch<D, 32>(a, nqb, nkb, n_first, n_local, key_sums, query_sums, lists, stream); break;
    case SELECT_TILE8: st = select_tile_launch<D, 8>(a, nqb, nkb, n_first, n_local, key_sums, query_sums, lists, stream); break;
    case SELECT_ONE:
        st = attn_set_smem((const void *)attn_select_kernel<T, D>);
        if (st) return st;
        attn_select_kernel<T, D><<<(unsigned)grid, 128, (size_t)nkb * 8, stream>>>(a, nqb, n_first, n_local, key_sums, query_sums, lists);
        break;
    }
    if (st) return st;
    SPAMM_CUDA_TRY(cudaGetLastError());
    return SPAMM_OK;
}

}  // namespace spamm

using namespace spamm;

extern "C" size_t spamm_attn_select_scratch_bytes(const spamm_attn *a)
{
    if (attn_check(a, false) || !a->batch || !a->max_q) return 0;
    const size_t lists = (size_t)a->batch * attn_query_blocks(*a) * a->kv_heads;
    size_t n = key_sums_bytes(*a) + lists * a->dim * sizeof(double);
    if (select_way(*a) == SELECT_SPREAD) n += lists * attn_max_blocks(*a) * sizeof(unsigned long long);
    return n;
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
