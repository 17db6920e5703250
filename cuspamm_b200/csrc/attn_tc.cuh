// What the tcgen05 attention kernels share.  Operand tiles lie in shared memory as panels of 64 values: rows of 128 bytes
// whose 16-byte pieces are XORed with the row number (the 128-byte swizzle), groups of 8 rows 1024 bytes apart.  The same
// tile serves as an operand whose rows are M or N (K-major: values along K) and as one whose rows are K (MN-major).
#pragma once
#include <cuda.h>
#include "attn.cuh"
#include "tc_utils.cuh"

namespace spamm {

// Byte offset of 16-byte piece c (0 .. D/8-1) of row r in a tile of `rows` rows.
__device__ __forceinline__ uint32_t panel_off(int rows, int r, int c)
{
    return (c >> 3) * (rows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);     // 8-row groups 1024 bytes apart, 128-byte swizzle
// Descriptor of a tile whose rows are M or N, and what K step ks of 16 values adds to it.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t tile)
{
    return ((uint64_t)DESC_HI << 32) | ((tile & 0x3ffffu) >> 4) | (1u << 16);
}
__host__ __device__ constexpr uint32_t step_k_major(int rows, int ks) { return ((ks >> 2) * (rows * 128) + (ks & 3) * 32) >> 4; }
// The same for a tile whose rows are K (steps of 16 rows); panels of 64 values of M or N lie rows * 128 bytes apart.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t tile, int rows)
{
    return ((uint64_t)DESC_HI << 32) | ((tile & 0x3ffffu) >> 4) | ((uint32_t)(rows * 128) >> 4 << 16);
}
__host__ __device__ constexpr uint32_t step_mn_major(int ks) { return ks * 2048 >> 4; }

// One lane of a converged warp.  The loops that issue products are walked by the whole warp, so that addresses and
// descriptors stay in uniform registers, and this lane issues: the issuing warp shares its scheduler with the busy ones, and
// every instruction that it needs for a product delays the next.
__device__ __forceinline__ bool elect_one()
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
    return ok != 0;
}

template <typename T> struct IsBf { static constexpr uint32_t value = 0; };
template <> struct IsBf<__nv_bfloat16> { static constexpr uint32_t value = 1; };
// Instruction descriptor: float accumulator, A and B of type T, M x N; a_mn / b_mn: the operand's rows are K.
template <typename T> __host__ __device__ constexpr uint32_t mma_desc(uint32_t m, uint32_t n, bool a_mn, bool b_mn)
{
    return (1u << 4) | (IsBf<T>::value << 7) | (IsBf<T>::value << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
           ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a_tmem), "l"(b), "r"(idesc),
                 "r"((uint32_t)add)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
                   "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t *v)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}
template <int N> __device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t *v)
{
    static_assert(N == 8 || N == 16 || N == 32, "columns of one load");
    if constexpr (N == 8) tmem_ld8(taddr, v);
    else if constexpr (N == 16) tmem_ld16(taddr, v);
    else tmem_ld32(taddr, v);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, "
                 "%24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
                 "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                 "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
                 "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
                 "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
                 : "memory");
}
// After tmem_wait_ld: keeps the compiler from using loaded values before the wait.
template <int N> __device__ __forceinline__ void tmem_landed(uint32_t *v)
{
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));
}
template <int COLS> __device__ __forceinline__ void tmem_alloc(uint32_t smem_slot)
{
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_slot), "r"(COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS> __device__ __forceinline__ void tmem_free(uint32_t base)
{
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(COLS) : "memory");
}
// Whether the phase with this parity is complete, without waiting.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}

// A tensor map over rows of q, k, v or do.  Packed: boxes of box_tokens x box_heads rows x 64 values, coordinates (value,
// head, token) or, swapped, (value, token, head).  Pages: boxes of box_tokens keys x 64 values, coordinates (value, 0,
// page * kv_heads + head).
struct RowMap {
    CUtensorMap map;
    int usable;          // 0: the strides do not fit a tensor map, rows are copied 16 bytes at a time
    int swapped;         // packed: the token is the second coordinate
};
void attn_row_map(const spamm_attn &a, const void *p, int64_t token, int64_t head, int heads, int box_heads, int box_tokens,
                  RowMap *out);
// Both maps of the keys, box_rows at a time, at most a block.
void attn_row_maps(const spamm_attn &a, int box_rows, RowMap *k, RowMap *v);

__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
                 : "memory");
}

// What this thread's ordinary stores (cp.async, st.shared) left in shared memory becomes visible to tcgen05.mma.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tiles of rows that span several query blocks
//
// A tile of 128 rows (queries x heads of a key head) reads the union of its query blocks' lists, at most 32 lists to a
// tile; a bit for each of them says which rows a block of keys counts for.  Neighbouring queries share most of their blocks,
// and where they do not, the union is still never more to copy than the lists one by one.
constexpr int UNION_LISTS = 32;
constexpr int UNION_BLOCKS = 8192;           // blocks of keys that a union is built over at a time

// Tiles of 128 rows or of 16, by the rows of a sequence and key head.  64 sequences, 8 key heads of 128, lists of up to 16 blocks
// of 64: 16 rows of as many keys take 29 us in a tile of 128 against 15 us in one of 16 (dq 26 us, 13 us), 48 rows 31 us
// against 39 us (dq 27 us, 33 us).  Over long ranges tiles of 16 read the keys once for each: 8 sequences of 8192 keys, 32 rows
// 71 us against 119 us, 16 rows (one tile either way) about the same.
inline bool attn_big_tiles(const spamm_attn &a, int64_t keys)
{
    const int64_t rows = (int64_t)a.max_q * (a.heads / a.kv_heads);
    return rows >= 36 || (rows > 16 && keys >= 4096);
}

struct TileRows {
    int rows;                 // of the tile; 0: there is none
    int row0;                 // first of the sequence's rows (query * G + head)
    int first, last;          // its first and last query
    int qb0, n_qb;            // its query blocks
};
__host__ __device__ inline int attn_tile_rows(const spamm_attn &a)
{
    if (!a.n_select) return 128;
    const int64_t most = (int64_t)UNION_LISTS * a.query_block * (a.heads / a.kv_heads);
    return most < 128 ? (int)most : 128;
}
__host__ __device__ inline int attn_tiles(const spamm_attn &a)
{
    const int rows = attn_tile_rows(a);
    return (int)(((int64_t)a.max_q * (a.heads / a.kv_heads) + rows - 1) / rows);
}
// Lists that meet in a tile, at most.
inline int attn_tile_lists(const spamm_attn &a)
{
    const int64_t per = (int64_t)a.query_block * (a.heads / a.kv_heads), rows = attn_tile_rows(a);
    const int64_t n = (rows + per - 1) / per + (rows % per && per % rows ? 1 : 0);
    return (int)(n < UNION_LISTS ? n : UNION_LISTS);
}
// Rows of a tile and the heads of a key head, made on the host (rows of a sequence are below 2^30).
struct TileShape {
    int rows;
    FastDiv G;
};
inline TileShape attn_tile_shape(const spamm_attn &a) { return TileShape{attn_tile_rows(a), fast_div((uint32_t)(a.heads / a.kv_heads))}; }
inline bool attn_tile_fits(const spamm_attn &a) { return (int64_t)a.max_q * (a.heads / a.kv_heads) < (1 << 30); }

__device__ __forceinline__ TileRows attn_tile(const spamm_attn &a, const TileShape &shape, const Seq &sq, int tile)
{
    TileRows t{};
    const int all = sq.nq * (int)shape.G.d, row0 = tile * shape.rows;
    if (row0 >= all) return t;
    t.rows = min(shape.rows, all - row0);
    t.row0 = row0;
    t.first = (int)shape.G.quotient(row0);
    t.last = (int)shape.G.quotient(row0 + t.rows - 1);
    t.qb0 = a.n_select ? t.first / a.query_block : 0;
    t.n_qb = a.n_select ? t.last / a.query_block - t.qb0 + 1 : 1;
    return t;
}
// The union of a tile's lists within the blocks [b0, b1): idx[e] = block - b0, ascending, bits[e] = the lists that have it
// (room for the sum of the lists' lengths, or b1 - b0).  `marks`: room for b1 - b0 words that nothing else uses until the
// return.  All threads call; `count` is shared.
template <int THREADS>
__device__ __forceinline__ int attn_union(const spamm_attn &a, const Seq &sq, int s, int h, const TileRows &t, int b0, int b1,
                                          uint32_t *marks, uint16_t *idx, uint32_t *bits, int *count)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = b1 - b0;
    const int nqb = ceil_div(a.max_q, a.query_block);
    for (int i = tid; i < n; i += THREADS) marks[i] = 0;
    __syncthreads();
    // (the last warps first: they are free while the others load the queries)
    for (int q = THREADS / 32 - 1 - warp; q < t.n_qb; q += THREADS / 32) {
        const int qb = t.qb0 + q;
        const int last = (int)min((int64_t)(qb + 1) * a.query_block, (int64_t)sq.nq) - 1;
        attn_for_list(a, s, qb, nqb, h, ceil_div(attn_limit(a, sq, sq.pos0 + last), a.block), lane, [&](int v, int) {
            if (v >= b0 && v < b1) atomicOr(marks + v - b0, 1u << q);
        });
    }
    __syncthreads();
    if (warp == 0) {
        int found = 0;
        for (int i0 = 0; i0 < n; i0 += 32) {
            uint32_t m = i0 + lane < n ? marks[i0 + lane] : 0;
            if (m && a.n_pages) {
                const int page = a.d_table[(int64_t)s * a.table_stride + b0 + i0 + lane];
                if (page < 0 || page >= a.n_pages) {
                    m = 0;
                    *a.d_status = SPAMM_ERR_INVALID;
                }
            }
            const unsigned there = __ballot_sync(~0u, m != 0);
            const int at = found + __popc(there & ((1u << lane) - 1));
            if (m) {
                idx[at] = (uint16_t)(i0 + lane);
                bits[at] = m;
            }
            found += __popc(there);
        }
        if (lane == 0) *count = found;
    }
    fence_async_smem();                      // tensor copies may now write where the marks were
    __syncthreads();
    return *count;
}

// Two float operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
// 2^x for two values below 128 without the special-function unit, which gives four results a clock and scheduler and would
// bound the softmax: x = n + r with r in [-1/2, 1/2] (n by adding and subtracting 1.5 * 2^23, whose sum has n in its low
// bits), 2^r by the polynomial of degree 4 with the smallest largest relative error there (2.7e-6, a Remez exchange), 2^n put
// together as bits.  At and below -127 the result is zero, and a NaN stays one.
__device__ __forceinline__ float2 poly_exp2(float2 x)
{
    const float2 magic = make_float2(12582912.f, 12582912.f), back = make_float2(-12582912.f, -12582912.f);
    x.x = max_nan(x.x, -127.f);
    x.y = max_nan(x.y, -127.f);
    const float2 t = add2(x, magic);
    const float2 n = add2(t, back);
    const float2 r = fma2(n, make_float2(-1.f, -1.f), x);
    float2 p = fma2(make_float2(0.009570102207362652f, 0.009570102207362652f), r, make_float2(0.05591785907745361f, 0.05591785907745361f));
    p = fma2(p, r, make_float2(0.240247443318367f, 0.240247443318367f));
    p = fma2(p, r, make_float2(0.6931217908859253f, 0.6931217908859253f));
    p = fma2(p, r, make_float2(0.9999992847442627f, 0.9999992847442627f));
    const float2 s = make_float2(__uint_as_float((__float_as_uint(t.x) << 23) + 0x3f800000u),
                                 __uint_as_float((__float_as_uint(t.y) << 23) + 0x3f800000u));
    return mul2(p, s);
}

// ---- results by way of shared memory
//
// A thread has a row of an accumulator; stored from there, every warp instruction would touch 32 lines.  The rows go to
// shared memory first (16-byte pieces XORed with the row, no bank conflicts either way) and leave as whole rows.
__device__ __forceinline__ uint32_t row_piece(int row_bytes, int r, int c) { return r * row_bytes + ((c ^ (r & 7)) << 4); }

// ---- rows taken key by key
//
// A tile multiplies every row with every key of its steps, those that the row does not read with p (or ds) = 0: a NaN or an
// infinity among their values would reach the row all the same, as 0 * NaN.  Rows whose result is not finite are therefore
// taken again over their own keys alone, one warp for a row, some 0.3 us a key.  As that would be minutes where every row of
// long sequences reads such a value, it is done only where it can change a result:
//   not for rows whose own scores are NaN, as their sum over visible keys tells (in the backward lse, or delta where they see a
//   key): all their results are;
//   not for rows whose results are not finite in columns alone where a value that they read is not either (sure_columns).

__device__ __forceinline__ bool not_finite(uint32_t v) { return (v & 0x7f800000u) == 0x7f800000u; }

// Elements lane * D/32 .. of a row of D values.
template <typename T, int D> __device__ __forceinline__ void row_load(const T *p, int lane, float *x)
{
#pragma unroll
    for (int i = 0; i < D / 32; i += 2) {
        const float2 f = Pack<T>::to2(*reinterpret_cast<const uint32_t *>(p + lane * (D / 32) + i));
        x[i] = f.x;
        x[i + 1] = f.y;
    }
}
template <int D> __device__ __forceinline__ float row_dot(const float *x, const float *y)
{
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; i++) z = fmaf(x[i], y[i], z);
#pragma unroll
    for (int d = 16; d; d >>= 1) z += __shfl_xor_sync(~0u, z, d);
    return z;
}
// Calls f(k row, v row) for every key below `limit` of the blocks that block(e) names for e in [0, n) (-1: not the row's).
template <typename T, typename Block, typename F>
__device__ __forceinline__ void row_keys(const spamm_attn &a, const Seq &sq, int s, int h, int n, int limit, Block block, F f)
{
    for (int e = 0; e < n; e++) {
        const int b = block(e);
        if (b < 0) continue;
        const int64_t k0 = attn_block_base(a, sq, s, h, b, a.k_token, a.k_head);
        if (k0 < 0) continue;
        const int64_t v0 = a.n_pages ? k0 : (int64_t)(sq.row0 + b * a.block) * a.v_token + h * a.v_head;
        const int64_t k_tok = a.n_pages ? a.dim : a.k_token, v_tok = a.n_pages ? a.dim : a.v_token;
        const int keys = min(a.block, limit - b * a.block);
        for (int i = 0; i < keys; i++) f(static_cast<const T *>(a.d_k) + k0 + i * k_tok, static_cast<const T *>(a.d_v) + v0 + i * v_tok);
    }
}
// For every column of k or v (`rows`) the lists, as bits, that read a value there that is not finite, at a position below `limit`,
// which all rows of the tile see: sure[D], zeros before, by `threads` threads.  Entries are blocks b0 + idx[e], blk[e] or b0 + e, and
// their lists bits[e], or all.
template <typename T, int D>
static __device__ __noinline__ void sure_columns(const spamm_attn &a, const Seq &sq, int s, int h, const T *rows, int64_t token, int64_t head,
                                                 int n_entries, int b0, const uint16_t *idx, const int *blk, const uint32_t *bits, int limit,
                                                 uint32_t *sure, int t, int threads)
{
    constexpr uint32_t ONE = IsBf<T>::value ? 0x00800080u : 0x04000400u;      // carries an exponent of all ones into the sign's place
    constexpr int AHEAD = 4;
    const int c = t % (D / 8), step = threads / (D / 8), log_block = 31 - __clz(a.block), n = n_entries << log_block;
    for (int i0 = t / (D / 8); i0 < n; i0 += AHEAD * step) {
        uint4 x[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const int i = i0 + u * step, e = i >> log_block, r = i & (a.block - 1);
            x[u] = make_uint4(0, 0, 0, 0);
            if (i >= n) continue;
            const int b = idx ? b0 + idx[e] : blk ? blk[e] : b0 + e;
            if (b * a.block + r >= limit) continue;
            const int64_t at = attn_block_base(a, sq, s, h, b, token, head);
            if (at >= 0) x[u] = *reinterpret_cast<const uint4 *>(rows + at + r * (a.n_pages ? (int64_t)D : token) + c * 8);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; u++) {
            const uint32_t y[4] = {x[u].x & 0x7fff7fffu, x[u].y & 0x7fff7fffu, x[u].z & 0x7fff7fffu, x[u].w & 0x7fff7fffu};
            if (!(((y[0] + ONE) | (y[1] + ONE) | (y[2] + ONE) | (y[3] + ONE)) & 0x80008000u)) continue;
            const uint32_t who = bits ? bits[(i0 + u * step) >> log_block] : ~0u;
            for (int k = 0; k < 4; k++) {
                if ((y[k] + ONE) & 0x8000u) atomicOr(sure + c * 8 + 2 * k, who);
                if ((y[k] + ONE) & 0x80000000u) atomicOr(sure + c * 8 + 2 * k + 1, who);
            }
        }
    }
}
// Whether some of a pair of results, columns d and d + 1, is not finite and not for sure.
__device__ __forceinline__ bool unsure(float2 x, const uint32_t *sure, int d, uint32_t bit)
{
    return (not_finite(__float_as_uint(x.x)) && !(sure[d] & bit)) || (not_finite(__float_as_uint(x.y)) && !(sure[d + 1] & bit));
}

// One key with the score z (times log2 e) joins a row's running maximum, sum and output.
template <int D> __device__ __forceinline__ void online_row(float z, const float *v, float *o, float *top, float *sum)
{
    const float next = fmaxf(*top, z);
    const float f = *top == next ? 1.f : fast_exp2(*top - next), w = fast_exp2(z - (next == -CUDART_INF_F ? 0.f : next));
    *top = next;
    *sum = *sum * f + w;
#pragma unroll
    for (int i = 0; i < D / 32; i++) o[i] = o[i] * f + w * v[i];
}
// Barriers of a kernel and its abort flag: a wait that runs out (never, unless the kernel is wrong) sets the flag, every
// role leaves its loop, and the results of the tile become NaN.
struct WaitState {
    volatile uint32_t *abort_flag;
    int32_t *err;                       // in shared memory
    __device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, int code) const
    {
        return wait_bounded(bar, parity & 1u, abort_flag, err, code);
    }
};

// After an aborted wait products may still be in flight; they end before their tensor memory is given back.
static __device__ __noinline__ void drain_products()
{
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 1000000ull) {}
}

}  // namespace spamm
