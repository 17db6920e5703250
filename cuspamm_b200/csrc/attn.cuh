// What the attention kernels share: argument checks, the geometry of sequences and lists on the device, and small
// wrappers of the warp-level instructions (16-byte asynchronous copies, ldmatrix, m16n8k16 products).
#pragma once
#include <cuda_bf16.h>
#include <math_constants.h>
#include "common.cuh"

namespace spamm {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// 0 when the fields that every attention entry point reads are in range.
int attn_check(const spamm_attn *a, bool need_lists);
bool attn_rows_ok(const void *p, int64_t token, int64_t head);   // 16-byte aligned rows
inline int attn_query_blocks(const spamm_attn &a) { return ceil_div(a.max_q, a.query_block); }
// Blocks of the longest sequence that a call may meet.
inline int attn_max_blocks(const spamm_attn &a) { return a.n_pages ? a.table_width : ceil_div(a.max_q, a.block); }
int attn_set_smem(const void *kernel);
int attn_refuse(const char *why);     // records the text, gives SPAMM_ERR_INVALID
int attn_too_large();                 // the same for a grid beyond 2^31 - 1, SPAMM_ERR_UNSUPPORTED

// Division of numbers below 2^31 by a fixed one: n / d = (n * m) >> (32 + s) with m = ceil(2^(32+s) / d), s = ceil(log2 d) - 1
// (m < 2^32 and the excess m*d - 2^(32+s) < d <= 2^(s+1) keeps the quotient exact for n < 2^31).
struct FastDiv {
    uint32_t d, m, s;
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return d == 1 ? n : __umulhi(n, m) >> s; }
};
inline FastDiv fast_div(uint32_t d)
{
    FastDiv f{d, 0, 0};
    if (d > 1) {
        while ((2u << f.s) < d) f.s++;
        f.m = (uint32_t)((((uint64_t)1 << (32 + f.s)) + d - 1) / d);
    }
    return f;
}

struct Seq {
    int row0;     // first row of q (and of packed k, v)
    int nq;       // queries that are computed
    int nk;       // keys held
    int pos0;     // position of the first query (may lie before 0, or behind nk)
};

__device__ __forceinline__ Seq attn_seq(const spamm_attn &a, int s)
{
    Seq r;
    r.row0 = min(max(a.d_cu[s], 0), a.tokens);
    const int all = min(max(a.d_cu[s + 1], r.row0), a.tokens) - r.row0;
    r.nq = min(all, a.max_q);
    if (all > a.max_q && a.d_status) *a.d_status = SPAMM_ERR_INVALID;
    if (a.n_pages) {
        const int64_t room = (int64_t)a.table_width * a.block;
        const int held = a.d_lengths[s];
        r.nk = (int)min((int64_t)max(held, 0), room);
        if (held != r.nk && a.d_status) *a.d_status = SPAMM_ERR_INVALID;
        r.pos0 = max(held, 0) - all;       // a length beyond the table moves no token from its position
    } else {
        r.nk = r.nq;
        r.pos0 = 0;
    }
    return r;
}

// First row behind the last sequence.
__device__ __forceinline__ int attn_rows_end(const spamm_attn &a)
{
    return min(max(a.d_cu[a.batch], 0), a.tokens);
}

// Keys that the query at position p sees: [0, this).
__device__ __forceinline__ int attn_limit(const spamm_attn &a, const Seq &sq, int pos)
{
    return a.causal ? min(max(pos + 1, 0), sq.nk) : sq.nk;
}

// Element offset of the first row of block b of key head h in k (packed or paged); -1 for a page that does not exist.
__device__ __forceinline__ int64_t attn_block_base(const spamm_attn &a, const Seq &sq, int s, int h, int b, int64_t token,
                                                   int64_t head)
{
    if (a.n_pages) {
        const int page = a.d_table[(int64_t)s * a.table_stride + b];
        if (page < 0 || page >= a.n_pages) {
            if (a.d_status) *a.d_status = SPAMM_ERR_INVALID;
            return -1;
        }
        return ((int64_t)page * a.kv_heads + h) * a.block * a.dim;
    }
    return (int64_t)(sq.row0 + b * a.block) * token + h * head;
}

// One warp walks the list of (s, qb, h) and calls f(entry, how many kept before it) for every entry that counts: no f for
// what is no block below n_blocks or not above every entry before it.  Returns how many there are.
template <typename F>
__device__ __forceinline__ int attn_for_list(const spamm_attn &a, int s, int qb, int nqb, int h, int n_blocks, int lane, F f)
{
    const int32_t *list = a.d_lists + (((int64_t)s * nqb + qb) * a.kv_heads + h) * a.n_select;
    int count = 0, top = -1;
    for (int base = 0; base < a.n_select; base += 32) {
        int v = base + lane < a.n_select ? list[base + lane] : -1;
        if (v >= n_blocks) v = -1;
        int run = max(v, -1);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(~0u, run, d);
            if (lane >= d) run = max(run, o);
        }
        int before = __shfl_up_sync(~0u, run, 1);
        before = max(lane ? before : -1, top);
        const bool keep = v > before;
        const unsigned m = __ballot_sync(~0u, keep);
        if (keep) f(v, count + __popc(m & ((1u << lane) - 1)));
        count += __popc(m);
        top = max(top, __shfl_sync(~0u, run, 31));
    }
    __syncwarp();
    return count;
}
// The same into an array with room for n_select.  n_blocks: of the whole query block, as what counts must not depend on the
// tile that asks; returns how many are below `reached`, those that the tile's rows may see.
__device__ __forceinline__ int attn_load_list(const spamm_attn &a, int s, int qb, int nqb, int h, int n_blocks, int reached, int *out, int lane)
{
    const int n = attn_for_list(a, s, qb, nqb, h, n_blocks, lane, [&](int v, int i) { out[i] = v; });
    if (reached >= n_blocks) return n;
    int below = 0;
    for (int i = lane; i < n; i += 32) below += out[i] < reached;
    return __reduce_add_sync(~0u, below);
}

// ---- types
template <typename T> struct Pack;
template <> struct Pack<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t two(float a, float b)
    {
        __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&x);
    }
    static __device__ __forceinline__ float2 to2(uint32_t v)
    {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ __nv_bfloat16 one(float a) { return __float2bfloat16_rn(a); }
};
template <> struct Pack<__half> {
    static __device__ __forceinline__ uint32_t two(float a, float b)
    {
        __half2 x = __floats2half2_rn(a, b);
        return *reinterpret_cast<uint32_t *>(&x);
    }
    static __device__ __forceinline__ float2 to2(uint32_t v)
    {
        return __half22float2(*reinterpret_cast<__half2 *>(&v));
    }
    static __device__ __forceinline__ __half one(float a) { return __float2half_rn(a); }
};

// ---- warp-level instructions
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes to shared memory, zeros when !ok (the address is then not read).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool ok)
{
    const int n = ok ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(n)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int n> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(n) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t *r)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t *r)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T> __device__ __forceinline__ void mma16816(float *c, const uint32_t *a, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float *c, const uint32_t *a, uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fast_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Byte offset of 16-byte piece `c` of row `r` in a shared tile of rows of D values: pieces are XORed with the row so
// that eight consecutive rows of one column touch all banks.
template <int D> __device__ __forceinline__ uint32_t tile_off(int r, int c) { return r * (D * 2) + ((c ^ (r & 7)) << 4); }

// Fragments of m16n8k16 from such tiles (lane = this thread's lane).
//   a_frag   A: rows r0..r0+15, values 16*ks..  (row-major)
//   b_frag2  B for two groups of 8 columns, where the tile's rows are the columns n of B: rows r0..r0+15, values 16*ks..
//            -> b[0], b[1] for columns r0..r0+7, b[2], b[3] for r0+8..r0+15
//   bt_frag2 B where the tile's rows are the k of B: rows r0..r0+15, values n0..n0+15
//            -> b[0], b[1] for columns n0..n0+7, b[2], b[3] for n0+8..n0+15
template <int D> __device__ __forceinline__ void a_frag(uint32_t tile, int r0, int ks, int lane, uint32_t *a)
{
    ldsm4(tile + tile_off<D>(r0 + (lane & 15), 2 * ks + (lane >> 4)), a);
}
template <int D> __device__ __forceinline__ void b_frag2(uint32_t tile, int r0, int ks, int lane, uint32_t *b)
{
    ldsm4(tile + tile_off<D>(r0 + (lane & 7) + ((lane >> 4) << 3), 2 * ks + ((lane >> 3) & 1)), b);
}
template <int D> __device__ __forceinline__ void bt_frag2(uint32_t tile, int r0, int n0, int lane, uint32_t *b)
{
    ldsm4t(tile + tile_off<D>(r0 + (lane & 15), (n0 >> 3) + (lane >> 4)), b);
}

}  // namespace spamm
