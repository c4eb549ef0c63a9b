// A cache of keys and values in pages: what its operators share, rows into pages and back, and attention of one row at a time.
//
// Pool of a layer: [page][keys, values][key / value head][token of the page][dimension], so that a page's tokens of one head lie one behind the other
// (attention reads them as one run).  A sequence's pages are in its row of a table of page numbers.  Elements are bf16, fp32, or e4m3 codes with one
// power of two per token and head (exponent + 127, a byte, [page][keys, values][head][token]).
//
// Why a power of two: e4m3 has the same relative precision over fourteen powers of two, so a finer scale buys nothing, and with this one every
// division, product and stored value is exact in fp32 and in bf16: a code read back is one value, whoever reads it.  One byte instead of four per head
// and token is 3 % of a cache of heads of 64.
#pragma once

#include <cfloat>
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include "../../include/gptb200.h"
#include "gemm_sm100.cuh"

namespace gptb200 {
namespace kvp {

enum Kind : int { KIND_BF16 = GPTB200_KV_BF16, KIND_F32 = GPTB200_KV_F32, KIND_E4M3 = GPTB200_KV_E4M3 };

// The smallest power of two whose 448 multiples reach a row's largest value lies in this range; beyond it codes saturate or vanish.  Every code times
// every such power is zero or a normal number of fp32 and of bf16.
constexpr int kMinExponent = -117, kMaxExponent = 119;

struct Pages {
    void *data;
    uint8_t *scales;   // e4m3 only
    int num_pages, page_shift, kv_heads, dim;

    // element (page, which, head, token, 0), in elements; without the last factor the place in `scales`
    __device__ __forceinline__ long long place(int page, int which, int head, int token) const
    {
        return ((((static_cast<long long>(page) * 2 + which) * kv_heads + head) << page_shift) + token);
    }
};

struct Batch {
    const int *row_starts, *lengths, *table;
    int sequences, table_pitch, rows;
    int capacity;      // tokens that a row of the table can hold, at most 2^30
    int *status;
};

// A sequence's new rows: row0 .. row0 + count - 1 at positions pos0, pos0 + 1, ...; positions below zero hold nothing and see nothing.
struct Sequence {
    int row0, count, pos0;
};

__host__ __device__ inline void report_bad(int *status)
{
#ifdef __CUDA_ARCH__
    atomicCAS(status, 0, DEV_BAD_PAGES);
#else
    if (*status == 0) *status = DEV_BAD_PAGES;
#endif
}

__host__ __device__ inline int smaller(int a, int b) { return a < b ? a : b; }
__host__ __device__ inline int larger(int a, int b) { return a > b ? a : b; }

// Whatever the three arrays hold, the rows lie inside the tensors and the positions inside the table.
__host__ __device__ inline Sequence sequence_of(const Batch &b, int s)
{
    const int first = b.row_starts[s], end = b.row_starts[s + 1], length = b.lengths[s];
    Sequence q;
    q.row0 = smaller(larger(first, 0), b.rows);
    q.count = smaller(larger(end, q.row0), b.rows) - q.row0;
    const int n = smaller(larger(length, 0), b.capacity);
    q.pos0 = n - q.count;
    if (q.row0 != first || q.row0 + q.count != end || n != length) report_bad(b.status);
    return q;
}

// Page of a sequence's token at a position within [0, capacity); -1 (and a report) when the table holds no page's number.
__host__ __device__ inline int page_of(const Batch &b, const Pages &p, int s, int position)
{
    const int page = b.table[static_cast<long long>(s) * b.table_pitch + (position >> p.page_shift)];
    if (page >= 0 && page < p.num_pages) return page;
    report_bad(b.status);
    return -1;
}

// ---- eight elements of one row

__device__ __forceinline__ void load8(float (&v)[8], const float *src)
{
    const float4 a = *reinterpret_cast<const float4 *>(src), b = *reinterpret_cast<const float4 *>(src + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ void load8(float (&v)[8], const __nv_bfloat16 *src)
{
    const uint4 w = *reinterpret_cast<const uint4 *>(src);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_low(x[i]);
        v[2 * i + 1] = bf16_high(x[i]);
    }
}
__device__ __forceinline__ void store8(float *dst, const float (&v)[8])
{
    *reinterpret_cast<float4 *>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4 *>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16 *dst, const float (&v)[8])
{
    *reinterpret_cast<uint4 *>(dst) = make_uint4(ptx::pack_bf16x2(v[0], v[1]), ptx::pack_bf16x2(v[2], v[3]), ptx::pack_bf16x2(v[4], v[5]), ptx::pack_bf16x2(v[6], v[7]));
}

// Two codes (the low sixteen bits) as fp32 values, exactly.
__device__ __forceinline__ float2 codes2(uint32_t pair)
{
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair), __NV_E4M3);
    return __half22float2(__half2(h));
}
// Rounded to nearest even, beyond 448 the largest code; neither infinities nor NaN come here
__device__ __forceinline__ uint32_t to_codes2(float a, float b)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ float scale_of(uint32_t stored) { return __uint_as_float(stored << 23); }

__device__ __forceinline__ void codes8(float (&v)[8], uint2 w, float scale)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 c = codes2((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
        v[2 * i] = c.x * scale;
        v[2 * i + 1] = c.y * scale;
    }
}

__device__ __forceinline__ void load8_codes(float (&v)[8], const uint8_t *src, float scale) { codes8(v, *reinterpret_cast<const uint2 *>(src), scale); }

// The smallest e with most <= 448 * 2^e, from most's exponent and mantissa (448 = 1.75 * 2^8).
__device__ __forceinline__ int exponent_for(float most)
{
    const uint32_t bits = __float_as_uint(most);
    const int e = static_cast<int>(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(e, kMinExponent), kMaxExponent);
}

// Rows of keys and values <-> pages.  A piece of sixteen elements per lane (eight where a head has an odd number of eights); as many lanes as a head has pieces (a power of two of them) hold a head, so that a row's
// largest value is a few shuffles.  A thread keeps to its piece of the row and walks down the rows: no index is formed twice.  Bound by DRAM as far as copies go; with
// codes by instructions (a row's largest value, a conversion per pair), which is why the largest value of bf16 rows is found two at a time on their bits.
constexpr int kRowThreads = 256;
constexpr int kRowMax = 64;    // rows per block, at most
constexpr int kCheckedStarts = 1024;   // sequences whose starts a block checks
// Pieces under way per thread, blocks per SM, rows per thread.  Writing (24 400 rows of 8 heads of 128 from bf16 to codes): 40 us with four blocks of four pieces each, 5.0 TB/s;
// 56 us with rows looked up by a warp each and two blocks.  Reading (16 600 rows of 4 heads back): 22.7 us with eight blocks and one piece, 4.8 TB/s; 33 us with
// four pieces each.
__host__ __device__ constexpr int row_batch(bool write) { return write ? 4 : 1; }
__host__ __device__ constexpr int row_blocks(bool write) { return write ? 4 : 8; }
__host__ __device__ constexpr int row_turns(bool write) { return write ? 8 : 4; }

struct RowsArgs {
    Pages pages;
    Batch batch;
    void *k, *v;
    long long k_pitch, v_pitch;
    int lanes_log2;      // lanes per head
    int columns;         // threads that share a row: all its pieces, or the block
    int rows_per_block;
    unsigned int row_blocks;   // blocks that have rows; those behind them check starts
};

// Eight elements as they lie in memory.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) { w = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void zero() { w = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const
    {
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = bf16_low(x[i]);
            v[2 * i + 1] = bf16_high(x[i]);
        }
    }
    // bits of the largest magnitude as fp32; not finite ones are larger than all others
    __device__ __forceinline__ uint32_t largest() const
    {
        const uint32_t m = __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
        return max(m & 0xffff0000u, m << 16);
    }
};
template <> struct Raw8<float> {
    uint4 w, u;
    __device__ __forceinline__ void load(const float *p)
    {
        w = *reinterpret_cast<const uint4 *>(p);
        u = *reinterpret_cast<const uint4 *>(p + 4);
    }
    __device__ __forceinline__ void zero() { w = u = make_uint4(0u, 0u, 0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const
    {
        const uint32_t x[8] = {w.x, w.y, w.z, w.w, u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(x[i]);
    }
    __device__ __forceinline__ uint32_t largest() const
    {
        constexpr uint32_t bits = 0x7fffffffu;
        return max(max(max(w.x & bits, w.y & bits), max(w.z & bits, w.w & bits)), max(max(u.x & bits, u.y & bits), max(u.z & bits, u.w & bits)));
    }
};

// WRITE: rows of T into pages of KIND, else the other way.
// EIGHTS: groups of eight elements per piece.
template <typename T, int KIND, bool WRITE, int EIGHTS>
__global__ void __launch_bounds__(kRowThreads, row_blocks(WRITE))
kv_rows_kernel(const RowsArgs a)
{
    constexpr int kRowBatch = row_batch(WRITE);
    __shared__ int where[kRowMax][2];   // page (-1: none) and token within it
    grid_dependency_wait();
    grid_dependency_launch();
    const int first = blockIdx.x * a.rows_per_block, rows = min(a.rows_per_block, a.batch.rows - first);   // of a block that has some
    // Starts out of order may leave sequences that no row leads to: blocks behind the rows' look at all of them.
    if (blockIdx.x >= a.row_blocks) {
        const long long from = static_cast<long long>(blockIdx.x - a.row_blocks) * kCheckedStarts;
        for (long long s = from + threadIdx.x; s < min(from + kCheckedStarts, static_cast<long long>(a.batch.sequences)); s += blockDim.x) {
            const int begin = a.batch.row_starts[s], end = a.batch.row_starts[s + 1];
            if (begin < 0 || end < begin || end > a.batch.rows) report_bad(a.batch.status);
        }
        return;
    }
    const int per = 1 << a.lanes_log2, heads = a.pages.kv_heads, dim = a.pages.dim, all_columns = 2 * heads << a.lanes_log2;
    const int row0 = threadIdx.x / a.columns, column0 = threadIdx.x - row0 * a.columns, step = blockDim.x / a.columns;
    // a thread per row: the loads of a look-up depend on one another, so the rows' chains run side by side
    for (int r = threadIdx.x; r < rows; r += blockDim.x) {
        const int row = first + r;
        int low = 0, high = a.batch.sequences, page = -1, token = 0;   // the last s with row_starts[s] <= row
        while (high - low > 1) {
            const int middle = low + (high - low) / 2;
            if (a.batch.row_starts[middle] <= row)
                low = middle;
            else
                high = middle;
        }
        const Sequence q = sequence_of(a.batch, low);
        const int nth = row - q.row0, position = q.pos0 + nth;
        if (nth >= 0 && nth < q.count && position >= 0) {
            page = page_of(a.batch, a.pages, low, position);
            token = position & ((1 << a.pages.page_shift) - 1);
        }
        where[r][0] = page;
        where[r][1] = token;
    }
    const long long head_tokens = 1LL << a.pages.page_shift, page_tokens = 2 * heads * head_tokens;
    bool begun = false;
    for (int c0 = 0; c0 < all_columns; c0 += a.columns) {
        const int column = c0 + column0, unit = column >> a.lanes_log2, piece = column & (per - 1), which = unit >= heads, h = which ? unit - heads : unit;
        const bool active = row0 < step && column < all_columns && piece * 8 * EIGHTS < dim;
        const long long pitch = which ? a.v_pitch : a.k_pitch, head_at = (which * heads + h) * head_tokens;
        T *column_rows = static_cast<T *>(which ? a.v : a.k) + first * pitch + h * dim + piece * 8 * EIGHTS;
        Raw8<T> raw[kRowBatch][EIGHTS];
        auto load_rows = [&](int base) {   // the rows' own addresses need no page
#pragma unroll
            for (int i = 0; i < kRowBatch; ++i) {
                const int r = base + i * step;
#pragma unroll
                for (int x = 0; x < EIGHTS; ++x) {
                    raw[i][x].zero();
                    if (active && r < rows) raw[i][x].load(column_rows + r * pitch + 8 * x);
                }
            }
        };
        if constexpr (WRITE) load_rows(row0);
        if (!begun) __syncthreads();
        begun = true;
        for (int base = 0; base < rows; base += kRowBatch * step) {   // the same for all threads: shuffles below
            if constexpr (!WRITE) {
                const int r = base + row0, page = active && r < rows ? where[r][0] : -1;
                if (page >= 0) {
                    const long long at = page * page_tokens + head_at + where[r][1], from = at * dim + piece * 8 * EIGHTS;
                    float v[EIGHTS][8];
                    if constexpr (KIND == KIND_E4M3) {
                        const float scale = scale_of(a.pages.scales[at]);
                        const uint8_t *codes = static_cast<const uint8_t *>(a.pages.data) + from;
                        if constexpr (EIGHTS == 2) {
                            const uint4 w = *reinterpret_cast<const uint4 *>(codes);
                            codes8(v[0], make_uint2(w.x, w.y), scale);
                            codes8(v[1], make_uint2(w.z, w.w), scale);
                        } else {
                            load8_codes(v[0], codes, scale);
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < EIGHTS; ++x) {
                            if constexpr (KIND == KIND_BF16)
                                load8(v[x], static_cast<const __nv_bfloat16 *>(a.pages.data) + from + 8 * x);
                            else
                                load8(v[x], static_cast<const float *>(a.pages.data) + from + 8 * x);
                        }
                    }
#pragma unroll
                    for (int x = 0; x < EIGHTS; ++x) store8(column_rows + r * pitch + 8 * x, v[x]);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kRowBatch; ++i) {
                    const int r = base + row0 + i * step, page = active && r < rows ? where[r][0] : -1;
                    const bool on = page >= 0;
                    const long long at = on ? page * page_tokens + head_at + where[r][1] : 0, to = at * dim + piece * 8 * EIGHTS;
                    float v[EIGHTS][8];
#pragma unroll
                    for (int x = 0; x < EIGHTS; ++x) raw[i][x].get(v[x]);
                    if constexpr (KIND == KIND_E4M3) {
                        constexpr uint32_t infinity = 0x7f800000u;
                        uint32_t most = raw[i][0].largest(), bad = 0;
                        if constexpr (EIGHTS == 2) most = max(most, raw[i][1].largest());
                        if (most >= infinity) {   // the largest finite one counts
                            most = 0;
#pragma unroll
                            for (int e = 0; e < 8 * EIGHTS; ++e) {
                                const uint32_t bits = __float_as_uint(v[e >> 3][e & 7]) & 0x7fffffffu;
                                if (bits >= infinity) {
                                    bad |= 1u << e;
                                    v[e >> 3][e & 7] = 0.0f;
                                } else {
                                    most = max(most, bits);
                                }
                            }
                        }
#pragma unroll
                        for (int o = 1; o < 16; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o < per ? o : 0));
                        const int exponent = exponent_for(__uint_as_float(most));
                        const float by = power_of_two(-exponent);
                        uint32_t w[2 * EIGHTS];
#pragma unroll
                        for (int x = 0; x < EIGHTS; ++x) {
                            uint32_t c[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) c[e] = to_codes2(v[x][2 * e] * by, v[x][2 * e + 1] * by);
                            if (bad) {   // the format has no infinity: both kinds become its NaN
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    if (bad >> (8 * x + 2 * e) & 1) c[e] = (c[e] & 0xff00u) | 0x7fu;
                                    if (bad >> (8 * x + 2 * e + 1) & 1) c[e] = (c[e] & 0x00ffu) | 0x7f00u;
                                }
                            }
                            w[2 * x] = __byte_perm(c[0], c[1], 0x5410);
                            w[2 * x + 1] = __byte_perm(c[2], c[3], 0x5410);
                        }
                        if (on) {
                            uint8_t *codes = static_cast<uint8_t *>(a.pages.data) + to;
                            if constexpr (EIGHTS == 2)
                                *reinterpret_cast<uint4 *>(codes) = make_uint4(w[0], w[1], w[2], w[3]);
                            else
                                *reinterpret_cast<uint2 *>(codes) = make_uint2(w[0], w[1]);
                            if (piece == 0) a.pages.scales[at] = static_cast<uint8_t>(exponent + 127);
                        }
                    } else if (on) {
#pragma unroll
                        for (int x = 0; x < EIGHTS; ++x) {
                            if constexpr (KIND == KIND_BF16)
                                store8(static_cast<__nv_bfloat16 *>(a.pages.data) + to + 8 * x, v[x]);
                            else
                                store8(static_cast<float *>(a.pages.data) + to + 8 * x, v[x]);
                        }
                    }
                }
                if (base + kRowBatch * step < rows) load_rows(base + kRowBatch * step + row0);
            }
        }
    }
}

// Division of numbers below 2^31 by a number known on the host, as a product and a shift (Granlund and Montgomery, Division by invariant integers using
// multiplication, 1994): a tile's positions take half a dozen divisions by the group's size, which were 3 000 cycles between two tiles.
struct Divisor {
    uint32_t by = 1, factor = 0;
    int shift = 0;
    __host__ __device__ inline int divide(int n) const
    {
#ifdef __CUDA_ARCH__
        return static_cast<int>((__umulhi(static_cast<uint32_t>(n), factor) + static_cast<uint32_t>(n)) >> shift);
#else
        return static_cast<int>((static_cast<uint32_t>((static_cast<uint64_t>(n) * factor) >> 32) + static_cast<uint32_t>(n)) >> shift);
#endif
    }
};
inline Divisor divisor(uint32_t by)
{
    Divisor d;
    d.by = by;
    while ((1ull << d.shift) < by) ++d.shift;
    d.factor = static_cast<uint32_t>((((1ull << d.shift) - by) << 32) / by + 1);
    return d;
}

// ---- attention

struct Attention {
    Pages pages;
    Batch batch;
    const void *q;
    void *out;
    float *lse;                // [rows][heads] or null
    long long q_pitch, out_pitch;
    int heads, share;          // share: query heads per key / value head
    Divisor shares;
    float scale, cap;          // cap 0: none
    int window, sinks;         // window 0: all earlier tokens
};

__host__ __device__ inline bool visible(const Attention &a, int key, int position)
{
    return key <= position && (a.window == 0 || key > position - a.window || key < a.sinks);
}

// ---- the line of work that the tiled kernels share
//
// A tile is a number of packed query rows of one sequence and key / value head: row i of the tile is head i % share of token i / share, so that a group's
// query heads meet keys and values once.  A tile's work is the blocks of keys that any of its rows sees; all tiles' blocks form one line (sequence, key / value
// head, tile, block), which is cut into equal ranges, one per block of the grid: whatever the lengths, all blocks do nearly the same work.  A range may begin and
// end inside a tile, though a cut within an eighth of a range from a tile's edge moves to the edge; such parts go to scratch as (maximum, sum, weighted values), and the block that arrives last at a tile adds them up in the order of
// the line, so that results do not depend on who that is.

struct KeyBlocks {
    int first_ones;   // blocks 0 .. first_ones - 1 (the first tokens that stay visible) ...
    int from;         // ... then from, from + 1, ...
    int count;        // in all, at least 1: a tile that sees nothing has its output to write
};

// Blocks of `keys` keys for rows at positions p0 .. p1.
__host__ __device__ inline KeyBlocks key_blocks(int p0, int p1, int window, int sinks, int keys)
{
    if (p1 < 0) return {0, 0, 1};
    const unsigned n = keys;
    const int from = window > 0 ? static_cast<int>(larger(0, p0 - window + 1) / n) : 0;
    const int ones = window > 0 ? smaller(static_cast<int>((smaller(sinks, p1 + 1) + n - 1) / n), from) : 0;
    return {ones, from, ones + static_cast<int>(p1 / n) - from + 1};
}
__host__ __device__ inline int block_key(const KeyBlocks &b, int i, int keys) { return (i < b.first_ones ? i : b.from + i - b.first_ones) * keys; }

// Tile t of a sequence's rows of one key / value head.
__host__ __device__ inline KeyBlocks tile_blocks(const Attention &a, const Sequence &q, int t, int tile_rows, int keys)
{
    const int first = t * tile_rows, last = smaller((t + 1) * tile_rows, q.count * a.share) - 1;
    return key_blocks(q.pos0 + a.shares.divide(first), q.pos0 + a.shares.divide(last), a.window, a.sinks, keys);
}
__host__ __device__ inline int tiles_of(const Attention &a, const Sequence &q, int tile_rows) { return (q.count * a.share + tile_rows - 1) / tile_rows; }

// How a kernel cuts the line: rows of a tile, keys of a block, blocks that a tile's own costs stand for, blocks per range at least.
struct Cut {
    int tile_rows, keys, lead, least;
};

__host__ __device__ inline long long blocks_of(const Attention &a, const Sequence &q, const Cut &cut)
{
    const int tiles = tiles_of(a, q, cut.tile_rows);
    long long n = 1LL * tiles * cut.lead;
    for (int t = 0; t < tiles; ++t) n += tile_blocks(a, q, t, cut.tile_rows, cut.keys).count;
    return n;
}

// Where a block of the grid stands on the line.
struct Place {
    Sequence q;
    KeyBlocks blocks;
    int s, g, tile, tiles;
    int off;              // place within the tile: `lead` ones without a block of keys, then its blocks
};

// Next tile that has rows; false behind the last one.
__host__ __device__ inline bool next_tile(const Attention &a, Place &p, const Cut &cut)
{
    p.off = 0;
    if (++p.tile >= p.tiles) {
        p.tile = 0;
        if (++p.g >= a.pages.kv_heads) {
            p.g = 0;
            do {
                if (++p.s >= a.batch.sequences) return false;
                p.q = sequence_of(a.batch, p.s);
            } while (p.q.count == 0);
            p.tiles = tiles_of(a, p.q, cut.tile_rows);
        }
    }
    p.blocks = tile_blocks(a, p.q, p.tile, cut.tile_rows, cut.keys);
    return true;
}

struct Range {
    long long begin, end;   // this block's part of the line; the last one's has no end
    long long per;          // of every block of the grid
    int snap;               // a cut this near to a tile's edge moves there
};

// Range c of a line of `total` places cut for `grid` blocks, before its beginning has moved to a tile's edge.
__host__ __device__ inline Range range_of(long long total, int c, int grid, const Cut &cut)
{
    Range r;
    r.per = (total + grid - 1) / grid;
    if (r.per < cut.least) r.per = cut.least;
    r.snap = static_cast<int>(r.per / 8 < 1 << 20 ? r.per / 8 : 1 << 20);
    if (r.snap < cut.lead) r.snap = cut.lead;   // no cut among the places in front of a tile's blocks
    r.begin = r.per * c;
    r.end = r.begin + r.per < total ? r.begin + r.per : total + r.snap + 1;
    if (r.begin >= total) r.begin = r.end = total;
    return r;
}
// The beginning moves to a near edge of the tile that holds it; false: nothing is left.
__host__ __device__ inline bool settle(const Attention &a, const Cut &cut, Range &r, Place &p)
{
    const int rest = cut.lead + p.blocks.count - p.off;
    if (p.off <= r.snap) {
        r.begin -= p.off;
        p.off = 0;
    } else if (rest <= r.snap) {
        r.begin += rest;
        if (!next_tile(a, p, cut)) return false;
    }
    return true;
}

// Whether the tile at `at` is the range's: one that goes on from the range before, one that ends in it, or one whose cut is not so near to its beginning that it moves there.
__host__ __device__ inline bool takes(const Range &r, const Place &p, long long at, const Cut &cut)
{
    return at < r.end && (p.off > 0 || r.end - at >= cut.lead + p.blocks.count || r.end - at > r.snap);
}
// On to the next tile of the range.
__host__ __device__ inline bool advance(const Attention &a, const Range &r, Place &p, long long at, const Cut &cut) { return at < r.end && next_tile(a, p, cut) && takes(r, p, at, cut); }

// What of the tile at `at` lies in a range: places of the line, and blocks of keys among them.
struct Part {
    int places, from, blocks;
    bool whole;     // all of the tile's blocks
    bool tail;      // the tile begins in this range
    int b0, b1;     // blocks of the grid that share the tile
};
__host__ __device__ inline Part part_of(const Place &p, const Range &r, long long at, const Cut &cut)
{
    Part t;
    const int all = cut.lead + p.blocks.count, rest = all - p.off;
    const long long first = at - p.off;
    t.places = r.end - at >= rest - r.snap ? rest : static_cast<int>(r.end - at);
    t.from = larger(p.off - cut.lead, 0);
    t.blocks = larger(p.off + t.places - cut.lead - t.from, 0);
    t.whole = t.blocks == p.blocks.count;
    t.tail = p.off == 0;
    t.b0 = t.whole ? 0 : static_cast<int>((first + r.snap) / r.per);              // before the first cut that stays inside the tile
    t.b1 = t.whole ? 0 : static_cast<int>((first + all - r.snap - 1) / r.per);    // behind the last one
    return t;
}

// blocks_of of 32 sequences, one per lane (count 0: none): a lane adds up a few tiles itself, many are added up by the whole warp.
__device__ inline long long blocks_of_lanes(const Attention &a, const Sequence &q, const Cut &cut, int lane)
{
    constexpr int kFew = 4;
    const int tiles = tiles_of(a, q, cut.tile_rows);
    long long n = tiles <= kFew ? blocks_of(a, q, cut) : 0;
    for (unsigned many = __ballot_sync(0xffffffffu, tiles > kFew); many; many &= many - 1) {
        const int from = __ffs(many) - 1;
        const Sequence other = {0, __shfl_sync(0xffffffffu, q.count, from), __shfl_sync(0xffffffffu, q.pos0, from)};
        long long sum = 0;
        for (int t = lane; t < tiles_of(a, other, cut.tile_rows); t += 32) sum += cut.lead + tile_blocks(a, other, t, cut.tile_rows, cut.keys).count;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == from) n = sum;
    }
    return n;
}

__device__ inline long long inclusive_sum(long long v, int lane)
{
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// The block's range of the line and the place where it begins; an empty range: nothing to do.  All threads of the block take part; a block has THREADS of them.
// Every warp adds up its share of the sequences; the one whose share holds the range's beginning finds the place.
template <int THREADS>
__device__ inline Range range_of_block(const Attention &a, const Cut &cut, Place &place)
{
    constexpr int kWarps = THREADS / 32;
    __shared__ long long sums[kWarps];
    __shared__ Place found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int share = (a.batch.sequences + kWarps - 1) / kWarps, s0 = warp * share, s1 = min(s0 + share, a.batch.sequences);
    auto of_lane = [&](int s, Sequence &q) {
        q = s < s1 ? sequence_of(a.batch, s) : Sequence{0, 0, 0};
        return blocks_of_lanes(a, q, cut, lane);
    };
    long long mine = 0;
    Sequence q;
    for (int s = s0; s < s1; s += 32) mine += of_lane(s + lane, q) * a.pages.kv_heads;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += sums[w];
        total += sums[w];
    }
    Range r = range_of(total, blockIdx.x, gridDim.x, cut);
    if (r.begin >= r.end) return r;
    if (before <= r.begin && r.begin < before + mine) {   // one warp of the block
        long long rest = r.begin - before;
        for (int s = s0; s < s1; s += 32) {
            const long long per_head = of_lane(s + lane, q), n = per_head * a.pages.kv_heads, upto = inclusive_sum(n, lane);
            const unsigned behind = __ballot_sync(0xffffffffu, rest < upto);
            if (behind == 0) {
                rest -= __shfl_sync(0xffffffffu, upto, 31);
                continue;
            }
            const int at = __ffs(behind) - 1;
            const long long head_blocks = __shfl_sync(0xffffffffu, per_head, at);
            Place p;
            p.s = s + at;
            p.q = {__shfl_sync(0xffffffffu, q.row0, at), __shfl_sync(0xffffffffu, q.count, at), __shfl_sync(0xffffffffu, q.pos0, at)};
            p.tiles = tiles_of(a, p.q, cut.tile_rows);
            rest -= __shfl_sync(0xffffffffu, upto - n, at);
            p.g = static_cast<int>(rest / head_blocks);
            rest -= p.g * head_blocks;
            for (int t = 0; t < p.tiles; t += 32) {
                const bool in = t + lane < p.tiles;
                KeyBlocks blocks = {0, 0, 0};
                if (in) blocks = tile_blocks(a, p.q, t + lane, cut.tile_rows, cut.keys);
                const int places = in ? cut.lead + blocks.count : 0;
                const long long end = inclusive_sum(places, lane);
                const unsigned past = __ballot_sync(0xffffffffu, in && rest < end);
                if (past == 0) {
                    rest -= __shfl_sync(0xffffffffu, end, 31);
                    continue;
                }
                if (lane == __ffs(past) - 1) {
                    p.tile = t + lane;
                    p.blocks = blocks;
                    p.off = static_cast<int>(rest - (end - places));
                    found = p;
                }
                break;
            }
            break;
        }
    }
    __syncthreads();
    place = found;
    if (!settle(a, cut, r, place) || !takes(r, place, r.begin, cut)) r.begin = r.end;
    return r;
}

// A part of a tile in scratch: block b of the grid has two, for a tile that began before its range and for one that goes on behind it.
struct Parts {
    float *base;              // [grid][2][floats]
    unsigned int *tickets;    // [grid]: parts arrived of the tile that begins in a block's range and goes on behind it; zero between launches
    int floats;
};

// Eight elements of a pool of a kind.
struct RawCodes8 {
    uint2 w;
    __device__ __forceinline__ void load(const uint8_t *p) { w = *reinterpret_cast<const uint2 *>(p); }
    __device__ __forceinline__ void zero() { w = make_uint2(0u, 0u); }
    __device__ __forceinline__ void get(float (&v)[8]) const { codes8(v, w, 1.0f); }
};
template <int KIND> struct Held8;
template <> struct Held8<KIND_BF16> { using Raw = Raw8<__nv_bfloat16>; using Element = __nv_bfloat16; };
template <> struct Held8<KIND_F32> { using Raw = Raw8<float>; using Element = float; };
template <> struct Held8<KIND_E4M3> { using Raw = RawCodes8; using Element = uint8_t; };

template <int KIND>
__device__ __forceinline__ void load8_held(float (&v)[8], const Pages &p, int page, int which, int head, int token, int piece)
{
    const long long at = p.place(page, which, head, token);
    if constexpr (KIND == KIND_E4M3)
        load8_codes(v, static_cast<const uint8_t *>(p.data) + at * p.dim + piece * 8, scale_of(p.scales[at]));
    else if constexpr (KIND == KIND_BF16)
        load8(v, static_cast<const __nv_bfloat16 *>(p.data) + at * p.dim + piece * 8);
    else
        load8(v, static_cast<const float *>(p.data) + at * p.dim + piece * 8);
}

// Keys `from` to `to` of a sequence's head in groups of eight, which lie side by side in a page: one per turn and half of a warp, by a team's warps in turn.  `take` gets the group's
// place in the pool (rows of keys or values; -1: the table names no page) and its first key; its page was looked up a turn before.  take: false ends it, for the whole warp.
template <typename Take>
__device__ __forceinline__ void over_groups(const Attention &a, int s, int g, int which, int from, int to, int rank, int warps, Take take)
{
    if (from > to) return;
    const int half = (threadIdx.x & 31) >> 4, mask = (1 << a.pages.page_shift) - 1;
    auto look_up = [&](int key0) { return key0 <= to && key0 + 7 >= from ? page_of(a.batch, a.pages, s, key0) : -1; };
    int key0 = (from & ~7) + 8 * (2 * rank + half), page = look_up(key0);
    for (; key0 - 8 * half <= to; key0 += 16 * warps) {   // the halves stay together: shuffles are the whole warp's
        const long long at = page >= 0 ? a.pages.place(page, which, g, key0 & mask) : -1;
        page = look_up(key0 + 16 * warps);
        if (!take(at, key0)) return;
    }
}

// One query row of one head, by a team of WARPS warps that `sync` brings together, from the definition: only keys that the row sees are read.  Sixteen lanes hold a head
// (eight elements each), so that the halves of a warp take a group of eight keys each (fp32: in two steps); a running maximum and sum per half, put together at the end, the warps'
// in `room` (kTeamRoom floats each).
constexpr int kTeamRoom = 132;
template <typename T, int KIND, int WARPS, typename Sync>
__device__ void attention_row(const Attention &a, int s, int position, int row, int head, int rank, int lane, float *room, Sync sync)
{
    constexpr int kAhead = KIND == KIND_F32 ? 4 : 8;
    using Raw = typename Held8<KIND>::Raw;
    const int piece = lane & 15, half = lane >> 4, dim = a.pages.dim, g = head / a.share;
    const bool active = piece < dim / 8;
    float q[8] = {}, acc[8] = {}, m = -INFINITY, l = 0.0f;
    if (active) load8(q, static_cast<const T *>(a.q) + row * a.q_pitch + head * dim + piece * 8);
    const auto *data = static_cast<const typename Held8<KIND>::Element *>(a.pages.data) + piece * 8;
    const long long value_rows = static_cast<long long>(a.pages.kv_heads) << a.pages.page_shift;   // from a key's row to its value's
    auto over = [&](int from, int to) {
        over_groups(a, s, g, 0, from, to, rank, WARPS, [&](long long at, int key0) {
#pragma unroll
            for (int u0 = 0; u0 < 8; u0 += kAhead) {
                Raw k[kAhead], v[kAhead];
                float k_scale[kAhead], v_scale[kAhead], x[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const int key = key0 + u0 + u;
                    const bool there = at >= 0 && key >= from && key <= to;
                    k[u].zero();
                    v[u].zero();
                    k_scale[u] = v_scale[u] = 1.0f;
                    x[u] = there ? 0.0f : -INFINITY;
                    if (there && active) {
                        k[u].load(data + (at + u0 + u) * dim);
                        v[u].load(data + (at + u0 + u + value_rows) * dim);
                        if (KIND == KIND_E4M3) {
                            k_scale[u] = scale_of(a.pages.scales[at + u0 + u]);
                            v_scale[u] = scale_of(a.pages.scales[at + u0 + u + value_rows]);
                        }
                    }
                }
                float dot[kAhead], now = m;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    float e8[8];
                    k[u].get(e8);
                    dot[u] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot[u] = fmaf(q[e], KIND == KIND_E4M3 ? e8[e] * k_scale[u] : e8[e], dot[u]);
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], o);
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) dot[u] = a.cap * tanhf(dot[u] * a.scale / a.cap);
                } else {
#pragma unroll
                    for (int u = 0; u < kAhead; ++u) dot[u] *= a.scale;
                }
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    if (x[u] == 0.0f) x[u] = dot[u];
                    now = fmaxf(now, x[u]);
                }
                const float keep = m == -INFINITY ? 0.0f : expf(m - now);
                m = now;
                l *= keep;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
                for (int u = 0; u < kAhead; ++u) {
                    const float w = x[u] == -INFINITY ? 0.0f : expf(x[u] - now);
                    float e8[8];
                    v[u].get(e8);
                    l += w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, KIND == KIND_E4M3 ? e8[e] * v_scale[u] : e8[e], acc[e]);
                }
            }
            return true;
        });
    };
    const int low = a.window ? max(0, position - a.window + 1) : 0;
    over(0, min(a.sinks, low) - 1);
    over(low, position);
    auto share_of = [](float of, float top) { return of == -INFINITY ? 1.0f : expf(of - top); };   // what saw nothing holds zeros (or NaN, which stay)
    const float both = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16)), f = share_of(m, both);
    l *= f;
    l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        acc[e] *= f;
        acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 16);
    }
    if (half == 0) {
        store8(room + rank * kTeamRoom + piece * 8, acc);
        if (piece == 0) *reinterpret_cast<float2 *>(room + rank * kTeamRoom + 128) = make_float2(both, l);
    }
    sync();
    if (rank == 0 && half == 0) {
        float top = -INFINITY, sum = 0.0f, out[8] = {};
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, room[w * kTeamRoom + 128]);
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float by = share_of(room[w * kTeamRoom + 128], top);
            float part[8];
            load8(part, room + w * kTeamRoom + piece * 8);
            sum = fmaf(room[w * kTeamRoom + 129], by, sum);
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = fmaf(part[e], by, out[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) out[e] = position >= 0 ? out[e] / sum : 0.0f;
        if (active) store8(static_cast<T *>(a.out) + row * a.out_pitch + head * dim + piece * 8, out);
        if (a.lse && piece == 0) a.lse[static_cast<long long>(row) * a.heads + head] = position >= 0 ? top + logf(sum) : -INFINITY;
    }
    sync();
}

// ---- rows whose output is not finite though the sum of their weights is
//
// Either the row sees a value that makes it so, or the tile's product multiplied one that the row does not see by zero, which is NaN, or sums against an old maximum left
// fp32's range.  In the first case the result stands: an element that is NaN where the row sees a NaN or infinities of both signs there, one that is infinite where it sees that
// infinity.  All rows of a tile see nearly the same keys, so a team of warps goes over the values that all of these rows see once, and stops as soon as every element is accounted
// for; each row then looks at the few others that it sees.  A NaN where the row sees one infinity alone becomes that infinity: every weight is positive, though the product may have
// met one that fp32 does not hold, or a negative second term.  (But without a cap a key that is not finite has weight 0, or the weights had no sum; 0 times an infinity is NaN.)  Rows with an element
// that none of this explains are formed again from their own keys alone.

constexpr uint32_t kSeenNan = 0xffu, kSeenInfinities = 0xffff00u;   // a bit per element: NaN, plus infinity, minus infinity

template <typename T>
__device__ __forceinline__ bool not_finite(const Raw8<T> &raw) { return raw.largest() >= 0x7f800000u; }
template <typename T>
__device__ __noinline__ uint32_t kinds_of(Raw8<T> raw)   // out of line: code that a tile runs through once has to be fetched each time (a prompt of 8192 with a NaN 920 us, 1010 with twice the code)
{
    uint32_t kinds = 0;
    float v[8];
    raw.get(v);
#pragma unroll
    for (int e = 0; e < 8; ++e) kinds |= (v[e] != v[e] ? 1u : v[e] > FLT_MAX ? 0x100u : v[e] < -FLT_MAX ? 0x10000u : 0u) << e;
    return kinds;
}
__device__ __forceinline__ bool not_finite(const RawCodes8 &raw) { return ((((raw.w.x & 0x7f7f7f7fu) + 0x01010101u) | ((raw.w.y & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u) != 0; }
__device__ __forceinline__ uint32_t kinds_of(RawCodes8 raw)   // the format's NaN: all bits but the sign
{
    const uint32_t x = ((raw.w.x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u, y = ((raw.w.y & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return ((x * 0x00204081u) >> 28) | (((y * 0x00204081u) >> 28) << 4);   // a word's four bits side by side
}
// Elements that are not finite for which nothing that was seen accounts.
__device__ __forceinline__ uint32_t open_kinds(uint32_t are, uint32_t seen) { return (are & ~(seen | ((seen >> 8) & (seen >> 16))) & kSeenNan) | (are & ~seen & kSeenInfinities); }

struct UnsureRows {   // in shared memory
    unsigned int rows[4], again[4];     // a bit per row; those that are formed again
    unsigned int are[16], seen[16];     // kinds by eights of dimensions: among these rows' outputs, among the values that all of them see
};

// `seen` and the kinds among the values of keys `from` to `to`, which all rows in question see, by a team's warps in turn, or as many of them as account for every element.
template <int KIND>
__device__ __noinline__ uint32_t look_through(const Attention &a, int s, int g, int from, int to, int rank, int warps, uint32_t are, uint32_t seen, unsigned int *shared)
{
    const int lane = threadIdx.x & 31, piece = lane & 15, dim = a.pages.dim;
    const bool active = piece < dim / 8;
    const auto *data = static_cast<const typename Held8<KIND>::Element *>(a.pages.data) + piece * 8;
    const long long to_key = static_cast<long long>(a.pages.kv_heads) << a.pages.page_shift;   // rows from a key's to its value's
    if (__all_sync(0xffffffffu, open_kinds(are, seen) == 0)) return seen;
    over_groups(a, s, g, 1, from, to, rank, warps, [&](long long at, int key0) {
        typename Held8<KIND>::Raw v[8];
        bool any = false;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            v[u].zero();
            if (at >= 0 && active && key0 + u >= from && key0 + u <= to) v[u].load(data + (at + u) * dim);
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) any = any || not_finite(v[u]);
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                uint32_t kinds = kinds_of(v[u]);
                if (a.cap == 0.0f && __any_sync(0xffffffffu, kinds & kSeenInfinities)) {
                    typename Held8<KIND>::Raw k;
                    k.zero();
                    if (at >= 0 && active && key0 + u >= from && key0 + u <= to) k.load(data + (at + u - to_key) * dim);
                    if ((__ballot_sync(0xffffffffu, not_finite(k)) >> (lane & 16)) & 0xffffu) kinds = (kinds | kinds >> 8 | kinds >> 16) & kSeenNan;
                }
                seen |= kinds;
            }
        }
        seen |= __shfl_xor_sync(0xffffffffu, seen, 16);
        if (shared) {
            if (lane < 16 && seen & ~*reinterpret_cast<volatile unsigned int *>(shared + piece)) atomicOr(shared + piece, seen);
            __syncwarp();
            seen |= *reinterpret_cast<volatile unsigned int *>(shared + piece);
        }
        return __all_sync(0xffffffffu, open_kinds(are, seen) == 0) == 0;
    });
    return seen;
}

// The rows of u.rows (row r: packed row packed0 + r), by a team of WARPS warps that `sync` brings together; the outputs have been stored, and u.rows is known to all.
// room: kTeamRoom floats per warp.
template <typename T, int KIND, int WARPS, typename Sync>
__device__ __noinline__ void settle_rows(const Attention &a, int s, int g, int row0, int pos0, int packed0, UnsureRows &u, int rank, float *room, Sync sync)
{
    const int lane = threadIdx.x & 31, piece = lane & 15, half = lane >> 4, dim = a.pages.dim;
    const bool active = piece < dim / 8;
    int first = 128, last = -1;
    for (int w = 0; w < 4; ++w)
        if (const unsigned int rows = u.rows[w]) {
            first = min(first, 32 * w + __ffs(rows) - 1);
            last = 32 * w + 31 - __clz(rows);
        }
    auto is_in = [&](int r) { return (u.rows[r >> 5] >> (r & 31) & 1) != 0; };
    auto token_of = [&](int r) { return a.shares.divide(packed0 + r); };
    auto head_of = [&](int r) { return g * a.share + packed0 + r - token_of(r) * a.share; };
    auto stored = [&](int r, Raw8<T> &raw) {
        raw.zero();
        if (active && r < 128 && is_in(r)) raw.load(static_cast<const T *>(a.out) + (row0 + token_of(r)) * a.out_pitch + head_of(r) * dim + piece * 8);
    };
    if (rank == 0 && half == 0) u.are[piece] = u.seen[piece] = u.again[piece & 3] = 0u;
    sync();
    uint32_t are = 0;
    for (int r = first + 2 * rank + half; r <= last; r += 16 * WARPS) {   // the same rounds for both halves or one more, without shuffles
        Raw8<T> raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) stored(r + 2 * WARPS * i, raw[i]);
#pragma unroll
        for (int i = 0; i < 8; ++i) are |= kinds_of(raw[i]);
    }
    if (are) atomicOr(u.are + piece, are);
    sync();
    const int p0 = pos0 + token_of(first), p1 = pos0 + token_of(last), low = a.window ? max(0, p1 - a.window + 1) : 0;
    are = u.are[piece];
    uint32_t seen = look_through<KIND>(a, s, g, 0, min(min(a.sinks, low) - 1, p0), rank, WARPS, are, 0, u.seen);
    look_through<KIND>(a, s, g, low, p0, rank, WARPS, are, seen, u.seen);
    sync();
    const uint32_t by_all = u.seen[piece];
    if (__all_sync(0xffffffffu, open_kinds(are, by_all) == 0)) last = -1;   // the same in all warps: what accounts for all rows' elements does so for each row's
    // by one warp; false: an element is left that nothing explains
    auto explained = [&](int r) {
        const int token = token_of(r), position = pos0 + token, from = a.window ? max(0, position - a.window + 1) : 0;
        Raw8<T> raw;
        stored(r, raw);
        are = kinds_of(raw);
        // what this row sees and the others may not: behind the first of them, in front of the last one's window
        seen = look_through<KIND>(a, s, g, max(p0 + 1, from), position, 0, 1, are, by_all, nullptr);
        seen = look_through<KIND>(a, s, g, p0 + 1, min(a.sinks, from) - 1, 0, 1, are, seen, nullptr);
        seen = look_through<KIND>(a, s, g, from, min(low - 1, p0), 0, 1, are, seen, nullptr);
        if (__all_sync(0xffffffffu, open_kinds(are, seen) == 0)) return true;
        const uint32_t open = open_kinds(are, seen), elements = open | open >> 8 | open >> 16;
        float v[8];
        raw.get(v);
#pragma unroll
        for (int e = 0; e < 8; ++e)   // not both: that accounts for a NaN, and an infinity has not met the other one
            if (elements >> e & 1 && seen >> e & 0x10100u) v[e] = seen >> e & 0x100u ? INFINITY : -INFINITY;
        if (active && half == 0) store8(static_cast<T *>(a.out) + (row0 + token) * a.out_pitch + head_of(r) * dim + piece * 8, v);
        return __all_sync(0xffffffffu, (elements & ~(seen >> 8 | seen >> 16) & kSeenNan) == 0) != 0;
    };
    for (int r = first, n = 0; r <= last; ++r)
        if (is_in(r) && n++ % WARPS == rank && !explained(r) && lane == 0) atomicOr(u.again + (r >> 5), 1u << (r & 31));
    sync();
    for (int w = 0; w < 4; ++w)
        for (unsigned int rest = u.again[w]; rest; rest &= rest - 1) {
            const int r = 32 * w + __ffs(rest) - 1, token = token_of(r);
            attention_row<T, KIND, WARPS>(a, s, pos0 + token, row0 + token, head_of(r), rank, lane, room, sync);
            if (rank == 0) explained(r);   // its sums may have met infinities, too
        }
    sync();   // what the next tile writes has been read
}

}  // namespace kvp
}  // namespace gptb200
