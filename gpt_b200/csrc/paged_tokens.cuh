// Attention of a few new rows per sequence (single tokens above all) over a paged cache, in bf16.
//
// A tile is eight (NT = 1) or sixteen packed query rows of one sequence and key / value head (kv_pages.cuh: the line of work).  Each warp of a block takes sixteen
// keys of every block of 64 in turn: asynchronous copies bring them, and their values, into a ring of its own; scores and weighted values are mma.sync products of
// 16 x 8 x 16 with keys, then dimensions, as their rows and the tile's rows as columns: a group of up to eight query heads fills them, where rows of the tile as rows
// of the product would leave half of it empty and hold twice the accumulators.  Maximum and sum run along in fp32.  The warps meet once per tile.
//
// Bound by the cache's bytes: 8 query rows against 4 * dim bytes of a bf16 key and value are 8 flops a byte, a twentieth of what mma.sync sustains, so the legacy
// instructions do here; what counts is bytes in flight and instructions per byte, hence the rings (40 to 100 KB per block) and no barrier inside the loop.
//
// Codes (e4m3) go through registers once, to fp16, which holds every code exactly; their powers of two never touch the products:
//   scores   q of a row is brought to [2^15, 2^16) at its largest by a power of two, so that fp16 holds all eight bits of a bf16 element down to 2^-32 of the largest
//            (and part of them down to 2^-40); the row's and the key's powers multiply the score
//   values   weight j enters the second product as 2^(x_j + e_j - R + 11), x_j the score in base 2, e_j the value's exponent, R their running maximum within 2^4: at most
//            2^15.  The sum of weights runs against the scores' own maximum, in fp32.
// Weights enter the products in two terms, so that their rounding stays below that of an fp32 sum's order: sixteen bits of bf16, which has fp32's exponents, or
// twenty-two of fp16, whose second term ends at 2^-35 of the row's largest: what a key adds is off by 2^-22 of itself and 2^-36 of the largest weight times power.
// The products' inner dimension may be permuted on both sides, and so may the output's columns: a lane takes neighbouring codes with one load, pairs two keys'
// codes with a byte permutation, and no transposition is needed.
#pragma once

#include <cuda_fp16.h>

#include "kv_pages.cuh"

namespace gptb200 {
namespace kvp {

constexpr int kTokensWarps = 4, kTokensThreads = kTokensWarps * 32;
constexpr int kTokensMaxRows = 16, kTokensKeys = 64;
constexpr int kTokensPart = kTokensMaxRows * 128 + 2 * kTokensMaxRows;   // floats of a part in scratch

__host__ __device__ constexpr int tokens_per_sm(bool codes) { return codes ? 3 : 2; }              // blocks on an SM
__host__ __device__ constexpr int tokens_blocks(bool codes) { return tokens_per_sm(codes) * 160; }   // of a grid, at most: so many parts' sums have room in shared memory

// D16: dimensions in steps of 16 (zeros behind the head's own)
template <int D16, bool CODES, int NT>
struct TokensShape {
    static constexpr int kDim = 16 * D16, kBytes = CODES ? 1 : 2;
    // copies: pieces of sixteen bytes per row (a power of two), rows that a warp takes in one turn, turns for sixteen rows
    static constexpr int kPieces = CODES ? (D16 > 4 ? 8 : D16) : (D16 > 4 ? 16 : 2 * D16), kRowsPerTurn = 32 / kPieces, kTurns = 16 / kRowsPerTurn;
    // pitches that spread what the lanes of one load touch over all banks
    static constexpr int kKeyPitch = CODES ? (D16 == 8 ? 144 : 16 * D16) : 2 * kDim + 16;
    static constexpr int kValuePitch = CODES ? (D16 == 8 ? 144 : D16 == 6 ? 112 : D16 == 4 ? 80 : 48) : 2 * kDim + 16;
    static constexpr int kStage = 16 * (kKeyPitch + kValuePitch) + (CODES ? 32 : 0);
    static constexpr int kStages = NT == 1 && !CODES ? 2 : 3;
    static constexpr int kRows = 8 * NT;
    static constexpr int kQPitch = 2 * kDim + 16;
    static constexpr int kRing = kTokensWarps * kStages * kStage;
    static constexpr int kMergePitch = kDim + 4;
    static constexpr int kMerge = kTokensWarps * kRows * kMergePitch * 4;
    static constexpr int kSmem = kRows * kQPitch + (kRing > kMerge ? kRing : kMerge);
    static_assert((kSmem - kRows * kQPitch) / 8 >= tokens_blocks(CODES) && kSmem - kRows * kQPitch >= kTokensWarps * kTeamRoom * 4);   // of the grid: a tile's parts, at most
};

namespace tok {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Factor that brings what stands against maximum m to maximum `top`.  A part that saw nothing holds zeros (or NaN, which stay) and counts as it is.
__device__ __forceinline__ float share_of(float m, float top) { return m == -INFINITY ? 1.0f : exp2_fast(m - top); }
template <int BYTES>
__device__ __forceinline__ void copy(uint32_t dst, const void *from)
{
    static_assert(BYTES == 16);
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
}
// zeros where `from` is not to be read
template <int BYTES>
__device__ __forceinline__ void copy_or_zero(uint32_t dst, const void *from, bool there)
{
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(there ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(from), "n"(BYTES), "r"(there ? BYTES : 0) : "memory");
}
__device__ __forceinline__ const uint8_t *shared_pointer(const uint8_t *p, int from)
{
    return reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), from));
}
__device__ __forceinline__ unsigned long long pair(float a, float b)
{
    unsigned long long v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpair(unsigned long long v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
// tanh of two values within [-1, 1]: x times a polynomial in x^2, the Chebyshev fit of degree 7 of tanh(x) / x (largest error 5e-9, with fp32 rounding 7e-8)
__device__ __forceinline__ unsigned long long tanh_inner2(unsigned long long x)
{
    constexpr float c[8] = {1.0f, -0.33333307504653931f, 0.13332527875900269f, -0.053887963294982910f, 0.021501919254660606f, -0.0079579148441553116f, 0.0023032133467495441f,
                            -0.00035729847149923444f};
    const unsigned long long u = ptx::mul2(x, x);
    unsigned long long p = ptx::both(c[7]);
#pragma unroll
    for (int i = 6; i >= 0; --i) p = ptx::fma2(p, u, ptx::both(c[i]));
    return ptx::mul2(p, x);
}
// four codes as two pairs of halves
__device__ __forceinline__ void halves(uint32_t four, uint32_t &first, uint32_t &second)
{
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}" : "=r"(first), "=r"(second) : "r"(four));
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b)
{
    uint32_t h;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(b), "f"(a));
    return h;
}
__device__ __forceinline__ float2 unpack_half2(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
// an 8 x 8 matrix of sixteen-bit values, a row per four lanes, transposed
__device__ __forceinline__ uint32_t transposed(uint32_t v)
{
    uint32_t t;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
    return t;
}
template <int WORDS>
__device__ __forceinline__ void lds_words(uint32_t (&v)[WORDS], uint32_t addr)
{
    static_assert(WORDS == 1 || WORDS == 2 || WORDS == 3 || WORDS == 4);
    if constexpr (WORDS == 4)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr));
    else if constexpr (WORDS == 2)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr));
    else
#pragma unroll
        for (int i = 0; i < WORDS; ++i) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[i]) : "r"(addr + 4 * i));
}

}  // namespace tok

struct TokensArgs {
    Attention a;
    Parts parts;
    Cut cut;
};

struct BlockSync {
    __device__ __forceinline__ void operator()() const { __syncthreads(); }
};

// The end of a tile, for a block of kTokensThreads threads that holds its rows' sums in shared memory: merge [SUMS][ROWS][pitch] weighted values (added up here) against
// total_ml [ROWS] = (maximum in base 2, sum).  A whole tile is stored; else the part goes to scratch, and the block that arrives last puts the parts together.
// sums: room for as many pairs, one per block of the grid and kTeamRoom / 2 per warp at least; it may be `merge` itself.  unsure.rows is zero on entry.
template <typename T, int KIND, int ROWS, int SUMS>
__device__ __forceinline__ void finish_tile(const Attention &a, const Parts &parts, const Place &place, const Part &part, int rows, const float *merge, int pitch,
                                            float (*total_ml)[2], float2 *sums, int room, UnsureRows &unsure, int *arrived_last)
{
    constexpr int kSlot = (ROWS > kTokensMaxRows ? ROWS : kTokensMaxRows) * 128;   // a part in scratch: values, then maxima and sums
    constexpr float kLn2 = 0.69314718055994531f;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, dim = a.pages.dim, pieces = dim / 8, packed0 = place.tile * ROWS;
    auto finish = [&](int r, int c, float (&v)[8], float top, float sum) {   // piece c of row r
        const int packed = packed0 + r, token = a.shares.divide(packed), row = place.q.row0 + token, head = place.g * a.share + packed - token * a.share;
        const bool sees = place.q.pos0 + token >= 0;   // itself at least
        const float inv = sees ? 1.0f / sum : 0.0f;
        bool fine = true;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] *= inv;
            fine = fine && fabsf(v[e]) <= FLT_MAX;
        }
        if (!fine && sum > 0.0f && sum <= FLT_MAX) atomicOr(unsure.rows, 1u << r);   // with any other sum the row is NaN by definition
        store8(static_cast<T *>(a.out) + row * a.out_pitch + head * dim + c * 8, v);
        if (a.lse && c == 0) a.lse[static_cast<long long>(row) * a.heads + head] = sees ? top * kLn2 + logf(sum) : -INFINITY;
    };
    float *own = parts.base + (2LL * blockIdx.x + part.tail) * parts.floats;
    for (int i = threadIdx.x; i < rows * pieces; i += kTokensThreads) {
        const int r = i / pieces, c = i % pieces;
        float v[8] = {};
#pragma unroll
        for (int w = 0; w < SUMS; ++w) {
            float u[8];
            load8(u, merge + (w * ROWS + r) * pitch + c * 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += u[e];
        }
        if (part.whole) {
            finish(r, c, v, total_ml[r][0], total_ml[r][1]);
        } else {
            store8(own + r * dim + c * 8, v);
            if (c == 0) *reinterpret_cast<float2 *>(own + kSlot + 2 * r) = make_float2(total_ml[r][0], total_ml[r][1]);
        }
    }
    if (!part.whole) {
        const int b0 = part.b0, b1 = part.b1, count = b1 - b0 + 1;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            const unsigned int before = atomicAdd(parts.tickets + b0, 1u);
            *arrived_last = before == static_cast<unsigned int>(b1 - b0);
            if (*arrived_last) parts.tickets[b0] = 0u;
            __threadfence();
        }
        __syncthreads();
        if (*arrived_last) {
            // the parts' maxima and sums first, all of them under way at once; a part's factor takes the place of its maximum
            auto slot = [&](int b) { return parts.base + (2LL * b + (b == b0)) * parts.floats; };
            const int most = min(rows, room / count);   // rows at a time
            for (int r0 = 0; r0 < rows; r0 += most) {
                const int n_rows = min(most, rows - r0);
                __syncthreads();
                for (int i = threadIdx.x; i < count * n_rows; i += kTokensThreads) sums[i] = __ldcg(reinterpret_cast<const float2 *>(slot(b0 + i / n_rows) + kSlot + 2 * (r0 + i % n_rows)));
                __syncthreads();
                for (int r = warp; r < n_rows; r += kTokensWarps) {
                    float top = -INFINITY, sum = 0.0f;
                    for (int i = lane; i < count; i += 32) top = fmaxf(top, sums[i * n_rows + r].x);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    for (int i = lane; i < count; i += 32) {
                        float2 &v = sums[i * n_rows + r];
                        v.x = tok::share_of(v.x, top);
                        sum = fmaf(v.y, v.x, sum);
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                    if (lane == 0) {
                        total_ml[r0 + r][0] = top;
                        total_ml[r0 + r][1] = sum;
                    }
                }
                __syncthreads();
                for (int i = threadIdx.x; i < n_rows * pieces; i += kTokensThreads) {
                    const int r = i / pieces, c = i % pieces;
                    float v[8] = {};
#pragma unroll 8
                    for (int n = 0; n < count; ++n) {
                        const float *from = slot(b0 + n) + (r0 + r) * dim + c * 8;
                        const float4 u0 = __ldcg(reinterpret_cast<const float4 *>(from)), u1 = __ldcg(reinterpret_cast<const float4 *>(from + 4));
                        const float f = sums[n * n_rows + r].x;
                        v[0] = fmaf(u0.x, f, v[0]); v[1] = fmaf(u0.y, f, v[1]); v[2] = fmaf(u0.z, f, v[2]); v[3] = fmaf(u0.w, f, v[3]);
                        v[4] = fmaf(u1.x, f, v[4]); v[5] = fmaf(u1.y, f, v[5]); v[6] = fmaf(u1.z, f, v[6]); v[7] = fmaf(u1.w, f, v[7]);
                    }
                    finish(r0 + r, c, v, total_ml[r0 + r][0], total_ml[r0 + r][1]);
                }
            }
        }
    }
    __syncthreads();
    if (__builtin_expect(unsure.rows[0] != 0u, 0)) settle_rows<T, KIND, kTokensWarps>(a, place.s, place.g, place.q.row0, place.q.pos0, packed0, unsure, warp, reinterpret_cast<float *>(sums), BlockSync());
    __syncthreads();   // what the next tile writes again has been read
}

template <int D16, bool CODES, int NT>
__global__ void __launch_bounds__(kTokensThreads, tokens_per_sm(CODES))
paged_tokens_kernel(const __grid_constant__ TokensArgs args)
{
    using namespace tok;
    using S = TokensShape<D16, CODES, NT>;
    constexpr int kRows = S::kRows;
    constexpr float kGrowth = CODES ? 4.0f : 32.0f;   // of a row's maximum, base 2, before what has been added up is scaled
    constexpr float kLift = CODES ? 11.0f : 0.0f;     // fp16 weights end at 2^16: the largest is 2^(kLift + kGrowth)
    constexpr int kind = CODES ? KIND_E4M3 : KIND_BF16;
    constexpr float kLog2e = 1.4426950408889634f;
    extern __shared__ __align__(16) uint8_t tokens_smem[];
    __shared__ float merge_ml[kTokensWarps][kRows][2], total_ml[kRows][2], row_power[kRows];
    __shared__ UnsureRows unsure;
    __shared__ int arrived_last;
    const Attention &a = args.a;
    grid_dependency_wait();
    grid_dependency_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    Place place;
    Range range = range_of_block<kTokensThreads>(a, args.cut, place);
    const uint32_t q_tile = ptx::smem_u32(tokens_smem), ring = q_tile + kRows * S::kQPitch + warp * S::kStages * S::kStage;
    const int dim = a.pages.dim, pieces = dim / 8, mask = (1 << a.pages.page_shift) - 1;
    // sixteen-byte pieces of a row per lane; where codes' rows begin at odd multiples of eight they are copied by eights
    const uint8_t *data = static_cast<const uint8_t *>(a.pages.data);
    const int row_bytes = dim * S::kBytes;
    const bool wide = row_bytes % 16 == 0;
    const long long head_bytes = static_cast<long long>(row_bytes) << a.pages.page_shift, value_bytes = head_bytes * a.pages.kv_heads, page_bytes = 2 * value_bytes;
    const int lane_row = lane / S::kPieces, lane_piece = lane % S::kPieces, lane_from = lane_row * row_bytes + lane_piece * 16;
    const bool lane_on = lane_piece * 16 < row_bytes;
    const uint32_t key_to = lane_row * S::kKeyPitch + lane_piece * 16, value_to = 16 * S::kKeyPitch + lane_row * S::kValuePitch + lane_piece * 16;
    // a head narrower than the padded width: its tail columns stay zero
    auto clear_tail = [&] {
        if (dim == S::kDim) return;
        for (int i = lane; i < S::kStages * S::kStage / 16; i += 32) ptx::sts128(ring + 16 * i, 0u, 0u, 0u, 0u);
        __syncwarp();
    };

    for (long long at = range.begin; at < range.end;) {
        const Part part = part_of(place, range, at, args.cut);
        at += part.places;
        const int n_blocks = part.blocks;
        const int packed0 = place.tile * kRows, rows = min(kRows, place.q.count * a.share - packed0);
        const int p0 = place.q.pos0 + a.shares.divide(packed0), p1 = place.q.pos0 + a.shares.divide(packed0 + rows - 1);
        const int low = a.window ? p0 - a.window + 1 : 0;   // keys below it are visible only among the first ones
        auto tile_key = [&](int i) { return block_key(place.blocks, part.from + i, kTokensKeys) + warp * 16; };
        auto wanted = [&](int key) { return key <= p1 && (key >= low || key < a.sinks); };   // by any row of the tile

        // ---- the ring
        // lanes with an even number look up where the tile's first eight keys lie, the others the last eight: those of a page's head lie one behind the other
        int next_entry = -1;
        bool next_wanted = false;
        auto look_up = [&](int i) {   // the table's entry is not looked at before the tile is fetched, a turn later
            const int key = tile_key(i) + 8 * (lane & 1);
            next_wanted = i < n_blocks && key <= p1 && (key + 7 >= low || key < a.sinks);
            if (next_wanted) next_entry = a.batch.table[static_cast<long long>(place.s) * a.batch.table_pitch + (key >> a.pages.page_shift)];
        };
        look_up(0);
        auto fetch = [&](int i) {
            const int stage = i % S::kStages;
            const uint32_t dst = ring + stage * S::kStage;
            const bool there = next_wanted && next_entry >= 0 && next_entry < a.pages.num_pages;
            if (next_wanted && !there) report_bad(a.batch.status);
            const int my_page = there ? next_entry : -1;
            const uint8_t *my_rows = data + max(my_page, 0) * page_bytes + place.g * head_bytes + ((tile_key(i) + 8 * (lane & 1)) & mask) * row_bytes;
            const int page[2] = {__shfl_sync(0xffffffffu, my_page, 0), __shfl_sync(0xffffffffu, my_page, 1)};
            const uint8_t *rows8[2] = {shared_pointer(my_rows, 0), shared_pointer(my_rows, 1)};
            look_up(i + 1);
            if (i < n_blocks) {
                const int t = tile_key(i);
                if (page[0] >= 0 && page[1] >= 0 && t + 15 <= p1 && (t >= low || t + 16 <= a.sinks) && wide) {   // every key is wanted
#pragma unroll
                    for (int j = 0; j < S::kTurns; ++j) {
                        const int first = j * S::kRowsPerTurn;
                        const uint8_t *from = S::kRowsPerTurn == 16 ? (lane_row >= 8 ? rows8[1] - 8 * row_bytes : rows8[0]) : rows8[first >> 3] + (first & 7) * row_bytes;
                        if (lane_on) {
                            copy<16>(dst + first * S::kKeyPitch + key_to, from + lane_from);
                            copy<16>(dst + first * S::kValuePitch + value_to, from + lane_from + value_bytes);
                        }
                    }
                } else {
                    const int step = wide ? 16 : 8, chunks = row_bytes / step;
                    for (int idx = lane; idx < 16 * chunks; idx += 32) {
                        const int r = idx / chunks, c = idx % chunks;
                        const bool on = page[r >> 3] >= 0 && wanted(t + r);
                        const uint8_t *from = on ? rows8[r >> 3] + (r & 7) * row_bytes + c * step : data;
                        const uint32_t key_at = dst + r * S::kKeyPitch + c * step, value_at = dst + 16 * S::kKeyPitch + r * S::kValuePitch + c * step;
                        if (wide) {
                            copy_or_zero<16>(key_at, from, on);
                            copy_or_zero<16>(value_at, on ? from + value_bytes : data, on);
                        } else {
                            copy_or_zero<8>(key_at, from, on);
                            copy_or_zero<8>(value_at, on ? from + value_bytes : data, on);
                        }
                    }
                }
                if (CODES && lane < 4) {   // powers of two: eight keys a copy, keys' then values'
                    const int half = lane & 1, which = lane >> 1, pg = page[half];
                    const uint8_t *src = pg >= 0 ? a.pages.scales + a.pages.place(pg, which, place.g, (t + 8 * half) & mask) : a.pages.scales;
                    copy_or_zero<8>(dst + 16 * (S::kKeyPitch + S::kValuePitch) + 16 * which + 8 * half, src, pg >= 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        clear_tail();
#pragma unroll
        for (int i = 0; i < S::kStages - 1; ++i) fetch(i);

        // ---- the queries: a row's eight dimensions per lane, sixteen lanes a row
        for (int r = threadIdx.x >> 4; r < kRows; r += kTokensThreads / 16) {
            const int c = threadIdx.x & 15;
            float v[8] = {};
            if (r < rows && c < pieces) {
                const int packed = packed0 + r, row = place.q.row0 + a.shares.divide(packed), head = place.g * a.share + packed - a.shares.divide(packed) * a.share;
                load8(v, static_cast<const __nv_bfloat16 *>(a.q) + row * a.q_pitch + head * dim + c * 8);
            }
            uint32_t w[4];
            if constexpr (CODES) {
                float most = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(v[e]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
                const int e2 = max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -111) - 15;   // infinite or zero: whatever, the row stays so
                const float by = power_of_two(-e2);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = pack_half2(v[2 * i] * by, v[2 * i + 1] * by);
                if (c == 0) row_power[r] = power_of_two(e2);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = ptx::pack_bf16x2(v[2 * i], v[2 * i + 1]);
            }
            if (c < 2 * D16) ptx::sts128(q_tile + r * S::kQPitch + c * 16, w[0], w[1], w[2], w[3]);
        }
        if (threadIdx.x < 4) unsure.rows[threadIdx.x] = 0u;
        __syncthreads();
        // queries as B operands: columns are rows of the tile
        uint32_t qf[NT][D16][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int k = 0; k < D16; ++k) {
                if constexpr (CODES) {
                    lds_words<2>(qf[n][k], q_tile + (8 * n + g8) * S::kQPitch + (t4 * 4 * D16 + 4 * k) * 2);
                } else {
                    lds_words<1>(reinterpret_cast<uint32_t(&)[1]>(qf[n][k][0]), q_tile + (8 * n + g8) * S::kQPitch + (16 * k + 2 * t4) * 2);
                    lds_words<1>(reinterpret_cast<uint32_t(&)[1]>(qf[n][k][1]), q_tile + (8 * n + g8) * S::kQPitch + (16 * k + 2 * t4 + 8) * 2);
                }
            }
        // a lane's rows: 2 t4 and 2 t4 + 1 of every eight
        int pos[NT][2];
        float small[NT][2], to_score[NT][2], m[NT][2], ref[NT][2], l[NT][2] = {};   // m: what the sums stand against, ref: what the weighted values stand against (codes; else m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * t4 + e;
                pos[n][e] = r < rows ? place.q.pos0 + a.shares.divide(packed0 + r) : -1;
                const float power = CODES ? row_power[r] : 1.0f;
                small[n][e] = fminf(power, 1.0f);
                to_score[n][e] = (a.cap > 0.0f ? a.scale / a.cap : a.scale * kLog2e) * fmaxf(power, 1.0f);   // over the cap, or in base 2
                m[n][e] = ref[n][e] = -INFINITY;
            }
        const float cap_log2 = a.cap * kLog2e;
        float O[NT][D16][4] = {};
        for (int it = 0; it < n_blocks; ++it) {
            fetch(it + S::kStages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(S::kStages - 1) : "memory");
            __syncwarp();
            const int t = tile_key(it);
            const uint32_t kt = ring + it % S::kStages * S::kStage, vt = kt + 16 * S::kKeyPitch, et = vt + 16 * S::kValuePitch;
            // scores: rows of the product are keys g8 and g8 + 8, columns rows of the tile
            float x[NT][4] = {}, x2[NT][4] = {};   // two sums: a product waits for the one before it in its sum
            float value_e[2] = {};   // exponents of the two keys' values
            if constexpr (CODES) {
                constexpr int kWords = D16 % 4 == 0 ? 4 : 2;
#pragma unroll
                for (int k = 0; k < D16; k += kWords) {
                    uint32_t u[kWords], v[kWords];
                    lds_words<kWords>(u, kt + g8 * S::kKeyPitch + t4 * 4 * D16 + 4 * k);
                    lds_words<kWords>(v, kt + (g8 + 8) * S::kKeyPitch + t4 * 4 * D16 + 4 * k);
#pragma unroll
                    for (int i = 0; i < kWords; ++i) {
                        uint32_t f[4];
                        halves(u[i], f[0], f[2]);
                        halves(v[i], f[1], f[3]);
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma<true>(i & 1 ? x2[n] : x[n], f, qf[n][k + i][0], qf[n][k + i][1]);
                    }
                }
                uint32_t ke[2], ve[2];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(ke[j]) : "r"(et + g8 + 8 * j));
                    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(ve[j]) : "r"(et + 16 + g8 + 8 * j));
                    value_e[j] = static_cast<float>(static_cast<int>(ve[j]) - 127);
#pragma unroll
                    for (int n = 0; n < NT; ++n)   // a small row's power in front of the key's, a large one's behind it: what lies between stays within fp32 where the score does
#pragma unroll
                        for (int e = 0; e < 2; ++e) x[n][2 * j + e] = (x[n][2 * j + e] + x2[n][2 * j + e]) * small[n][e] * scale_of(ke[j]) * to_score[n][e];
                }
            } else {
#pragma unroll
                for (int k = 0; k < D16; ++k) {
                    uint32_t f[4];
                    ldsm4(f, kt + (lane & 15) * S::kKeyPitch + (k * 16 + ((lane >> 4) << 3)) * 2);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma<false>(k & 1 ? x2[n] : x[n], f, qf[n][k][0], qf[n][k][1]);
                }
            }
            const bool all_seen = t + 15 <= p0 && (a.window == 0 || t > p1 - a.window || t + 15 < a.sinks) && p0 >= 0;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (!CODES) x[n][i] = (x[n][i] + x2[n][i]) * to_score[n][i & 1];
                if (a.cap > 0.0f) {   // a polynomial where all of the warp's scores lie within the cap
                    if (__all_sync(0xffffffffu, fmaxf(fmaxf(fabsf(x[n][0]), fabsf(x[n][1])), fmaxf(fabsf(x[n][2]), fabsf(x[n][3]))) <= 1.0f)) {
                        unpair(tanh_inner2(pair(x[n][0], x[n][1])), x[n][0], x[n][1]);
                        unpair(tanh_inner2(pair(x[n][2], x[n][3])), x[n][2], x[n][3]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[n][i] = tanhf(x[n][i]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[n][i] *= cap_log2;
                }
            }
            if (!all_seen) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (!visible(a, t + g8 + 8 * (i >> 1), pos[n][i & 1])) x[n][i] = -INFINITY;
            }
            // A row's maximum only has to be near: as long as no score is far beyond it, nothing is exchanged between the lanes.
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float top = fmaxf(x[n][e], x[n][2 + e]);
                    grow = grow || top > m[n][e] + kGrowth || (m[n][e] == -INFINITY && top > -INFINITY);
                    if (CODES) grow = grow || fmaxf(x[n][e] + value_e[0], x[n][2 + e] + value_e[1]) > ref[n][e] + kGrowth;
                }
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(x[n][e], x[n][2 + e]), top_ref = CODES ? fmaxf(x[n][e] + value_e[0], x[n][2 + e] + value_e[1]) : 0.0f;
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) {
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                            if (CODES) top_ref = fmaxf(top_ref, __shfl_xor_sync(0xffffffffu, top_ref, o));
                        }
                        const float now = fmaxf(m[n][e], top), now_ref = CODES ? fmaxf(ref[n][e], top_ref) : now;
                        const float f = now == -INFINITY ? 1.0f : exp2_fast(m[n][e] - now), f_ref = now_ref == -INFINITY ? 1.0f : exp2_fast(ref[n][e] - now_ref);
                        l[n][e] *= f;
                        m[n][e] = now;
                        ref[n][e] = now_ref;
#pragma unroll
                        for (int u = 0; u < D16; ++u) {
                            O[n][u][e] *= f_ref;
                            O[n][u][2 + e] *= f_ref;
                        }
                    }
            }
            // weights: from rows of keys to the B operand's columns of rows of the tile by one transposition of 8 x 8 each
            uint32_t weights[NT][2], weights_rest[NT][2];   // two terms each
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = i & 1;
                    const float against = m[n][e] == -INFINITY ? 0.0f : m[n][e];   // nothing seen yet: every weight is 2^-inf = 0
                    const float p = exp2_fast(x[n][i] - against);
                    l[n][e] += p;
                    w[i] = CODES ? exp2_fast(x[n][i] + value_e[i >> 1] - (ref[n][e] == -INFINITY ? 0.0f : ref[n][e] - kLift)) : p;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if constexpr (CODES) {
                        const uint32_t first = pack_half2(w[2 * j], w[2 * j + 1]);
                        const float2 held = unpack_half2(first);
                        weights[n][j] = transposed(first);
                        weights_rest[n][j] = transposed(pack_half2(w[2 * j] - held.x, w[2 * j + 1] - held.y));
                    } else {
                        const uint32_t first = ptx::pack_bf16x2(w[2 * j], w[2 * j + 1]);
                        weights[n][j] = transposed(first);
                        weights_rest[n][j] = transposed(ptx::pack_bf16x2(w[2 * j] - bf16_low(first), w[2 * j + 1] - bf16_high(first)));
                    }
                }
            }
            if constexpr (CODES) {
                // dimensions g8 * 2 D16 + ... of keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9: the product's rows g8 and g8 + 8 of step u are dimensions 2 u and 2 u + 1 among them
                constexpr int kWords = D16 / 2;
                uint32_t c[4][kWords];
#pragma unroll
                for (int r = 0; r < 4; ++r) lds_words<kWords>(c[r], vt + (2 * t4 + (r & 1) + 8 * (r >> 1)) * S::kValuePitch + g8 * 2 * D16);
#pragma unroll
                for (int i = 0; i < kWords; ++i) {
                    uint32_t f0[4], f1[4];
                    halves(__byte_perm(c[0][i], c[1][i], 0x5140), f0[0], f0[1]);
                    halves(__byte_perm(c[2][i], c[3][i], 0x5140), f0[2], f0[3]);
                    halves(__byte_perm(c[0][i], c[1][i], 0x7362), f1[0], f1[1]);
                    halves(__byte_perm(c[2][i], c[3][i], 0x7362), f1[2], f1[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma<true>(O[n][2 * i], f0, weights[n][0], weights[n][1]);
                        mma<true>(O[n][2 * i + 1], f1, weights[n][0], weights[n][1]);
                        mma<true>(O[n][2 * i], f0, weights_rest[n][0], weights_rest[n][1]);
                        mma<true>(O[n][2 * i + 1], f1, weights_rest[n][0], weights_rest[n][1]);
                    }
                }
            } else {
#pragma unroll
                for (int u = 0; u < D16; ++u) {
                    uint32_t f[4];
                    ldsm4t(f, vt + ((lane & 7) + ((lane >> 4) << 3)) * S::kValuePitch + (16 * u + (((lane >> 3) & 1) << 3)) * 2);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma<false>(O[n][u], f, weights[n][0], weights[n][1]);
                        mma<false>(O[n][u], f, weights_rest[n][0], weights_rest[n][1]);
                    }
                }
            }
            __syncwarp();   // this stage may be filled again
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // ---- the warps' parts
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], o);
                if (g8 == 0) {
                    merge_ml[warp][8 * n + 2 * t4 + e][0] = m[n][e];
                    merge_ml[warp][8 * n + 2 * t4 + e][1] = l[n][e];
                }
            }
        __syncthreads();   // every warp is done with its ring: the sums take its place
        float *merge = reinterpret_cast<float *>(tokens_smem + kRows * S::kQPitch);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = 8 * n + 2 * t4 + e;
                float top = merge_ml[0][r][0];
#pragma unroll
                for (int w = 1; w < kTokensWarps; ++w) top = fmaxf(top, merge_ml[w][r][0]);
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kTokensWarps; ++w) sum += merge_ml[w][r][1] * share_of(merge_ml[w][r][0], top);
                if (warp == 0 && g8 == 0) {
                    total_ml[r][0] = top;
                    total_ml[r][1] = sum;
                }
                const float f = share_of(CODES ? ref[n][e] - kLift : m[n][e], top);
                float *to = merge + (warp * kRows + r) * S::kMergePitch;
#pragma unroll
                for (int u = 0; u < D16; ++u) {
                    to[CODES ? g8 * 2 * D16 + 2 * u : 16 * u + g8] = O[n][u][e] * f;
                    to[CODES ? g8 * 2 * D16 + 2 * u + 1 : 16 * u + g8 + 8] = O[n][u][2 + e] * f;
                }
            }
        __syncthreads();
        finish_tile<__nv_bfloat16, kind, kRows, kTokensWarps>(a, args.parts, place, part, rows, merge, S::kMergePitch, total_ml, reinterpret_cast<float2 *>(merge), (S::kSmem - kRows * S::kQPitch) / 8, unsure, &arrived_last);
        if (!advance(a, range, place, at, args.cut)) break;
    }
}

}  // namespace kvp
}  // namespace gptb200
