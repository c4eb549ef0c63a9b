// Attention of prompts and portions of prompts over a paged cache on the tensor cores, in bf16.
//
// A tile is 256 packed query rows of one sequence and key / value head (kv_pages.cuh: the line of work), worked on as two halves of 128; per block of 128 keys
//   S = Q K^T   tcgen05.mma from shared memory, S in TMEM
//   softmax     a thread per row: the row's scores in registers, running reference and sum in fp32; weights go back to TMEM over S, rounded to bf16 (the output has
//               no more bits) and divided at the end by the sum of the rounded ones: what rounding does to all of them alike cancels, and where a few weights
//               make up a row so does the rest (error of such rows 1.65 -> 1.05 times that of rounding the output alone; two terms per weight, which would do
//               the same for all rows, cost 25 %).  SUMS: the logarithm of the sum is asked for, which takes the unrounded sum besides
//   O += P V    tcgen05.mma with P from TMEM and V from shared memory as stored (MN-major)
// The halves take turns on the tensor pipe: while one is in softmax the other's products run.  O is scaled only when a row's maximum has grown by more than
// 2^32 since the last time: weights of bf16 have fp32's exponents, so that neither they nor their sums leave the range before (with a limit of 2^8 a third of the blocks
// of a prompt with uneven keys paid 1 200 cycles for it).  The grid is one block per SM, each with an equal range of the line; queries of the next tile are fetched while the last one is stored.
//
//   warps 0-1, 2-3   keys, values (named barriers 2 and 3): pages are looked up per key, rows come by asynchronous 16-byte copies into the swizzled layout that the tensor core reads (a
//                    page is as small as eight tokens; an e4m3 row goes through registers and becomes bf16 there, exactly); all four fetch queries
//   warp 4           issues the products, one elected lane
//   warp 5           walks along the line and hands the others each tile's part of the range through a ring in shared memory
//   warps 8-11       softmax and output of half 0;  warps 12-15: half 1
// Keys and values that no row of the tile sees are zeros in shared memory, whatever the pages hold there.  Every wait is bounded; its time stands still while a half looks at rows
// that are not finite (settle_rows), which ends by itself.
#pragma once

#include "paged_tokens.cuh"

namespace gptb200 {
namespace kvp {

constexpr int kPromptThreads = 512, kPromptRows = 256, kPromptKeys = 128;
constexpr int kPromptBlock = 128 * 128;   // bytes of [128 rows x 64 bf16]
constexpr int kPromptMaxStages = 3;
constexpr int kPromptPart = kPromptRows * 128 + 4 * kPromptRows;   // floats of a part in scratch

template <int NB>   // 64-column blocks of a head
struct PromptShape {
    static constexpr int kStages = NB == 1 ? 3 : 2;
    static constexpr int kTile = NB * kPromptBlock;
    static constexpr int kStaging = 8 * 2048;   // per softmax warp 64 bytes of 32 output rows
    static constexpr int kSmem = (2 + 2 * kStages) * kTile + kStaging + 1024 + 256;
};

struct alignas(64) PromptArgs {
    CUtensorMap map;           // bf16 pools: [page, keys / values, head, token][dimension in words], boxes of box_rows x 64 elements
    int box_rows;              // tokens of a page, at most 128; 0: no map (codes, or more rows than a map has)
    Attention a;
    Parts parts;
    Cut cut;
    float scale_log2;          // scale * log2(e)
    float cap_log2, cap_arg;   // cap * log2(e), scale / cap
};

namespace pro {

__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred P;\n\t"
        "setp.ne.b32 P, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, P;\n\t}"
        :
        : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        :
        : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
          "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]),
          "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// All threads of a named barrier learn whether all of them bring true.
__device__ __forceinline__ bool all_of(int barrier, int threads, bool mine)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(ok)
        : "r"(static_cast<uint32_t>(mine)), "r"(barrier), "r"(threads)
        : "memory");
    return ok != 0;
}

struct HalfSync {   // the four softmax warps of a half
    int barrier;
    __device__ __forceinline__ void operator()() const { asm volatile("barrier.cta.sync %0, 128;" ::"r"(barrier) : "memory"); }
};

// bounded_wait whose time does not run while softmax warps look at rows once more: that ends by itself, however long the row.
__device__ __forceinline__ bool patient_wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, const volatile unsigned int *working, int *status, int code)
{
    if (ptx::mbar_try_wait(bar, parity)) return true;
    long long t0 = clock64();
    uint32_t spins = 0;
    while (true) {
        if (ptx::mbar_try_wait(bar, parity)) return true;
        if ((++spins & 31u) == 0) {
            if (*abort_flag) return false;
            if (*working) {
                t0 = clock64();
            } else if (clock64() - t0 > kWaitTimeoutCycles) {
                *abort_flag = 1u;
                atomicCAS(status, 0, code);
                return false;
            }
        }
    }
}

// Bits 0 .. n - 1 of a word.
__device__ __forceinline__ uint32_t bits_below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }

__device__ __forceinline__ float rcp_fast(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
using tok::pair;
using tok::tanh_inner2;
using tok::unpair;
// tanh(x) of two values of any size: 1 - 2 / (1 + exp(2 x)), which is off by a share of 1, not of x, so that the polynomial stands up to 1
__device__ __forceinline__ unsigned long long tanh2(float x, float y)
{
    auto beyond = [](float v) { return fmaf(-2.0f, rcp_fast(1.0f + tok::exp2_fast(v * 2.8853900817779268f)), 1.0f); };
    float u, v;
    unpair(tanh_inner2(pair(x, y)), u, v);
    return pair(fabsf(x) <= 1.0f ? u : beyond(x), fabsf(y) <= 1.0f ? v : beyond(y));
}
// Eight codes as bf16 values times a power of two.  A code's bits in a bf16's place (exponent and mantissa side by side) stand for code * 2^-120, subnormal
// ones among them; one product by 2^(120 + e) puts them right, exactly, for e up to 7 (values up to 57344).
__device__ __forceinline__ uint32_t bf16_mul(uint32_t a, uint32_t b)
{
    uint32_t d;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
__device__ __forceinline__ uint4 codes8_to_bf16(uint2 w, uint32_t power)
{
    const uint32_t e0 = bf16_mul(((w.x << 4) & 0x07f007f0u) | ((w.x << 8) & 0x80008000u), power), o0 = bf16_mul(((w.x >> 4) & 0x07f007f0u) | (w.x & 0x80008000u), power);
    const uint32_t e1 = bf16_mul(((w.y << 4) & 0x07f007f0u) | ((w.y << 8) & 0x80008000u), power), o1 = bf16_mul(((w.y >> 4) & 0x07f007f0u) | (w.y & 0x80008000u), power);
    return make_uint4(__byte_perm(e0, o0, 0x5410), __byte_perm(e0, o0, 0x7632), __byte_perm(e1, o1, 0x5410), __byte_perm(e1, o1, 0x7632));
}
// A bit set: one of sixteen codes is the format's NaN (all bits but the sign).
__device__ __forceinline__ uint32_t nan_among(const uint4 &w)
{
    return (((w.x & 0x7f7f7f7fu) + 0x01010101u) | ((w.y & 0x7f7f7f7fu) + 0x01010101u) | ((w.z & 0x7f7f7f7fu) + 0x01010101u) | ((w.w & 0x7f7f7f7fu) + 0x01010101u)) & 0x80808080u;
}
// The same for what is rare: exponents from 8 on, NaN.
__device__ __noinline__ uint4 codes8_to_bf16_any(uint2 w, float scale)
{
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = codes2((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
        r[i] = ptx::pack_bf16x2(v.x * scale, v.y * scale);
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}

}  // namespace pro

// A tile's part of a range, as the roles need it.
struct Segment {
    int blocks;               // 0: the range is done
    int s, g, row0, pos0, packed0, rows;
    int from;                 // first block among the tile's
    KeyBlocks keys;
    int first[2], last[2], low[2];   // positions of each half's first and last row; keys below `low` are visible only among the first ones
    bool whole, tail;         // all of the tile's blocks; the tile begins in this range
    int b0, b1;               // blocks of the grid that share the tile
};
constexpr float kPromptGrowth = 32.0f;   // of a row's maximum, base 2, before what has been added up is scaled
constexpr int kPromptSegments = 4, kPromptSegmentWarps = 13;   // ring; warps that read it

template <int NB, bool CODES, bool CAPPED, bool SUMS>
__global__ void __launch_bounds__(kPromptThreads, 1)
paged_prompt_kernel(const __grid_constant__ PromptArgs args)
{
    using S = PromptShape<NB>;
    constexpr int kind = CODES ? KIND_E4M3 : KIND_BF16;
    constexpr float kLn2 = 0.69314718055994531f;
    extern __shared__ uint8_t prompt_smem[];
    __shared__ long long row_at[2][2][kPromptKeys];   // keys / values, in turn: element of a key's row, -1: zeros
    __shared__ int row_e[2][2][kPromptKeys];          // codes: exponent
    __shared__ int arrived_last[2];
    __shared__ UnsureRows unsure[2];
    __shared__ unsigned int working;   // halves that look at rows once more, which may take longer than any wait's limit
    __shared__ Segment segments[kPromptSegments];
    const Attention &a = args.a;
    const uint32_t base = (ptx::smem_u32(prompt_smem) + 1023u) & ~1023u;
    uint8_t *gen = prompt_smem + (base - ptx::smem_u32(prompt_smem));
    const uint32_t q_base = base, k_base = q_base + 2 * S::kTile, v_base = k_base + S::kStages * S::kTile, staging = v_base + S::kStages * S::kTile, bar = staging + S::kStaging;
    auto k_full = [&](int s) { return bar + 8u * s; };
    auto k_empty = [&](int s) { return bar + 8u * (3 + s); };
    auto v_full = [&](int s) { return bar + 8u * (6 + s); };
    auto v_empty = [&](int s) { return bar + 8u * (9 + s); };
    auto s_full = [&](int h) { return bar + 8u * (12 + h); };
    auto p_full = [&](int h) { return bar + 8u * (14 + h); };
    auto o_full = [&](int h) { return bar + 8u * (16 + h); };
    auto p_half = [&](int h) { return bar + 8u * (18 + h); };
    const uint32_t q_full = bar + 8u * 20, q_empty = bar + 8u * 21, drain = bar + 8u * 22;
    auto seg_full = [&](int i) { return bar + 8u * (23 + i % kPromptSegments); };
    auto seg_empty = [&](int i) { return bar + 8u * (23 + kPromptSegments + i % kPromptSegments); };
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(gen + (bar - base) + 8 * (23 + 2 * kPromptSegments));
    volatile uint32_t *abort_flag = tmem_slot + 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int *status = a.batch.status;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPromptMaxStages; ++s) {
            ptx::mbar_init(k_full(s), 64);
            ptx::mbar_init(k_empty(s), 1);
            ptx::mbar_init(v_full(s), 64);
            ptx::mbar_init(v_empty(s), 1);
        }
        for (int h = 0; h < 2; ++h) {
            ptx::mbar_init(s_full(h), 1);
            ptx::mbar_init(p_half(h), 128);
            ptx::mbar_init(p_full(h), 128);
            ptx::mbar_init(o_full(h), 1);
        }
        if (!CODES && args.box_rows) ptx::prefetch_tensormap(&args.map);
        for (int i = 0; i < kPromptSegments; ++i) {
            ptx::mbar_init(seg_full(i), 1);
            ptx::mbar_init(seg_empty(i), kPromptSegmentWarps);
        }
        ptx::mbar_init(q_full, 128);
        ptx::mbar_init(q_empty, 1);
        ptx::mbar_init(drain, 1);
        *abort_flag = 0u;
        working = 0u;
        ptx::fence_mbar_init();
    }
    if (warp == 4) {
        ptx::tmem_alloc(ptx::smem_u32(tmem_slot), 512);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *tmem_slot;   // columns: S / P of half h at 128 h, O at 256 + 128 h
    grid_dependency_wait();
    grid_dependency_launch();
    Place place;
    const Range range = range_of_block<kPromptThreads>(a, args.cut, place);
    const int dim = a.pages.dim, steps = (dim + 15) / 16;

    auto segment = [&](int i) -> const Segment & { return segments[i % kPromptSegments]; };
    auto segment_phase = [&](int i) { return (i / kPromptSegments) & 1; };
    auto release = [&](int i) {   // by every warp that reads segments
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(seg_empty(i));
    };
    auto needs = [&](const Segment &s, int h, int key) { return key <= s.last[h] && (key + kPromptKeys - 1 >= s.low[h] || key < a.sinks); };   // any row of the half, of a block of keys

    if (warp < 4) {
        ptx::reg_dec<104>();
        const int which = warp >> 1, t = threadIdx.x & 63;
        const uint32_t ring = which ? v_base : k_base;
        const int pieces = dim / 8, mask = (1 << a.pages.page_shift) - 1;
        int n = 0, tile = 0, b = 0;   // blocks and tiles so far, block of the tile's part
        bool boxes = false;
        // the rows that this block of keys comes from, two keys per thread
        auto look_up = [&] {
            const Segment &seg = segment(tile);
            const int key0 = block_key(seg.keys, seg.from + b, kPromptKeys), turn = n & 1;
            const int low = a.window ? seg.first[0] - a.window + 1 : 0, p1 = max(seg.last[0], seg.last[1]);
            // wanted as a whole: whole boxes out of the pages, a thread each
            boxes = !CODES && args.box_rows > 0 && key0 + kPromptKeys - 1 <= p1 && (key0 >= low || key0 + kPromptKeys <= a.sinks);
            if (boxes) {
                if (t * args.box_rows < kPromptKeys) {
                    const int key = key0 + t * args.box_rows, page = page_of(a.batch, a.pages, seg.s, key);
                    row_at[which][turn][t * args.box_rows] = page >= 0 ? a.pages.place(page, which, seg.g, key & mask) : -args.box_rows;   // no page: a box in front of the pool, zeros
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int key = key0 + t + 64 * i;
                const bool wanted = key <= p1 && (key >= low || key < a.sinks);
                const int page = wanted ? page_of(a.batch, a.pages, seg.s, key) : -1;
                const long long row = page >= 0 ? a.pages.place(page, which, seg.g, key & mask) : -1;
                row_at[which][turn][t + 64 * i] = row;
                if (CODES) row_e[which][turn][t + 64 * i] = row >= 0 ? static_cast<int>(a.pages.scales[row]) - 127 : 0;
            }
        };
        // the two warps learn together whether there is another tile
        auto another = [&] {
            const bool ok = pro::patient_wait(seg_full(tile), segment_phase(tile), abort_flag, &working, status, DEV_TIMEOUT_PRODUCER);
            return pro::all_of(2 + which, 64, ok) && segment(tile).blocks > 0;
        };
        bool more = another();
        if (more) look_up();
        while (more) {
            const int stage = n % S::kStages, turn = n & 1;
            const bool first = b == 0, by_box = boxes;
            const int packed0 = segment(tile).packed0, rows = segment(tile).rows, q_turn = tile & 1;
            const __nv_bfloat16 *q = static_cast<const __nv_bfloat16 *>(a.q) + segment(tile).row0 * a.q_pitch + segment(tile).g * a.share * dim;
            const uint32_t full = which ? v_full(stage) : k_full(stage);
            bool ok = pro::patient_wait(which ? v_empty(stage) : k_empty(stage), ((n / S::kStages) & 1) ^ 1, abort_flag, &working, status, DEV_TIMEOUT_PRODUCER);
            if (!pro::all_of(2 + which, 64, ok)) break;
            const uint32_t dst = ring + stage * S::kTile;
            if constexpr (!CODES) {
                if (by_box) {
                    if (t * args.box_rows < kPromptKeys) {
                        const int page_row = static_cast<int>(row_at[which][turn][t * args.box_rows]);
#pragma unroll
                        for (int c = 0; c < NB; ++c) ptx::tma_load_2d(dst + c * kPromptBlock + t * args.box_rows * 128, &args.map, 32 * c, page_row, full);
                    }
                } else {
                    const __nv_bfloat16 *data = static_cast<const __nv_bfloat16 *>(a.pages.data);
#pragma unroll 8
                    for (int i = 0; i < kPromptKeys * 8 * NB / 64; ++i) {
                        const int idx = i * 64 + t, r = idx / (8 * NB), c = idx % (8 * NB);
                        const long long row = row_at[which][turn][r];
                        const bool on = row >= 0 && c < pieces;
                        if (c < 2 * steps) tok::copy_or_zero<16>(dst + (c >> 3) * kPromptBlock + r * 128 + (((c & 7) ^ (r & 7)) << 4), on ? data + row * dim + c * 8 : data, on);
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            // on to the next block: its pages are looked up while this one's rows are on their way
            ++n;
            if (++b == segment(tile).blocks) {
                b = 0;
                release(tile++);
                more = another();
            }
            if (!CODES && more) look_up();
            if constexpr (CODES) {
                // its look-up in three steps between the conversions, so that nothing waits for the table or the powers of two
                int table_entry[2] = {-1, -1};
                long long next_row[2] = {-1, -1};
                uint32_t stored[2] = {127, 127};
                bool wanted[2] = {false, false};
                if (more) {
                    const Segment &seg = segment(tile);
                    const int key0 = block_key(seg.keys, seg.from + b, kPromptKeys), low = a.window ? seg.first[0] - a.window + 1 : 0, p1 = max(seg.last[0], seg.last[1]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int key = key0 + t + 64 * i;
                        wanted[i] = key <= p1 && (key >= low || key < a.sinks);
                        next_row[i] = key & mask;
                        if (wanted[i]) table_entry[i] = a.batch.table[static_cast<long long>(seg.s) * a.batch.table_pitch + (key >> a.pages.page_shift)];
                    }
                }
                auto second_step = [&] {
                    if (!more) return;
                    const int g = segment(tile).g;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const bool there = wanted[i] && table_entry[i] >= 0 && table_entry[i] < a.pages.num_pages;
                        if (wanted[i] && !there) report_bad(status);
                        next_row[i] = there ? a.pages.place(table_entry[i], which, g, static_cast<int>(next_row[i])) : -1;
                        if (there) stored[i] = a.pages.scales[next_row[i]];
                    }
                };
                auto third_step = [&] {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        row_at[which][n & 1][t + 64 * i] = next_row[i];
                        row_e[which][n & 1][t + 64 * i] = static_cast<int>(stored[i]) - 127;
                    }
                };
                // pieces of sixteen codes (two of eight where rows begin at odd multiples of eight); four are on their way while the four before become bf16
                const uint8_t *data = static_cast<const uint8_t *>(a.pages.data);
                constexpr int kPer = 4, kBatches = kPromptKeys * 4 * NB / 64 / kPer;
                const bool wide = dim % 16 == 0;
                const int c = t % (4 * NB), r0 = t / (4 * NB);   // the thread's columns 16 c .. 16 c + 15 of every (64 / 4 NB)-th row
                const bool low_on = c * 16 < dim, high_on = c * 16 + 8 < dim;
                uint4 w[2][kPer];
                auto load = [&](int batch, uint4 (&to)[kPer]) {
#pragma unroll
                    for (int u = 0; u < kPer; ++u) {
                        const long long row = row_at[which][turn][r0 + (batch * kPer + u) * (16 / NB)];
                        const uint8_t *from = data + row * dim + c * 16;
                        to[u] = make_uint4(0u, 0u, 0u, 0u);
                        if (row >= 0 && wide && low_on) {
                            to[u] = *reinterpret_cast<const uint4 *>(from);
                        } else if (row >= 0 && !wide) {
                            if (low_on) *reinterpret_cast<uint2 *>(&to[u].x) = *reinterpret_cast<const uint2 *>(from);
                            if (high_on) *reinterpret_cast<uint2 *>(&to[u].z) = *reinterpret_cast<const uint2 *>(from + 8);
                        }
                    }
                };
                load(0, w[0]);
#pragma unroll
                for (int batch = 0; batch < kBatches; ++batch) {
                    if (batch + 1 < kBatches) load(batch + 1, w[(batch + 1) & 1]);
                    if (batch == 1) second_step();
                    uint32_t rare = 0;   // a branch per batch, not per piece: four conversions run side by side
                    auto put = [&](int r, const uint4 &x, const uint4 &y) {
                        const uint32_t at = dst + (c >> 2) * kPromptBlock + r * 128;
                        if (2 * c < 2 * steps) ptx::sts128(at + (((2 * c & 7) ^ (r & 7)) << 4), x.x, x.y, x.z, x.w);
                        if (2 * c + 1 < 2 * steps) ptx::sts128(at + ((((2 * c + 1) & 7) ^ (r & 7)) << 4), y.x, y.y, y.z, y.w);
                    };
#pragma unroll
                    for (int u = 0; u < kPer; ++u) {
                        const int r = r0 + (batch * kPer + u) * (16 / NB), e = row_e[which][turn][r];
                        const uint4 v = w[batch & 1][u];
                        const uint32_t power = ((120 + min(e, 7) + 127) << 7) * 0x10001u;
                        rare |= pro::nan_among(v) | static_cast<uint32_t>(e > 7);
                        put(r, pro::codes8_to_bf16(make_uint2(v.x, v.y), power), pro::codes8_to_bf16(make_uint2(v.z, v.w), power));
                    }
                    if (rare) {
#pragma unroll
                        for (int u = 0; u < kPer; ++u) {
                            const int r = r0 + (batch * kPer + u) * (16 / NB);
                            const float scale = scale_of(row_e[which][turn][r] + 127);
                            const uint4 v = w[batch & 1][u];
                            put(r, pro::codes8_to_bf16_any(make_uint2(v.x, v.y), scale), pro::codes8_to_bf16_any(make_uint2(v.z, v.w), scale));
                        }
                    }
                }
                if (more) third_step();
            }
            if (by_box) {
                if (t == 0)
                    ptx::mbar_arrive_expect_tx(full, S::kTile);
                else
                    ptx::mbar_arrive(full);
            } else {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(full);
            }
            if (first) {   // queries, when the tile before has no more use for its own: all four warps, a row's pieces of eight side by side
                ok = pro::patient_wait(q_empty, q_turn ^ 1, abort_flag, &working, status, DEV_TIMEOUT_PRODUCER);   // run out: the warps leave together at the next block
#pragma unroll 4
                for (int i = threadIdx.x; ok && i < kPromptRows * 8 * NB; i += 128) {
                    const int r = i / (8 * NB), c = i % (8 * NB), packed = packed0 + r, token = a.shares.divide(packed);
                    const bool on = r < rows && c < pieces;
                    if (c < 2 * steps)
                        tok::copy_or_zero<16>(q_base + (r >> 7) * S::kTile + (c >> 3) * kPromptBlock + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4),
                                      on ? q + token * a.q_pitch + (packed - token * a.share) * dim + c * 8 : q, on);
                }
                asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
                ptx::fence_proxy_async_smem();
                ptx::mbar_arrive(q_full);
            }
        }
    } else if (warp < 8) {
        ptx::reg_dec<40>();
        if (warp == 4) {
            const bool issuer = ptx::elect_one();
            constexpr uint32_t idesc_s = ptx::make_idesc_bf16(128, 128, false, false);
            const uint32_t idesc_o = ptx::make_idesc_bf16(128, 16 * steps, false, true);
            const ptx::SmemDesc dq = ptx::smem_desc_words(q_base, 16, 1024, ptx::kLayoutSw128), dk = ptx::smem_desc_words(k_base, 16, 1024, ptx::kLayoutSw128),
                                dv = ptx::smem_desc_words(v_base, kPromptBlock, 1024, ptx::kLayoutSw128);
            auto wait = [&](uint32_t b, uint32_t parity, int code) { return __all_sync(0xffffffffu, pro::patient_wait(b, parity, abort_flag, &working, status, code)); };
            bool ok = true;
            int n = 0, turns[2] = {0, 0};
            for (int tile = 0; ok; ++tile) {
                ok = wait(seg_full(tile), segment_phase(tile), DEV_TIMEOUT_MMA_FULL);
                if (!ok) break;
                const Segment &seg = segment(tile);
                if (seg.blocks == 0) break;
                bool begun[2] = {false, false}, wanted[2] = {false, false};
                ok = wait(q_full, tile & 1, DEV_TIMEOUT_MMA_FULL);
                for (int b = -1; ok && b < seg.blocks; ++b) {
                    const int vs = (n + b) % S::kStages, ks = (n + b + 1) % S::kStages;
                    const bool more = b + 1 < seg.blocks;
                    const int next_key = more ? block_key(seg.keys, seg.from + b + 1, kPromptKeys) : 0;
                    if (b >= 0) ok = wait(v_full(vs), ((n + b) / S::kStages) & 1, DEV_TIMEOUT_MMA_FULL);
                    bool have_k = false;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (ok && b >= 0 && wanted[h]) {
#pragma unroll
                            for (int part = 0; part < 2; ++part) {
                                if (ok) ok = wait(part ? p_full(h) : p_half(h), turns[h] & 1, DEV_TIMEOUT_MMA_TMEM);
                                if (!ok) break;
                                ptx::tc_fence_after();
                                if (issuer) {
#pragma unroll
                                    for (int k = 4 * part; k < 4 * part + 4; ++k)
                                        pro::mma_ts(tmem + 256 + 128 * h, tmem + 128 * h + 8 * k, dv.at(vs * S::kTile + k * 2048), idesc_o, k > 0 || begun[h]);
                                }
                                __syncwarp();
                            }
                            if (!ok) break;
                            begun[h] = true;
                            turns[h]++;
                        }
                        if (!ok) break;
                        wanted[h] = more && needs(seg, h, next_key);
                        if (more && !have_k) {
                            ok = wait(k_full(ks), ((n + b + 1) / S::kStages) & 1, DEV_TIMEOUT_MMA_FULL);
                            if (!ok) break;
                            ptx::tc_fence_after();
                            have_k = true;
                        }
                        if (wanted[h]) {
                            if (issuer) {
                                uint32_t acc = 0;
                                for (int k = 0; k < steps; ++k) {
                                    const uint32_t off = (k >> 2) * kPromptBlock + (k & 3) * 32;
                                    ptx::mma_f16_ss(tmem + 128 * h, dq.at(h * S::kTile + off), dk.at(ks * S::kTile + off), idesc_s, acc);
                                    acc = 1;
                                }
                                ptx::mma_commit(s_full(h));
                            }
                            __syncwarp();
                        }
                    }
                    if (!ok) break;
                    if (issuer) {
                        if (b >= 0) ptx::mma_commit(v_empty(vs));
                        if (more) ptx::mma_commit(k_empty(ks));
                        if (b + 2 == seg.blocks) ptx::mma_commit(q_empty);   // the last scores
                        if (!more) {   // a half without products has nothing to wait for: its phases are those that its warps have weights for, so that none passes unseen
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                if (begun[h]) ptx::mma_commit(o_full(h));
                        }
                    }
                    __syncwarp();
                }
                if (!ok) break;
                n += seg.blocks;
                release(tile);
            }
            if (issuer) ptx::mma_commit(drain);
            __syncwarp();
            pro::patient_wait(drain, 0u, abort_flag, &working, status, DEV_TIMEOUT_DRAIN);
        } else if (warp == 5) {
            int n = 0;
            bool go = range.begin < range.end;
            for (long long at = range.begin, ended = 0; !ended;) {
                Segment seg{};
                if (go) {
                    const Part part = part_of(place, range, at, args.cut);
                    seg.blocks = part.blocks;
                    seg.s = place.s;
                    seg.g = place.g;
                    seg.row0 = place.q.row0;
                    seg.pos0 = place.q.pos0;
                    seg.packed0 = place.tile * kPromptRows;
                    seg.rows = min(kPromptRows, place.q.count * a.share - seg.packed0);
                    seg.from = part.from;
                    seg.keys = place.blocks;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool there = h * 128 < seg.rows;
                        seg.first[h] = there ? seg.pos0 + a.shares.divide(seg.packed0 + h * 128) : -1;
                        seg.last[h] = there ? seg.pos0 + a.shares.divide(seg.packed0 + min(seg.rows, h * 128 + 128) - 1) : -1;
                        seg.low[h] = a.window ? seg.first[h] - a.window + 1 : 0;
                    }
                    seg.whole = part.whole;
                    seg.tail = part.tail;
                    seg.b0 = part.b0;
                    seg.b1 = part.b1;
                    at += part.places;
                    go = advance(a, range, place, at, args.cut);
                } else {
                    ended = 1;   // the last entry: no blocks
                }
                if (!__all_sync(0xffffffffu, pro::patient_wait(seg_empty(n), segment_phase(n) ^ 1, abort_flag, &working, status, DEV_TIMEOUT_PRODUCER))) break;
                if (lane == 0) {
                    segments[n % kPromptSegments] = seg;
                    ptx::mbar_arrive(seg_full(n));
                }
                ++n;
            }
        }
        __syncwarp();
    } else {
        ptx::reg_inc<184>();
        const int h = warp >= 12, quarter = warp & 3;
        const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
        const uint32_t s_addr = tmem + lanes + 128 * h, o_addr = tmem + lanes + 256 + 128 * h;
        const int r = quarter * 32 + lane;   // row within the half
        auto wait = [&](uint32_t b, uint32_t parity) { return __all_sync(0xffffffffu, pro::patient_wait(b, parity, abort_flag, &working, status, DEV_TIMEOUT_EPILOGUE)); };
        bool ok = true;
        int turns = 0, outputs = 0;   // blocks with scores of this half so far, tiles with outputs of it
        for (int tile = 0;; ++tile) {
            if (!pro::all_of(4 + h, 128, wait(seg_full(tile), segment_phase(tile)))) break;
            const Segment &seg = segment(tile);
            if (seg.blocks == 0) break;
            const int packed = seg.packed0 + h * 128 + r;
            const bool there = h * 128 + r < seg.rows;
            const int token = a.shares.divide(packed), position = there ? seg.pos0 + token : -1;
            float ref = -INFINITY, sum = 0.0f, sum_rounded = 0.0f;   // what the weights stand against (base 2), their sum, that of the rounded ones
            bool begun = false;
            const int blocks = seg.blocks, half_first = seg.first[h], half_last = seg.last[h], half_low = seg.low[h];
            const KeyBlocks keys = seg.keys;
            int index = seg.from;
            for (int b = 0; b < blocks; ++b, ++index) {
                const int key0 = block_key(keys, index, kPromptKeys);
                if (key0 > half_last || (key0 + kPromptKeys - 1 < half_low && key0 >= a.sinks)) continue;   // not needed, as below
                ok = wait(s_full(h), turns & 1);
                if (!ok) break;
                ptx::tc_fence_after();
                turns++;
                const bool whole = key0 + kPromptKeys - 1 <= half_first && (a.window == 0 || key0 > half_last - a.window || key0 + kPromptKeys - 1 < a.sinks);
                uint32_t x[4][32];
#pragma unroll
                for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(s_addr + 32 * c, x[c]);
                ptx::tmem_ld_wait();
                if (CAPPED) {
                    // no score of the warp's rows beyond the cap: tanh is a polynomial; else the scores go through TMEM once more, 32 at a time (rare, and little code)
                    float widest[4] = {};
#pragma unroll
                    for (int i = 0; i < kPromptKeys; ++i) widest[i & 3] = fmaxf(widest[i & 3], fabsf(__uint_as_float(x[i >> 5][i & 31])));
                    const float most = fmaxf(fmaxf(widest[0], widest[1]), fmaxf(widest[2], widest[3]));
                    if (__all_sync(0xffffffffu, most * args.cap_arg <= 1.0f)) {
#pragma unroll
                        for (int i = 0; i < kPromptKeys; i += 2) {
                            float u, v;
                            const unsigned long long t = ptx::mul2(pro::pair(__uint_as_float(x[i >> 5][i & 31]), __uint_as_float(x[i >> 5][(i & 31) + 1])), ptx::both(args.cap_arg));
                            pro::unpair(ptx::mul2(pro::tanh_inner2(t), ptx::both(args.cap_log2)), u, v);
                            x[i >> 5][i & 31] = __float_as_uint(u);
                            x[i >> 5][(i & 31) + 1] = __float_as_uint(v);
                        }
                    } else {
#pragma unroll 1
                        for (int c = 0; c < 8; ++c) {
                            uint32_t y[16];
                            pro::tmem_ld_32x16(s_addr + 16 * c, y);
                            ptx::tmem_ld_wait();
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                float u, v;
                                pro::unpair(ptx::mul2(pro::tanh2(__uint_as_float(y[i]) * args.cap_arg, __uint_as_float(y[i + 1]) * args.cap_arg), ptx::both(args.cap_log2)), u, v);
                                y[i] = __float_as_uint(u);
                                y[i + 1] = __float_as_uint(v);
                            }
                            pro::tmem_st_32x16(s_addr + 16 * c, y);
                        }
                        pro::tmem_st_wait();
#pragma unroll
                        for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(s_addr + 32 * c, x[c]);
                        ptx::tmem_ld_wait();
                    }
                }
                if (!whole) {
                    // keys up to `high`, but only those from `low` on or before `first`: a bit per key
                    const int high = position - key0, low = a.window ? high - a.window + 1 : 0, first = a.sinks - key0;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint32_t seen = pro::bits_below(high + 1 - 32 * c) & (~pro::bits_below(low - 32 * c) | pro::bits_below(first - 32 * c));
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[c][i] = seen & (1u << i) ? x[c][i] : 0xff800000u;   // minus infinity
                    }
                }
                float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kPromptKeys; i += 2)
                    most[(i >> 1) & 3] = fmaxf(fmaxf(most[(i >> 1) & 3], __uint_as_float(x[i >> 5][i & 31])), __uint_as_float(x[i >> 5][(i & 31) + 1]));
                float top = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
                if (!CAPPED) top *= args.scale_log2;
                const bool grow = top > ref + kPromptGrowth || (ref == -INFINITY && top > -INFINITY);
                if (!begun) {
                    ref = top;
                } else if (__any_sync(0xffffffffu, grow)) {
                    // earlier weights stand against the old maximum: scale O (complete: this block's scores come after it) and the sum
                    const float f = grow ? tok::exp2_fast(ref - top) : 1.0f;
                    if (grow) ref = top;
                    sum *= f;
                    sum_rounded *= f;
#pragma unroll 1
                    for (int c = 0; c < 16 * steps; c += 16) {
                        uint32_t o[16];
                        pro::tmem_ld_32x16(o_addr + c, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        pro::tmem_st_32x16(o_addr + c, o);
                    }
                }
                begun = true;
                const float use = ref == -INFINITY ? 0.0f : ref;   // nothing seen yet: every weight is 2^-inf = 0
                const unsigned long long scale2 = ptx::both(args.scale_log2), minus_ref = ptx::both(-use);
                unsigned long long sums[2] = {0, 0}, rounded[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const unsigned long long v = pro::pair(__uint_as_float(x[c][2 * i]), __uint_as_float(x[c][2 * i + 1]));
                        float e0, e1;
                        pro::unpair(CAPPED ? ptx::add2(v, minus_ref) : ptx::fma2(v, scale2, minus_ref), e0, e1);
                        e0 = tok::exp2_fast(e0);
                        e1 = tok::exp2_fast(e1);
                        if (SUMS) sums[i & 1] = ptx::add2(sums[i & 1], pro::pair(e0, e1));
                        w[i] = ptx::pack_bf16x2(e0, e1);
                        rounded[i & 1] = ptx::add2(rounded[i & 1], pro::pair(bf16_low(w[i]), bf16_high(w[i])));
                    }
                    pro::tmem_st_32x16(s_addr + 16 * c, w);
                    if (c == 1) {   // the first 64 keys' weights: their products may begin
                        pro::tmem_st_wait();
                        ptx::tc_fence_before();
                        ptx::mbar_arrive(p_half(h));
                    }
                }
                float e0, e1;
                if (SUMS) {
                    pro::unpair(ptx::add2(sums[0], sums[1]), e0, e1);
                    sum += e0 + e1;
                }
                pro::unpair(ptx::add2(rounded[0], rounded[1]), e0, e1);
                sum_rounded += e0 + e1;
                pro::tmem_st_wait();
                ptx::tc_fence_before();
                ptx::mbar_arrive(p_full(h));
            }
            // where the outputs go, while the last products run
            const bool sees = position >= 0;
            const int head = seg.g * a.share + packed - token * a.share, piece = lane & 3;
            const long long row = seg.row0 + token;
            const uint32_t stage = staging + (4 * h + quarter) * 2048;
            __nv_bfloat16 *to[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int rr = h * 128 + quarter * 32 + 8 * i + (lane >> 2), pr = seg.packed0 + rr, tk = a.shares.divide(pr);
                to[i] = rr < seg.rows ? static_cast<__nv_bfloat16 *>(a.out) + (seg.row0 + tk) * a.out_pitch + (seg.g * a.share + pr - tk * a.share) * dim + 8 * piece : nullptr;
            }
            const float by_whole = 1.0f / sum_rounded;
            if (ok && begun) ok = wait(o_full(h), outputs++ & 1);
            ptx::tc_fence_after();
            if (!pro::all_of(4 + h, 128, ok)) break;
            if (h * 128 < seg.rows) {
                // 32 columns of the warp's rows at a time go through shared memory, so that four lanes store a row's 64 bytes side by side
                float check = 0.0f;   // zero times every output: NaN where one is not finite
                auto store = [&](int c, const float (&o)[32], float by) {   // columns c .. c + 31
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float u = o[2 * i] * by, v = o[2 * i + 1] * by;
                        if (c + 2 * i < dim) check = fmaf(v, 0.0f, fmaf(u, 0.0f, check));
                        w[i] = sees ? ptx::pack_bf16x2(u, v) : 0u;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) ptx::sts128(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4), w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int rr = 8 * i + (lane >> 2);
                        const float4 v = ptx::lds128(stage + rr * 64 + ((piece ^ ((rr >> 1) & 3)) << 4));
                        if (to[i] && c + 8 * piece < dim) *reinterpret_cast<float4 *>(to[i] + c) = v;
                    }
                    __syncwarp();
                };
                auto store_sum = [&](float top, float total) {
                    if (SUMS && there) a.lse[row * a.heads + head] = sees ? top * kLn2 + logf(total) : -INFINITY;
                };
                bool done = seg.whole;
                float divisor = sum_rounded;
                if (seg.whole) {
                    for (int c = 0; c < 16 * steps; c += 32) {
                        uint32_t o[32];
                        ptx::tmem_ld_32x32(o_addr + c, o);
                        ptx::tmem_ld_wait();
                        float v[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(o[i]);
                        store(c, v, by_whole);
                    }
                    store_sum(ref, sum);
                } else {
                    // four columns of all rows side by side, so that the rows' threads write and read runs
                    float *part = args.parts.base + (2LL * blockIdx.x + seg.tail) * args.parts.floats + h * (128 * 128 + 512);
                    for (int c = 0; c < 16 * steps; c += 32) {
                        uint32_t o[32];
                        ptx::tmem_ld_32x32(o_addr + c, o);
                        ptx::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<uint4 *>(part + ((c / 4 + i) * 128 + r) * 4) = begun ? make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]) : make_uint4(0u, 0u, 0u, 0u);
                    }
                    *reinterpret_cast<float4 *>(part + 128 * 128 + 4 * r) = make_float4(ref, sum, sum_rounded, 0.0f);
                    const int b0 = seg.b0, b1 = seg.b1;
                    __threadfence();
                    pro::all_of(4 + h, 128, true);
                    if (r == 0) {
                        const unsigned int before = atomicAdd(args.parts.tickets + 2 * b0 + h, 1u);
                        arrived_last[h] = before == static_cast<unsigned int>(b1 - b0);
                        if (arrived_last[h]) args.parts.tickets[2 * b0 + h] = 0u;
                        __threadfence();
                    }
                    pro::all_of(4 + h, 128, true);
                    done = arrived_last[h];
                    if (done) {
                        auto slot = [&](int b) { return args.parts.base + (2LL * b + (b == b0)) * args.parts.floats + h * (128 * 128 + 512); };
                        float top = -INFINITY, total = 0.0f, total_rounded = 0.0f;
                        for (int b = b0; b <= b1; ++b) top = fmaxf(top, __ldcg(slot(b) + 128 * 128 + 4 * r));
                        for (int b = b0; b <= b1; ++b) {
                            const float4 ml = __ldcg(reinterpret_cast<const float4 *>(slot(b) + 128 * 128 + 4 * r));
                            const float f = tok::share_of(ml.x, top);
                            total = fmaf(ml.y, f, total);
                            total_rounded = fmaf(ml.z, f, total_rounded);
                        }
                        const float by = 1.0f / total_rounded;
                        divisor = total_rounded;
                        for (int c = 0; c < 16 * steps; c += 32) {
                            float v[32] = {};
                            for (int b = b0; b <= b1; ++b) {
                                const float *from = slot(b);
                                const float f = tok::share_of(__ldcg(from + 128 * 128 + 4 * r), top);
#pragma unroll
                                for (int i = 0; i < 8; ++i) {
                                    const float4 u = __ldcg(reinterpret_cast<const float4 *>(from + ((c / 4 + i) * 128 + r) * 4));
                                    v[4 * i] = fmaf(u.x, f, v[4 * i]); v[4 * i + 1] = fmaf(u.y, f, v[4 * i + 1]);
                                    v[4 * i + 2] = fmaf(u.z, f, v[4 * i + 2]); v[4 * i + 3] = fmaf(u.w, f, v[4 * i + 3]);
                                }
                            }
                            store(c, v, by);
                        }
                        store_sum(top, total);
                    }
                }
                const uint32_t bad = __ballot_sync(0xffffffffu, done && there && sees && check != 0.0f && divisor > 0.0f && divisor <= FLT_MAX);
                if (lane == 0) unsure[h].rows[quarter] = bad;
                if (__builtin_expect(!pro::all_of(4 + h, 128, bad == 0), 0)) {
                    if (r == 0) atomicAdd(&working, 1u);
                    settle_rows<__nv_bfloat16, kind, 4>(a, seg.s, seg.g, seg.row0, seg.pos0, seg.packed0 + h * 128, unsure[h], quarter, reinterpret_cast<float *>(gen + (staging - base) + 4 * h * 2048),
                                                        pro::HalfSync{4 + h});
                    if (r == 0) atomicSub(&working, 1u);
                }
            }
            ptx::tc_fence_before();   // the accumulator has been read: the next tile's products may write it (they wait for its weights)
            release(tile);
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);   // copies still in flight land before the memory is handed on
    }
    __syncthreads();
    if (warp == 4) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, 512);
    }
}

}  // namespace kvp
}  // namespace gptb200
