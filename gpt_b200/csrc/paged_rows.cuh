// Attention over a paged cache on fp32 FMAs: queries or cache in fp32 (GPT-2's own precision), any kind of pages.  Both forms share the line of work and the end of a tile
// with the tensor-core form of few rows (kv_pages.cuh, paged_tokens.cuh).
//
//   paged_few_kernel    a row at a time (single tokens): half a warp holds a row of 128 (eight dimensions a lane) and takes every second key straight from the pages; eight
//                       keys per warp are under way at a time.  Bound by the cache's bytes, and by latency where they are few.
//   paged_rows_kernel   16 or 32 packed rows against blocks of 32 keys in shared memory: a warp's four or eight rows meet a key per lane, then four dimensions per lane.  Eight
//                       (twelve) wavefronts of shared memory for 16 (32) FMAs a lane in the scores, five (six) in the weighted values.
#pragma once

#include "paged_tokens.cuh"

namespace gptb200 {
namespace kvp {

constexpr int kFewKeys = 64, kFewPerSm = 3;
constexpr int kRowsKeys = 32, kRowsPerSm = 3;
__host__ __device__ constexpr int rows_tile(int each) { return kTokensWarps * each; }                  // rows of a tile, `each` per warp
__host__ __device__ constexpr int rows_part(int each) { return rows_tile(each) * 128 + 2 * rows_tile(each); }   // floats of a part in scratch
constexpr float kFmaGrowth = 32.0f;   // of a row's maximum, base 2, before what has been added up is scaled
constexpr float kLog2E = 1.4426950408889634f;

constexpr int kFewBlocks = kFewPerSm * 160, kRowsBlocks = kRowsPerSm * 160;   // of a grid, at most: so many parts' sums have room in shared memory
constexpr int kFewSmem = kFewBlocks * 8;   // the warps' sums, 132 floats each, have room in it
static_assert(kFewSmem >= kTokensWarps * 132 * 4 && kTeamRoom <= 132);
__host__ __device__ constexpr int rows_smem(int each) { return (rows_tile(each) + 2 * kRowsKeys) * 132 * 4 + kTokensWarps * kRowsKeys * each * 4; }
static_assert(rows_smem(4) / 8 >= kRowsBlocks);

// A score in base 2.
__device__ __forceinline__ float score2(const Attention &a, float dot)
{
    const float x = dot * a.scale;
    return (a.cap > 0.0f ? a.cap * tanhf(x / a.cap) : x) * kLog2E;
}

template <typename T, int KIND>
__global__ void __launch_bounds__(kTokensThreads, kFewPerSm)
paged_few_kernel(const __grid_constant__ TokensArgs args)
{
    using tok::exp2_fast;
    extern __shared__ __align__(16) float rows_shared[];
    __shared__ float warp_ml[kTokensWarps][2], total_ml[1][2];
    __shared__ UnsureRows unsure;
    __shared__ int arrived_last;
    const Attention &a = args.a;
    grid_dependency_wait();
    grid_dependency_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane & 15, half = lane >> 4;
    Place place;
    const Range range = range_of_block<kTokensThreads>(a, args.cut, place);
    const int dim = a.pages.dim, mask = (1 << a.pages.page_shift) - 1;
    const bool active = piece < dim / 8;
    for (long long at = range.begin; at < range.end;) {
        const Part part = part_of(place, range, at, args.cut);
        at += part.places;
        const int packed = place.tile, token = a.shares.divide(packed), position = place.q.pos0 + token, low = a.window ? position - a.window + 1 : 0;
        float q[8] = {}, acc[8] = {}, m = -INFINITY, l = 0.0f;
        if (active) load8(q, static_cast<const T *>(a.q) + (place.q.row0 + token) * a.q_pitch + (place.g * a.share + packed - token * a.share) * dim + piece * 8);
        auto first_key = [&](int i) { return block_key(place.blocks, part.from + i, kFewKeys) + warp * 16; };
        auto wanted = [&](int key) { return key <= position && (key >= low || key < a.sinks); };
        // pages of the warp's two groups of eight keys, one block ahead
        int pages[2];
        auto look_up = [&](int i) {
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const int key = i < part.blocks ? first_key(i) + 8 * g : 0;
                pages[g] = i < part.blocks && key <= position && (key + 7 >= low || key < a.sinks) ? page_of(a.batch, a.pages, place.s, key) : -1;
            }
        };
        look_up(0);
        if (threadIdx.x < 4) unsure.rows[threadIdx.x] = 0u;
        for (int it = 0; it < part.blocks; ++it) {
            const int t = first_key(it), page[2] = {pages[0], pages[1]};
            look_up(it + 1);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (page[g] < 0) continue;   // the same for the whole warp
                float k[4][8] = {}, v[4][8] = {};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int key = t + 8 * g + 2 * u + half;
                    if (active && wanted(key)) {
                        load8_held<KIND>(k[u], a.pages, page[g], 0, place.g, key & mask, piece);
                        load8_held<KIND>(v[u], a.pages, page[g], 1, place.g, key & mask, piece);
                    }
                }
                float x[4], top = -INFINITY;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    x[u] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[u] = fmaf(q[e], k[u][e], x[u]);
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1)
#pragma unroll
                    for (int u = 0; u < 4; ++u) x[u] += __shfl_xor_sync(0xffffffffu, x[u], o);
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    x[u] = wanted(t + 8 * g + 2 * u + half) ? score2(a, x[u]) : -INFINITY;
                    top = fmaxf(top, x[u]);
                }
                if (top > m + kFmaGrowth || (m == -INFINITY && top > -INFINITY)) {   // the same for the half warp
                    const float f = exp2_fast(m - top);
                    m = top;
                    l *= f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] *= f;
                }
                const float against = m == -INFINITY ? 0.0f : m;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float p = exp2_fast(x[u] - against);
                    l += p;
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[e] = fmaf(p, v[u][e], acc[e]);
                }
            }
        }
        // the halves, then the warps
        const float both = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16)), to_both = tok::share_of(m, both);
        m = both;
        l *= to_both;
        l += __shfl_xor_sync(0xffffffffu, l, 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            acc[e] *= to_both;
            acc[e] += __shfl_xor_sync(0xffffffffu, acc[e], 16);
        }
        if (lane == 0) {
            warp_ml[warp][0] = m;
            warp_ml[warp][1] = l;
        }
        __syncthreads();
        float top = warp_ml[0][0], sum = 0.0f;
#pragma unroll
        for (int w = 1; w < kTokensWarps; ++w) top = fmaxf(top, warp_ml[w][0]);
#pragma unroll
        for (int w = 0; w < kTokensWarps; ++w) sum += warp_ml[w][1] * tok::share_of(warp_ml[w][0], top);
        if (threadIdx.x == 0) {
            total_ml[0][0] = top;
            total_ml[0][1] = sum;
        }
        const float to_top = tok::share_of(m, top);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= to_top;
        if (half == 0) store8(rows_shared + warp * 132 + piece * 8, acc);
        __syncthreads();
        finish_tile<T, KIND, 1, kTokensWarps>(a, args.parts, place, part, 1, rows_shared, 132, total_ml, reinterpret_cast<float2 *>(rows_shared), kFewBlocks, unsure, &arrived_last);
        if (!advance(a, range, place, at, args.cut)) break;
    }
}

// kRowsEach: rows of a warp, 4 or 8
template <typename T, int KIND, int kRowsEach>
__global__ void __launch_bounds__(kTokensThreads, kRowsPerSm)
paged_rows_kernel(const __grid_constant__ TokensArgs args)
{
    using tok::exp2_fast;
    constexpr int kRowsTile = rows_tile(kRowsEach);
    constexpr int kPitch = 132;   // floats: lanes that read a row each touch all banks
    extern __shared__ __align__(16) float rows_shared[];
    __shared__ float total_ml[kRowsTile][2];
    __shared__ long long key_row[2][kRowsKeys];   // in turn: a key's row among its page's, -1: zeros
    __shared__ UnsureRows unsure;
    __shared__ int arrived_last;
    float *queries = rows_shared, *keys = queries + kRowsTile * kPitch, *values = keys + kRowsKeys * kPitch, *weights = values + kRowsKeys * kPitch;   // weights [warp][key][row of the warp]
    const Attention &a = args.a;
    grid_dependency_wait();
    grid_dependency_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Place place;
    const Range range = range_of_block<kTokensThreads>(a, args.cut, place);
    const int dim = a.pages.dim, pieces = dim / 8, mask = (1 << a.pages.page_shift) - 1;
    // weighted values: four dimensions a lane; heads of up to 64 leave half of the lanes to every second key
    const bool narrow = dim <= 64;
    const int lane_d = 4 * (narrow ? lane & 15 : lane), lane_key = narrow ? lane >> 4 : 0, key_step = narrow ? 2 : 1;
    const long long values_at = static_cast<long long>(a.pages.kv_heads) << a.pages.page_shift;   // from a key's row to its value's
    for (long long at = range.begin; at < range.end;) {
        const Part part = part_of(place, range, at, args.cut);
        at += part.places;
        const int packed0 = place.tile * kRowsTile, rows = min(kRowsTile, place.q.count * a.share - packed0);
        const int p0 = place.q.pos0 + a.shares.divide(packed0), p1 = place.q.pos0 + a.shares.divide(packed0 + rows - 1), low = a.window ? p0 - a.window + 1 : 0;
        auto look_up = [&](int i) {   // by the first warp
            const int key = block_key(place.blocks, part.from + i, kRowsKeys) + lane;
            const int page = key <= p1 && (key >= low || key < a.sinks) ? page_of(a.batch, a.pages, place.s, key) : -1;
            key_row[i & 1][lane] = page >= 0 ? a.pages.place(page, 0, place.g, key & mask) : -1;
        };
        for (int i = threadIdx.x; i < kRowsTile * pieces; i += kTokensThreads) {
            const int r = i / pieces, c = i % pieces, packed = packed0 + r, token = a.shares.divide(packed);
            float v[8] = {};
            if (r < rows) load8(v, static_cast<const T *>(a.q) + (place.q.row0 + token) * a.q_pitch + (place.g * a.share + packed - token * a.share) * dim + c * 8);
            store8(queries + r * kPitch + c * 8, v);
        }
        if (warp == 0) look_up(0);
        if (threadIdx.x < 4) unsure.rows[threadIdx.x] = 0u;
        float m[kRowsEach], l[kRowsEach], O[kRowsEach][4] = {};
        int pos[kRowsEach];
#pragma unroll
        for (int i = 0; i < kRowsEach; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
            pos[i] = kRowsEach * warp + i < rows ? place.q.pos0 + a.shares.divide(packed0 + kRowsEach * warp + i) : -1;
        }
        for (int it = 0; it < part.blocks; ++it) {
            __syncthreads();   // the block before has been read, this one's rows are known
            for (int i = threadIdx.x; i < 2 * kRowsKeys * pieces; i += kTokensThreads) {
                const int rr = i / pieces, c = i % pieces, which = rr >= kRowsKeys, r = rr & (kRowsKeys - 1);
                const long long row = key_row[it & 1][r];
                float v[8] = {};
                if (row >= 0) {
                    const long long from = row + (which ? values_at : 0), element = from * dim + c * 8;
                    if constexpr (KIND == KIND_E4M3)
                        load8_codes(v, static_cast<const uint8_t *>(a.pages.data) + element, scale_of(a.pages.scales[from]));
                    else if constexpr (KIND == KIND_BF16)
                        load8(v, static_cast<const __nv_bfloat16 *>(a.pages.data) + element);
                    else
                        load8(v, static_cast<const float *>(a.pages.data) + element);
                }
                store8((which ? values : keys) + r * kPitch + c * 8, v);
            }
            if (warp == 0 && it + 1 < part.blocks) look_up(it + 1);
            __syncthreads();
            if (kRowsEach * warp >= rows) continue;
            const int key = block_key(place.blocks, part.from + it, kRowsKeys) + lane;
            float x[kRowsEach] = {};
#pragma unroll 4
            for (int d = 0; d < dim; d += 4) {
                const float4 kk = *reinterpret_cast<const float4 *>(keys + lane * kPitch + d);
#pragma unroll
                for (int i = 0; i < kRowsEach; ++i) {
                    const float4 qq = *reinterpret_cast<const float4 *>(queries + (kRowsEach * warp + i) * kPitch + d);
                    x[i] = fmaf(qq.x, kk.x, fmaf(qq.y, kk.y, fmaf(qq.z, kk.z, fmaf(qq.w, kk.w, x[i]))));
                }
            }
            float w[kRowsEach];
#pragma unroll
            for (int i = 0; i < kRowsEach; ++i) {
                x[i] = visible(a, key, pos[i]) ? score2(a, x[i]) : -INFINITY;
                if (__any_sync(0xffffffffu, x[i] > m[i] + kFmaGrowth || (m[i] == -INFINITY && x[i] > -INFINITY))) {
                    float top = x[i];
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                    top = fmaxf(top, m[i]);
                    const float f = exp2_fast(m[i] - top);
                    m[i] = top;
                    l[i] *= f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) O[i][e] *= f;
                }
                w[i] = exp2_fast(x[i] - (m[i] == -INFINITY ? 0.0f : m[i]));
                l[i] += w[i];
            }
            float *mine = weights + warp * kRowsKeys * kRowsEach;
#pragma unroll
            for (int i = 0; i < kRowsEach; i += 4) *reinterpret_cast<float4 *>(mine + lane * kRowsEach + i) = make_float4(w[i], w[i + 1], w[i + 2], w[i + 3]);
            __syncwarp();
            if (lane_d < dim) {
#pragma unroll 8
                for (int j = lane_key; j < kRowsKeys; j += key_step) {
                    float pp[kRowsEach];
#pragma unroll
                    for (int i = 0; i < kRowsEach; i += 4) {
                        const float4 p = *reinterpret_cast<const float4 *>(mine + j * kRowsEach + i);
                        pp[i] = p.x; pp[i + 1] = p.y; pp[i + 2] = p.z; pp[i + 3] = p.w;
                    }
                    const float4 v = *reinterpret_cast<const float4 *>(values + j * kPitch + lane_d);
#pragma unroll
                    for (int i = 0; i < kRowsEach; ++i) {
                        O[i][0] = fmaf(pp[i], v.x, O[i][0]);
                        O[i][1] = fmaf(pp[i], v.y, O[i][1]);
                        O[i][2] = fmaf(pp[i], v.z, O[i][2]);
                        O[i][3] = fmaf(pp[i], v.w, O[i][3]);
                    }
                }
            }
            __syncwarp();
        }
        __syncthreads();
        // the queries' place takes the sums
#pragma unroll
        for (int i = 0; i < kRowsEach; ++i) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], o);
            if (lane == 0) {
                total_ml[kRowsEach * warp + i][0] = m[i];
                total_ml[kRowsEach * warp + i][1] = l[i];
            }
            if (narrow) {
#pragma unroll
                for (int e = 0; e < 4; ++e) O[i][e] += __shfl_xor_sync(0xffffffffu, O[i][e], 16);
            }
            if (lane_d < dim && lane_key == 0) *reinterpret_cast<float4 *>(queries + (kRowsEach * warp + i) * kPitch + lane_d) = make_float4(O[i][0], O[i][1], O[i][2], O[i][3]);
        }
        __syncthreads();
        finish_tile<T, KIND, kRowsTile, 1>(a, args.parts, place, part, rows, queries, kPitch, total_ml, reinterpret_cast<float2 *>(rows_shared), rows_smem(kRowsEach) / 8, unsure, &arrived_last);
        if (!advance(a, range, place, at, args.cut)) break;
    }
}

}  // namespace kvp
}  // namespace gptb200
