// Entry points of the paged cache of keys and values (include/gptb200.h: gptb200_kv_pages_*, gptb200_attention_paged): checks, choice of kernel, launches.
#include <algorithm>
#include <climits>
#include <cmath>

#include "ctx_internal.h"
#include "paged_prompt_sm100.cuh"
#include "paged_rows.cuh"

using namespace gptb200;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool aligned4(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

// The device that is current at the call stays so.
struct OnDevice {
    int before = -1;
    bool changed = false;
    cudaError_t enter(int device)
    {
        cudaError_t e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device) {
            e = cudaSetDevice(device);
            changed = e == cudaSuccess;
        }
        return e;
    }
    ~OnDevice()
    {
        if (changed) cudaSetDevice(before);
    }
};

int check_pages(gptb200_ctx *ctx, const gptb200_kv_pages *p, const gptb200_kv_rows *b, kvp::Pages *pages, kvp::Batch *batch)
{
    if (!p || !b) return fail(ctx, GPTB200_ERR_INVALID_ARG, "no pages or no rows given");
    if (p->kind < GPTB200_KV_BF16 || p->kind > GPTB200_KV_E4M3) return fail(ctx, GPTB200_ERR_INVALID_ARG, "kind %d of pages is unknown", p->kind);
    if (p->num_pages < 0 || p->kv_heads <= 0 || p->dim < 8 || p->dim > 128 || p->dim % 8 || p->page_tokens < 8 || p->page_tokens > 4096 || (p->page_tokens & (p->page_tokens - 1)))
        return fail(ctx, GPTB200_ERR_INVALID_ARG, "pages: %d of %d tokens (a power of two from 8 to 4096), %d heads of %d (a multiple of 8, at most 128)", p->num_pages, p->page_tokens, p->kv_heads,
                    p->dim);
    if (b->sequences < 0 || b->rows < 0 || b->max_new < 0 || b->table_pitch < 0)
        return fail(ctx, GPTB200_ERR_INVALID_ARG, "rows: %d sequences, %d rows, %d new at most, %d pages each", b->sequences, b->rows, b->max_new, b->table_pitch);
    if (b->sequences == INT_MAX) return fail(ctx, GPTB200_ERR_TOO_LARGE, "too many sequences");
    if (b->sequences > 0 && b->rows > 0) {
        if (!p->data || !aligned16(p->data) || (p->kind == GPTB200_KV_E4M3 && (!p->scales || !aligned16(p->scales))))
            return fail(ctx, GPTB200_ERR_INVALID_ARG, "pages: no memory, or not aligned to 16 bytes");
        if (!b->row_starts || !b->lengths || (!b->page_table && b->table_pitch > 0)) return fail(ctx, GPTB200_ERR_INVALID_ARG, "rows: no starts, lengths or page table");
        if (!aligned4(b->row_starts) || !aligned4(b->lengths) || !aligned4(b->page_table)) return fail(ctx, GPTB200_ERR_INVALID_ARG, "rows: an array of int32 is not aligned to 4 bytes");
    }
    int shift = 0;
    while ((1 << shift) < p->page_tokens) ++shift;
    *pages = {p->data, p->kind == GPTB200_KV_E4M3 ? p->scales : nullptr, p->num_pages, shift, p->kv_heads, p->dim};
    const long long capacity = std::min<long long>(static_cast<long long>(b->table_pitch) << shift, 1 << 30);
    *batch = {b->row_starts, b->lengths, b->page_table, b->sequences, b->table_pitch, b->rows, static_cast<int>(capacity), ctx ? ctx->d_status : nullptr};
    return GPTB200_OK;
}

// rows of `width` elements with a pitch: 16-byte pieces everywhere
int check_rows(gptb200_ctx *ctx, const char *what, const void *p, long long pitch, long long width, int dtype)
{
    const int per16 = dtype == GPTB200_DTYPE_F32 ? 4 : 8;
    if (!p || !aligned16(p) || pitch < width || pitch % per16)
        return fail(ctx, GPTB200_ERR_INVALID_ARG, "%s: no memory, not aligned to 16 bytes, or a pitch of %lld for rows of %lld (a multiple of %d)", what, pitch, width, per16);
    return GPTB200_OK;
}

template <bool WRITE>
int run_rows(gptb200_ctx *ctx, void *k, long long k_pitch, void *v, long long v_pitch, int dtype, const gptb200_kv_pages *pages, const gptb200_kv_rows *rows)
{
    if (!ctx) return GPTB200_ERR_INVALID_ARG;
    if (dtype != GPTB200_DTYPE_BF16 && dtype != GPTB200_DTYPE_F32) return fail(ctx, GPTB200_ERR_INVALID_ARG, "dtype %d is unknown", dtype);
    kvp::RowsArgs a{};
    int rc = check_pages(ctx, pages, rows, &a.pages, &a.batch);
    if (rc != GPTB200_OK) return rc;
    if (rows->sequences == 0 || rows->rows == 0) return GPTB200_OK;
    const long long width = 1LL * pages->kv_heads * pages->dim;
    if ((rc = check_rows(ctx, "keys", k, k_pitch, width, dtype)) != GPTB200_OK || (rc = check_rows(ctx, "values", v, v_pitch, width, dtype)) != GPTB200_OK) return rc;
    if (width > INT_MAX / 64) return fail(ctx, GPTB200_ERR_TOO_LARGE, "rows of %lld elements", width);
    OnDevice device;
    CUDA_TRY(ctx, device.enter(ctx->device));
    a.k = k; a.v = v; a.k_pitch = k_pitch; a.v_pitch = v_pitch;
    const bool sixteens = pages->dim % 16 == 0;
    while ((1 << a.lanes_log2) < pages->dim / (sixteens ? 16 : 8)) ++a.lanes_log2;
    // a row's threads, as many rows side by side as the block has room for; a few rows per thread while that fills the GPU
    const int all_columns = 2 * pages->kv_heads << a.lanes_log2;
    a.columns = std::min(all_columns, kvp::kRowThreads);
    const int side = kvp::kRowThreads / a.columns, threads = (side * a.columns + 31) / 32 * 32;
    a.rows_per_block = std::max(1, std::min({kvp::kRowMax, kvp::row_turns(WRITE) * side, rows->rows / (2 * ctx->num_sms)}));
    a.row_blocks = static_cast<unsigned int>((1LL * rows->rows + a.rows_per_block - 1) / a.rows_per_block);
    const unsigned int checkers = static_cast<unsigned int>((1LL * rows->sequences + kvp::kCheckedStarts - 1) / kvp::kCheckedStarts);
    auto launch = [&](auto kernel) { return launch_chained(ctx, kernel, dim3(a.row_blocks + checkers), dim3(threads), 0, a); };
    auto launch_kind = [&](auto type) {
        using T = decltype(type);
        switch (pages->kind) {
            case GPTB200_KV_E4M3: return sixteens ? launch(kvp::kv_rows_kernel<T, kvp::KIND_E4M3, WRITE, 2>) : launch(kvp::kv_rows_kernel<T, kvp::KIND_E4M3, WRITE, 1>);
            case GPTB200_KV_F32: return sixteens ? launch(kvp::kv_rows_kernel<T, kvp::KIND_F32, WRITE, 2>) : launch(kvp::kv_rows_kernel<T, kvp::KIND_F32, WRITE, 1>);
            default: return sixteens ? launch(kvp::kv_rows_kernel<T, kvp::KIND_BF16, WRITE, 2>) : launch(kvp::kv_rows_kernel<T, kvp::KIND_BF16, WRITE, 1>);
        }
    };
    CUDA_TRY(ctx, dtype == GPTB200_DTYPE_F32 ? launch_kind(float()) : launch_kind(__nv_bfloat16()));
    ctx->launches++;
    return GPTB200_OK;
}

// Which kernel attends, and how its grid is made; host logic.
struct PagedPlan {
    int kernel;       // 0: nothing to do, 1 few rows on mma.sync, 2 prompts on tcgen05, 3 / 4 single / 16 or 32 rows on FMAs
    int tile_rows, per_sm, most_blocks, part_floats;

    // of the grid: per_sm on every SM, as far as the kernel has room for the parts of a tile
    int blocks(int sms) const { return static_cast<int>(std::min<long long>(1LL * sms * per_sm, most_blocks)); }
    size_t scratch(int sms) const { return size_t(2) * blocks(sms) * part_floats * sizeof(float); }
};
enum { PAGED_NONE = 0, PAGED_TOKENS = 1, PAGED_PROMPT = 2, PAGED_FEW = 3, PAGED_ROWS = 4 };

// max_rows: of a head, for a sequence; all_rows: of all heads and sequences
PagedPlan plan_paged(int dtype, int kind, long long max_rows, long long all_rows)
{
    const bool codes = kind == GPTB200_KV_E4M3;
    if (dtype == GPTB200_DTYPE_F32 || kind == GPTB200_KV_F32) {
        // a row at a time: 4 sequences of 1024, 12 heads of 64, 2 / 4 / 8 rows a head: 21 / 21 / 28 us, 32 of 4096, 8 heads of 128, 4 / 8 / 16 rows: 396 / 373 / 671 us;
        // sixteen at a time 26 / 27 / 30 us and 394 / 364 / 453 us
        if (max_rows <= 8) return {PAGED_FEW, 1, kvp::kFewPerSm, kvp::kFewBlocks, kvp::kTokensPart};
        // four or eight rows a warp, in us, 16 sequences of 2048: 10 / 32 rows a head 36 / 48 against 46 / 54, 64 / 128 rows (3016 / 5488 in all) 99 / 169 against 89 / 142;
        // 2000 rows 909 against 663; but with 2124 in all, 100 a head at most, 32 against 43: too few tiles
        const int each = max_rows > 32 && all_rows >= 2560 ? 8 : 4;
        return {PAGED_ROWS, kvp::rows_tile(each), kvp::kRowsPerSm, kvp::kRowsBlocks, kvp::rows_part(each)};
    }
    // 16 sequences of 4096, 8 heads of 128, in us: bf16, 32 / 40 / 48 rows a head: streamed 64 / 69 / 78, prompt 67 / 68 / 63; e4m3, 64 / 96 rows: 109 / 142 against 151 / 148
    // (by rows alone, whatever there is to do: with 2 sequences, 64 rows, the streamed kernel takes 27 against 40 and 31 against 53)
    if (max_rows > (codes ? 96 : 40)) return {PAGED_PROMPT, kvp::kPromptRows, 1, kPagedTickets / 2, kvp::kPromptPart};
    // tiles of eight or sixteen rows: bf16, 12 / 16 rows: 46 / 55 against 49 / 50; e4m3, 16 / 32 rows: 47 / 72 against 48 / 65
    return {PAGED_TOKENS, max_rows <= (codes ? 16 : 12) ? 8 : 16, kvp::tokens_per_sm(codes), kvp::tokens_blocks(codes), kvp::kTokensPart};
}

int check_attention(gptb200_ctx *ctx, int dtype, int heads, const gptb200_kv_pages *pages, const gptb200_kv_rows *rows, float scale, float cap, int window, int sinks, kvp::Attention *a)
{
    if (dtype != GPTB200_DTYPE_BF16 && dtype != GPTB200_DTYPE_F32) return fail(ctx, GPTB200_ERR_INVALID_ARG, "dtype %d is unknown", dtype);
    const int rc = check_pages(ctx, pages, rows, &a->pages, &a->batch);
    if (rc != GPTB200_OK) return rc;
    if (heads <= 0 || heads % pages->kv_heads) return fail(ctx, GPTB200_ERR_INVALID_ARG, "%d heads are not a multiple of the cache's %d", heads, pages->kv_heads);
    if (!(scale > 0.0f) || !std::isfinite(scale) || !(cap >= 0.0f) || !std::isfinite(cap) || window < 0 || sinks < 0)
        return fail(ctx, GPTB200_ERR_INVALID_ARG, "scale %g, cap %g, window %d, first tokens %d", scale, cap, window, sinks);
    // the kernels' factors: scores in base 2, scores over the cap
    if (!std::isfinite(scale * kLog2e) || (cap > 0.0f && (!std::isfinite(cap * kLog2e) || !std::isnormal(scale / cap))))
        return fail(ctx, GPTB200_ERR_INVALID_ARG, "scale %g and cap %g, or their quotient, leave the range of fp32", scale, cap);
    if (1LL * heads * pages->dim > INT_MAX / 64 || 1LL * rows->rows * heads > INT_MAX - 256)
        return fail(ctx, GPTB200_ERR_TOO_LARGE, "%d rows of %lld elements", rows->rows, 1LL * heads * pages->dim);
    a->heads = heads;
    a->share = heads / pages->kv_heads;
    a->shares = kvp::divisor(a->share);
    a->scale = scale;
    a->cap = cap;
    a->window = window >= a->batch.capacity ? 0 : window;   // no sequence is longer: it hides nothing
    a->sinks = a->window ? sinks : 0;
    return GPTB200_OK;
}

static_assert(kvp::kFewBlocks <= kPagedTickets && kvp::kRowsBlocks <= kPagedTickets && kvp::tokens_blocks(true) <= kPagedTickets && kvp::tokens_blocks(false) <= kPagedTickets);

// A kernel that cuts the line of work into equal ranges, a part of a tile in scratch for either end of a range.
template <typename Args>
int run_line(gptb200_ctx *ctx, const PagedPlan &plan, void (*kernel)(Args), Args &args, int threads, int smem)
{
    const void *key = reinterpret_cast<const void *>(kernel);
    if (!ctx->configured.count(key)) {
        CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        ctx->configured.insert(key);
    }
    const int sms = ctx->max_sms > 0 ? std::min(ctx->max_sms, ctx->num_sms) : ctx->num_sms;
    const int rc = ensure_workspace(ctx, plan.scratch(sms));
    if (rc != GPTB200_OK) return rc;
    args.parts = {ctx->ws, ctx->d_paged_tickets, plan.part_floats};
    args.cut.tile_rows = plan.tile_rows;
    CUDA_TRY(ctx, launch_chained(ctx, kernel, dim3(plan.blocks(sms)), dim3(threads), smem, args));
    ctx->launches++;
    return GPTB200_OK;
}

template <int D16, bool CODES, int NT>
int run_tokens(gptb200_ctx *ctx, const PagedPlan &plan, kvp::TokensArgs &args)
{
    return run_line(ctx, plan, kvp::paged_tokens_kernel<D16, CODES, NT>, args, kvp::kTokensThreads, kvp::TokensShape<D16, CODES, NT>::kSmem);
}

template <int D16>
int run_tokens(gptb200_ctx *ctx, const PagedPlan &plan, kvp::TokensArgs &args, bool codes)
{
    if (codes) return plan.tile_rows == 8 ? run_tokens<D16, true, 1>(ctx, plan, args) : run_tokens<D16, true, 2>(ctx, plan, args);
    return plan.tile_rows == 8 ? run_tokens<D16, false, 1>(ctx, plan, args) : run_tokens<D16, false, 2>(ctx, plan, args);
}

int attention_tokens(gptb200_ctx *ctx, const PagedPlan &plan, const kvp::Attention &a, int kind)
{
    kvp::TokensArgs args{a, {}, {0, kvp::kTokensKeys, 1, 5}};
    const bool codes = kind == GPTB200_KV_E4M3;
    switch ((a.pages.dim + 31) / 32) {
        case 1: return run_tokens<2>(ctx, plan, args, codes);
        case 2: return run_tokens<4>(ctx, plan, args, codes);
        case 3: return run_tokens<6>(ctx, plan, args, codes);
        default: return run_tokens<8>(ctx, plan, args, codes);
    }
}

template <typename T, int KIND>
int run_fma(gptb200_ctx *ctx, const PagedPlan &plan, const kvp::Attention &a)
{
    kvp::TokensArgs args{a, {}, {0, kvp::kFewKeys, 1, 5}};
    if (plan.kernel == PAGED_FEW) return run_line(ctx, plan, kvp::paged_few_kernel<T, KIND>, args, kvp::kTokensThreads, kvp::kFewSmem);
    args.cut.keys = kvp::kRowsKeys;
    return plan.tile_rows == kvp::rows_tile(4) ? run_line(ctx, plan, kvp::paged_rows_kernel<T, KIND, 4>, args, kvp::kTokensThreads, kvp::rows_smem(4))
                                               : run_line(ctx, plan, kvp::paged_rows_kernel<T, KIND, 8>, args, kvp::kTokensThreads, kvp::rows_smem(8));
}

template <int NB, bool CODES, bool CAPPED>
int run_prompt(gptb200_ctx *ctx, const PagedPlan &plan, kvp::PromptArgs &args)
{
    return run_line(ctx, plan, args.a.lse ? kvp::paged_prompt_kernel<NB, CODES, CAPPED, true> : kvp::paged_prompt_kernel<NB, CODES, CAPPED, false>, args, kvp::kPromptThreads,
                    kvp::PromptShape<NB>::kSmem);
}

template <int NB>
int run_prompt(gptb200_ctx *ctx, const PagedPlan &plan, kvp::PromptArgs &args, bool codes)
{
    if (args.a.cap > 0.0f) return codes ? run_prompt<NB, true, true>(ctx, plan, args) : run_prompt<NB, false, true>(ctx, plan, args);
    return codes ? run_prompt<NB, true, false>(ctx, plan, args) : run_prompt<NB, false, false>(ctx, plan, args);
}

int attention_prompt(gptb200_ctx *ctx, const PagedPlan &plan, const kvp::Attention &a, int kind)
{
    const bool codes = kind == GPTB200_KV_E4M3;
    kvp::PromptArgs args{};
    args.a = a;
    args.cut = {0, kvp::kPromptKeys, 2, 4};
    args.scale_log2 = a.scale * kLog2e;
    args.cap_log2 = a.cap * kLog2e;
    args.cap_arg = a.cap > 0.0f ? a.scale / a.cap : 0.0f;
    const long long rows = (2LL * a.pages.num_pages * a.pages.kv_heads) << a.pages.page_shift;
    if (!codes && rows > 0 && rows <= INT_MAX) {
        args.box_rows = std::min(1 << a.pages.page_shift, kvp::kPromptKeys);
        const int rc = bf16_operand_map(ctx, &args.map, a.pages.data, rows, a.pages.dim, a.pages.dim, args.box_rows);
        if (rc != GPTB200_OK) return rc;
    }
    return a.pages.dim <= 64 ? run_prompt<1>(ctx, plan, args, codes) : run_prompt<2>(ctx, plan, args, codes);
}

}  // namespace

extern "C" {

int gptb200_kv_pages_write(gptb200_ctx *ctx, const gptb200_kv_pages *pages, const gptb200_kv_rows *rows, const void *k, long long k_pitch, const void *v, long long v_pitch, int dtype)
{
    return run_rows<true>(ctx, const_cast<void *>(k), k_pitch, const_cast<void *>(v), v_pitch, dtype, pages, rows);
}

int gptb200_kv_pages_read(gptb200_ctx *ctx, void *k, long long k_pitch, void *v, long long v_pitch, int dtype, const gptb200_kv_pages *pages, const gptb200_kv_rows *rows)
{
    return run_rows<false>(ctx, k, k_pitch, v, v_pitch, dtype, pages, rows);
}

int gptb200_attention_paged(gptb200_ctx *ctx, void *out, long long out_pitch, float *lse, const void *q, long long q_pitch, int dtype, int heads, const gptb200_kv_pages *pages,
                            const gptb200_kv_rows *rows, float scale, float cap, int window, int sinks)
{
    if (!ctx) return GPTB200_ERR_INVALID_ARG;
    kvp::Attention a{};
    int rc = check_attention(ctx, dtype, heads, pages, rows, scale, cap, window, sinks, &a);
    if (rc != GPTB200_OK) return rc;
    if (rows->sequences == 0 || rows->rows == 0) return GPTB200_OK;
    const long long width = 1LL * heads * pages->dim;
    if ((rc = check_rows(ctx, "q", q, q_pitch, width, dtype)) != GPTB200_OK || (rc = check_rows(ctx, "out", out, out_pitch, width, dtype)) != GPTB200_OK) return rc;
    if (!aligned4(lse)) return fail(ctx, GPTB200_ERR_INVALID_ARG, "lse is not aligned to 4 bytes");
    if (out == q) return fail(ctx, GPTB200_ERR_INVALID_ARG, "out is q");
    OnDevice device;
    CUDA_TRY(ctx, device.enter(ctx->device));
    a.q = q; a.out = out; a.lse = lse; a.q_pitch = q_pitch; a.out_pitch = out_pitch;
    const PagedPlan plan = plan_paged(dtype, pages->kind, 1LL * rows->max_new * a.share, 1LL * rows->rows * a.heads);
    if (plan.kernel == PAGED_PROMPT) return attention_prompt(ctx, plan, a, pages->kind);
    if (plan.kernel == PAGED_TOKENS) return attention_tokens(ctx, plan, a, pages->kind);
    if (dtype == GPTB200_DTYPE_BF16) return run_fma<__nv_bfloat16, kvp::KIND_F32>(ctx, plan, a);
    return pages->kind == GPTB200_KV_E4M3 ? run_fma<float, kvp::KIND_E4M3>(ctx, plan, a)
           : pages->kind == GPTB200_KV_F32 ? run_fma<float, kvp::KIND_F32>(ctx, plan, a) : run_fma<float, kvp::KIND_BF16>(ctx, plan, a);
}

int gptb200_plan_attention_paged(int num_sms, int dtype, int heads, const gptb200_kv_pages *pages, const gptb200_kv_rows *rows, float scale, float cap, int window, int sinks, int *plan4)
{
    if (num_sms <= 0 || !plan4) return GPTB200_ERR_INVALID_ARG;
    kvp::Attention a{};
    const int rc = check_attention(nullptr, dtype, heads, pages, rows, scale, cap, window, sinks, &a);
    if (rc != GPTB200_OK) return rc;
    PagedPlan plan{};
    if (rows->sequences > 0 && rows->rows > 0) plan = plan_paged(dtype, pages->kind, 1LL * rows->max_new * a.share, 1LL * rows->rows * a.heads);
    const int out[4] = {plan.kernel, plan.tile_rows, plan.blocks(num_sms), static_cast<int>(plan.scratch(num_sms) >> 10)};
    for (int i = 0; i < 4; ++i) plan4[i] = out[i];
    return GPTB200_OK;
}

}  // extern "C"
