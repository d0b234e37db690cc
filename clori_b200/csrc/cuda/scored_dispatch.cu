// Checks, kernel selection and split planning of scored attention.
#include "scored.cuh"

namespace yvx {

static int scored_refuse(int code, const char *text)
{
    yvx_cuda_set_error_text(text);
    return code;
}

// Tokens a call's rows can see, as far as the host knows: a causal window bounds them.
static unsigned long long scored_span(const yvx_scored_problem *p)
{
    const unsigned long long all = ((unsigned long long)p->kv_tokens_max + 63ull) / 64ull * 64ull;
    if (!p->window || !p->causal || p->row_end) return all;
    const unsigned long long seen = (unsigned long long)p->window + p->query_rows + 62ull;
    return seen < all ? (seen + 63ull) / 64ull * 64ull : all;
}

static int scored_check(const yvx_scored_problem *p)
{
    if (!p || !p->query || !p->output || !p->key || !p->value || !p->status)
        return scored_refuse(YVEX_ERR_INVALID_ARG, "scored attention: query, output, key, value and status are required");
    if (!p->sessions || !p->query_rows || !p->query_heads || !p->kv_heads || !p->head_dim ||
        p->query_heads % p->kv_heads || !p->kv_tokens_max || (!p->kv_tokens && p->kv_tokens_uniform > p->kv_tokens_max) ||
        !(p->scale > 0.0f) || !isfinite(p->scale) || !(p->cap >= 0.0f) || !isfinite(p->cap) ||
        (p->cap > 0.0f && (p->cap < 1e-30f || !isfinite(4.0f * p->scale / p->cap))))
        return scored_refuse(YVEX_ERR_INVALID_ARG, "scored attention: inconsistent geometry, scale or cap");
    if (p->head_dim > 256u || (p->query_dtype != YVEX_DTYPE_F32 && p->query_dtype != YVEX_DTYPE_BF16) ||
        (p->output_dtype != YVEX_DTYPE_F32 && p->output_dtype != YVEX_DTYPE_BF16) || p->kv_code < YVX_KV_PLAIN ||
        p->kv_code > YVX_KV_I8 ||
        (p->kv_code == YVX_KV_PLAIN && p->kv_dtype != YVEX_DTYPE_F32 && p->kv_dtype != YVEX_DTYPE_BF16))
        return scored_refuse(YVEX_ERR_UNSUPPORTED, "scored attention: head_dim above 256 or a type it does not read");
    if (p->kv_code != YVX_KV_PLAIN && (!p->block_table || !p->key_scales || !p->value_scales))
        return scored_refuse(YVEX_ERR_INVALID_ARG, "scored attention: codes need a block table and scales");
    if (p->block_table && (!p->block_tokens || !p->pool_blocks || p->pool_blocks > 0x7fffffffu ||
                           (unsigned long long)p->block_table_stride * p->block_tokens < p->kv_tokens_max))
        return scored_refuse(YVEX_ERR_INVALID_ARG, "scored attention: the block table does not cover kv_tokens_max");
    if (!p->chunk_tokens || (p->chunk_tokens & 63u) || !p->max_splits)
        return scored_refuse(YVEX_ERR_INVALID_ARG, "scored attention: yvx_cuda_scored_plan has not been called");
    if (p->kv_tokens_max > 0x7fffffffu - 1024u || p->sessions > 65535u || p->max_splits > 8192u)
        return scored_refuse(YVEX_ERR_BOUNDS, "scored attention: lengths below 2^31 - 1024, at most 65535 sessions and 8192 splits");
    // what the kernels' grids hold, whichever of them runs: refused before the first is enqueued
    const unsigned long long vectors = (unsigned long long)p->query_rows * (p->query_heads / p->kv_heads);
    if ((vectors + 15ull) / 16ull * p->kv_heads > 0x7fffffffull ||
        (p->max_splits > 1u && (unsigned long long)p->sessions * p->query_rows > 0x7fffffffull / p->query_heads))
        return scored_refuse(YVEX_ERR_BOUNDS, "scored attention: more rows and heads than a grid holds");
    if ((unsigned long long)p->chunk_tokens * p->max_splits < scored_span(p))
        return scored_refuse(YVEX_ERR_INVALID_ARG, "scored attention: the splits do not cover the tokens: planned for another call");
    return 0;
}

// The sessions of `whole` from `begin` on, `count` of them, as a call of their own.
static yvx_scored_problem scored_group(const yvx_scored_problem &whole, unsigned int begin, unsigned int count)
{
    yvx_scored_problem p = whole;
    const unsigned long long rows = (unsigned long long)begin * whole.query_rows, items = rows * whole.query_heads;
    p.sessions = count;
    p.query = static_cast<const unsigned char *>(whole.query) +
              (unsigned long long)begin * whole.query_session_stride * (whole.query_dtype == YVEX_DTYPE_BF16 ? 2ull : 4ull);
    p.output = static_cast<unsigned char *>(whole.output) + items * whole.head_dim * (whole.output_dtype == YVEX_DTYPE_BF16 ? 2ull : 4ull);
    p.block_table = whole.block_table + (unsigned long long)begin * whole.block_table_stride;
    if (whole.kv_tokens) p.kv_tokens += begin;
    if (whole.query_start) p.query_start += begin;
    if (whole.row_first) p.row_first += rows;
    if (whole.row_end) p.row_end += rows;
    if (whole.workspace)
        p.workspace = static_cast<unsigned char *>(whole.workspace) + items * whole.max_splits * (whole.head_dim + 4ull) * sizeof(float);
    return p;
}

// Caches that the tensor-core kernel does not read in place: codes, and pages that are no multiple of 64 tokens.
static bool scored_needs_stage(const yvx_scored_problem *p)
{
    return p->kv_code != YVX_KV_PLAIN || (p->block_table && p->block_tokens % 64u);
}

// Calls of more than 32 vectors (query rows x heads of a KV head) on the shapes of the tensor cores, of more than 64
// where the cache has to be staged first. One session of 131072 tokens, 8 KV heads, groups of 4, the decode kernel
// against this one: 8 rows 103 / 101 us, 12 rows 153 / 101, 16 rows 177 / 102; with e4m3 codes 16 rows 182 / 253,
// 32 rows about 360 / 256. Decided by the shape, types and alignment alone, before the plan.
static bool scored_prompt_shape(const yvx_scored_problem *p)
{
    const unsigned long long bytes = p->kv_code == YVX_KV_PLAIN ? 2ull : 1ull;
    const unsigned long long strides = p->key_token_stride | p->value_token_stride | p->key_head_stride | p->value_head_stride |
                                       p->key_outer_stride | p->value_outer_stride;
    const unsigned long long q_strides = p->query_row_stride | p->query_session_stride | p->query_head_stride;
    return !p->force_general && p->head_dim == 128u && p->query_dtype == YVEX_DTYPE_BF16 &&
           (p->kv_code != YVX_KV_PLAIN || p->kv_dtype == YVEX_DTYPE_BF16) &&
           (unsigned long long)p->query_rows * (p->query_heads / p->kv_heads) > (scored_needs_stage(p) ? 64ull : 32ull) &&
           // that kernel holds the mask, and the bias, in units of the raw product unless a cap comes between
           ((p->cap > 0.0f && !p->slopes) || (p->scale >= 1e-12f && p->scale <= 1e12f)) &&
           p->cap <= 1e36f &&                     // and the cap in log2 units
           !((reinterpret_cast<uintptr_t>(p->key) | reinterpret_cast<uintptr_t>(p->value) |
              reinterpret_cast<uintptr_t>(p->query) | reinterpret_cast<uintptr_t>(p->output) | strides * bytes | q_strides * 2ull) & 15ull);
}

// Partial rows of all splits, a multiple of 256 bytes; staged rows lie behind them.
static unsigned long long scored_partial_bytes(const yvx_scored_problem *p)
{
    if (p->max_splits <= 1u) return 0ull;
    const unsigned long long items = (unsigned long long)p->sessions * p->query_rows * p->query_heads;
    return (items * p->max_splits * (p->head_dim + 4ull) * 4ull + 255ull) / 256ull * 256ull;
}

}  // namespace yvx

extern "C" {

// Splits fill the machine: two CTAs of the split kernels run on an SM, so a wave is 2 * sm_count items. Every
// wave costs its chunk's tiles of 64 tokens and about four tiles more (start, first data, merge of the warps,
// partial rows); the chunk with the smallest sum is taken, at most 8192 tokens. One session of 4096 tokens:
// 128 tokens 10.3 us, 64 tokens 15.4, 512 tokens 13.0; 64 sessions behind a window of 4096: one chunk 177 us,
// two 193, four 190; one session of 131072 tokens: 3584 (one wave) 95 us, 1792 107, 4096 105.
// Prompt-sized calls are split only to fill the machine: one CTA on an SM, a piece of work is two row tiles, a split
// costs its tiles of 128 tokens and about five more, the fold two tiles and its traffic. 32 heads in groups of 4 over
// 131072 tokens, 20 rows: one split 1307 us, four 348, sixteen 108, eighteen (taken) 102, twenty-four 143; 256 rows:
// 1565, four 490, nine (taken) 479, sixteen 582; 2048 rows over 16384: one (taken) 440, two 679.
void yvx_cuda_scored_plan(yvx_scored_problem *p, int sm_count)
{
    if (!p || !p->kv_heads || !p->query_rows || !p->kv_tokens_max) return;
    const unsigned long long wave = 2ull * (unsigned long long)(sm_count > 0 ? sm_count : 148);
    const unsigned long long vectors = (unsigned long long)p->query_rows * (p->query_heads / p->kv_heads);
    const unsigned long long span = yvx::scored_span(p);
    const unsigned long long lanes = (unsigned long long)p->sessions * p->kv_heads * ((vectors + 15ull) / 16ull);
    unsigned long long best = span, best_cost = ~0ull;
    if (yvx::scored_prompt_shape(p)) {
        const unsigned long long heads = yvx::scored_packed_heads(*p), rows = 2ull * (128ull / heads);   // of a piece of work
        const unsigned long long together = yvx::scored_needs_stage(p) ? yvx::scored_stage_sessions(*p) : p->sessions;
        const unsigned long long pieces = together * (p->query_heads / heads) * ((p->query_rows + rows - 1ull) / rows);
        const unsigned long long moved = together * p->query_rows * p->query_heads * 1056ull;
        for (unsigned long long splits = 1ull; splits <= (span + 127ull) / 128ull && splits <= 8192ull; ++splits) {
            const unsigned long long tiles = ((span + 127ull) / 128ull + splits - 1ull) / splits;
            const unsigned long long cost = (pieces * splits + wave / 2ull - 1ull) / (wave / 2ull) * (tiles + 5ull) +
                                            (splits > 1ull ? 2ull + splits * moved / (8ull << 20) : 0ull);
            if (cost < best_cost) {
                best_cost = cost;
                best = splits > 1ull ? tiles * 128ull : span;
            }
            if (pieces * splits >= 2ull * wave) break;
        }
    } else if (vectors <= 64ull || lanes < wave) {
        for (unsigned long long chunk = 64ull; chunk <= 8192ull; chunk += 64ull) {
            const unsigned long long splits = (span + chunk - 1ull) / chunk;
            const unsigned long long cost = (lanes * splits + wave - 1ull) / wave * (4ull + chunk / 64ull);
            if (splits <= 8192ull && cost < best_cost) {
                best_cost = cost;
                best = chunk;
            }
            if (splits == 1ull) break;
        }
        while ((span + best - 1ull) / best > 8192ull) best += 64ull;
    }
    p->chunk_tokens = (unsigned int)best;
    p->max_splits = (unsigned int)((span + best - 1ull) / best);
}

unsigned long long yvx_cuda_scored_workspace_bytes(const yvx_scored_problem *p)
{
    if (!p || !p->kv_heads || !p->query_rows || !p->kv_tokens_max) return 0ull;
    return yvx::scored_partial_bytes(p) +
           (yvx::scored_prompt_shape(p) && yvx::scored_needs_stage(p) ? yvx::scored_stage_bytes(*p) : 0ull);
}

int yvx_cuda_scored_attention(const yvx_scored_problem *p, void *stream, unsigned int *launches)
{
    if (launches) *launches = 0u;
    int rc = yvx::scored_check(p);
    if (rc != 0) return rc;
    if (yvx::scored_prompt_shape(p) && yvx::scored_needs_stage(p) && p->kv_heads > 65535u)
        return yvx::scored_refuse(YVEX_ERR_BOUNDS, "scored attention: more than 65535 KV heads over codes or small pages");
    const unsigned long long needed = yvx_cuda_scored_workspace_bytes(p);
    if (needed && (!p->workspace || p->workspace_bytes < needed || (reinterpret_cast<uintptr_t>(p->workspace) & 255u)))
        return yvx::scored_refuse(YVEX_ERR_BOUNDS, "scored attention: the workspace is missing, misaligned or too small");
    cudaStream_t s = (cudaStream_t)stream;
    unsigned int count = 0u;
    rc = 0;  // specialised kernels answer 1 when they took the call, 0 when its shape is not theirs
    if (yvx::scored_prompt_shape(p)) {
        if (yvx::scored_needs_stage(p)) {
            unsigned char *rows = static_cast<unsigned char *>(p->workspace) + yvx::scored_partial_bytes(p);
            const unsigned int together = yvx::scored_stage_sessions(*p);
            for (unsigned int begin = 0; begin < p->sessions; begin += together) {
                const yvx_scored_problem group = yvx::scored_group(*p, begin, p->sessions - begin < together ? p->sessions - begin : together);
                yvx_scored_problem staged;
                rc = yvx::scored_stage_launch(group, rows, &staged, s);
                if (rc == 0) rc = yvx::scored_prompt_launch(staged, true, s);
                if (rc == 0) rc = yvx::scored_general_launch(group, s);
                if (rc < 0) return rc;
                count += 2u;
            }
            --count;   // the last one is counted below
            rc = 1;
        } else {
            rc = yvx::scored_prompt_launch(*p, false, s);
        }
    } else if (!p->force_general && (unsigned long long)p->query_rows * (p->query_heads / p->kv_heads) <= 64ull) {
        rc = yvx::scored_decode_launch(*p, s);
    }
    if (rc == 0) rc = yvx::scored_general_launch(*p, s);
    else if (rc > 0) rc = 0;
    if (rc != 0) return rc;
    ++count;
    if (p->max_splits > 1u) {
        rc = yvx::scored_combine_launch(*p, s);
        if (rc != 0) return rc;
        ++count;
    }
    if (launches) *launches = count;
    return 0;
}

}  // extern "C"
