/* Scored attention, the 8-bit cache and page copies at the operator level: argument checks against
 * the tensors' bytes, then one call into the shim each. The reference has no counterpart of any;
 * status codes follow the operators beside them (batch_attention.c, latent_ops.c). */
#include "private.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

static const unsigned long long max_tokens = 0x7fffffffull - 1024ull;

static int view_ok(const yvex_backend *backend, const yvex_device_tensor *tensor, yvex_dtype dtype,
                   unsigned long long elements)
{
    unsigned long long bytes;
    return yvx_tensor_owned(backend, tensor) && tensor->dtype == dtype &&
           yvx_u64_mul(elements, yvx_dtype_bytes(dtype), &bytes) && tensor->bytes >= bytes;
}

static int float_type(yvex_dtype dtype) { return dtype == YVEX_DTYPE_F32 || dtype == YVEX_DTYPE_BF16; }

/* (count - 1) * stride added to *extent; 0 on overflow. */
static int extend(unsigned long long count, unsigned long long stride, unsigned long long *extent)
{
    unsigned long long span;
    return count && yvx_u64_mul(count - 1ull, stride, &span) && yvx_u64_add(*extent, span, extent);
}

static int finish(yvex_backend *backend, yvex_backend_operation_facts *facts, unsigned int launches,
                  unsigned long long temporary, const char *where, yvex_error *err)
{
    facts->kernel_launches = launches;
    facts->temporary_bytes = temporary;
    facts->compulsory_memory_facts_available = 1;
    if (backend->synchronous) return yvx_backend_status_collect(backend, facts, where, err);
    backend->status_pending = 1;
    return YVEX_OK;
}

/* A refusal of the shim leaves the device as it was; a launch error is the backend's failure. */
static int shim_failed(yvex_backend *backend, int rc, const char *where, yvex_error *err)
{
    return rc == YVEX_ERR_BACKEND ? yvx_backend_device_fail(backend, rc, where, err)
                                  : yvx_fail(err, (yvex_status)rc, where, yvx_cuda_last_error_text());
}

int yvex_b200_attention_scored_execute(yvex_backend *backend, const yvex_b200_attention_scored_request *r,
                                       yvex_backend_operation_facts *facts, yvex_error *err)
{
    const char *where = "b200.attention.scored";
    unsigned long long query_width, kv_width, rows, elements, extent, token_stride, head_stride, outer_stride;
    unsigned long long workspace, element, pages, pages_value;
    yvex_dtype kv_dtype;
    yvx_scored_problem p;
    unsigned int launches = 0u;
    void *scratch = NULL;
    int rc, paged, codes;
    if (!r || !facts || !r->query || !r->key || !r->value || !r->kv_tokens || !r->output)
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "query, key, value, lengths, output and result facts are required");
    memset(facts, 0, sizeof(*facts));
    if (!r->session_count || !r->query_tokens || !r->query_heads || !r->key_value_heads || !r->head_dimension ||
        !r->key_value_tokens || r->query_heads % r->key_value_heads || !(r->scale >= 0.0f) || !isfinite(r->scale) ||
        !(r->score_cap >= 0.0f) || !isfinite(r->score_cap) ||
        !yvx_u64_mul(r->query_heads, r->head_dimension, &query_width) ||
        !yvx_u64_mul(r->key_value_heads, r->head_dimension, &kv_width) ||
        !yvx_u64_mul(r->session_count, r->query_tokens, &rows) ||
        (r->query_token_stride && r->query_token_stride < query_width))
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "complete scored attention geometry is required");
    codes = r->kv_code != YVX_KV_PLAIN;
    paged = r->kv_layout == YVEX_B200_KV_BLOCK_TABLE;
    kv_dtype = r->key->dtype;
    if (r->kv_code < YVX_KV_PLAIN || r->kv_code > YVX_KV_I8 || r->head_dimension > 256ull || !float_type(r->query->dtype) ||
        !float_type(r->output->dtype) || r->value->dtype != kv_dtype || (codes ? kv_dtype != YVEX_DTYPE_I8 : !float_type(kv_dtype)) ||
        (!paged && (r->kv_layout != YVEX_B200_KV_CONTIGUOUS || codes)))
        return yvx_fail(err, YVEX_ERR_UNSUPPORTED, where, "unsupported head dimension, layout, code or dtype combination");
    if (r->session_count > 0xffffull || r->query_tokens > max_tokens || r->key_value_tokens > max_tokens ||
        r->query_heads > 0xffffffull || r->window > 0xffffffffull)
        return yvx_fail(err, YVEX_ERR_BOUNDS, where, "sessions, rows, tokens or heads beyond the launch limits");
    rc = yvx_backend_admit(backend, where, err);
    if (rc != YVEX_OK) return rc;

    element = yvx_dtype_bytes(kv_dtype);
    memset(&p, 0, sizeof(p));
    if (paged) {
        if (!r->block_table || !r->block_tokens || r->block_tokens > max_tokens || !r->max_blocks_per_session ||
            r->max_blocks_per_session > 0xffffffffull ||
            (r->key_value_tokens + r->block_tokens - 1ull) / r->block_tokens > r->max_blocks_per_session ||
            (codes && (!r->key_scales || !r->value_scales)))
            return yvx_fail(err, YVEX_ERR_INVALID_ARG, where,
                            "a block table covering the longest session (and scales for codes) is required");
        token_stride = r->kv_token_stride ? r->kv_token_stride : codes ? r->head_dimension : kv_width;
        if (!yvx_u64_mul(r->block_tokens, codes ? r->head_dimension : 0ull, &head_stride)) head_stride = 0ull;
        head_stride = r->kv_head_stride ? r->kv_head_stride : codes ? head_stride : r->head_dimension;
        extent = r->head_dimension;
        if (!extend(r->block_tokens, token_stride, &extent) || !extend(r->key_value_heads, head_stride, &extent) ||
            (!r->kv_outer_stride && !yvx_u64_mul(r->block_tokens, kv_width, &elements)))
            return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "page strides overflow");
        outer_stride = r->kv_outer_stride ? r->kv_outer_stride : elements;
        if (outer_stride < extent)
            return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "kv_outer_stride does not hold a page");
        pages = yvx_tensor_owned(backend, r->key) ? r->key->bytes / element / outer_stride : 0ull;
        pages_value = yvx_tensor_owned(backend, r->value) ? r->value->bytes / element / outer_stride : 0ull;
        if (pages_value < pages) pages = pages_value;
        if (codes && yvx_tensor_owned(backend, r->key_scales) && yvx_tensor_owned(backend, r->value_scales)) {
            const unsigned long long a = r->key_scales->bytes / sizeof(float) / r->key_value_heads;
            const unsigned long long b = r->value_scales->bytes / sizeof(float) / r->key_value_heads;
            if (a < pages) pages = a;
            if (b < pages) pages = b;
        }
        if (!pages || pages > 0x7fffffffull || !yvx_u64_mul(r->session_count, r->max_blocks_per_session, &elements) ||
            !view_ok(backend, r->block_table, YVEX_DTYPE_I32, elements) ||
            (codes && (!view_ok(backend, r->key_scales, YVEX_DTYPE_F32, r->key_value_heads) ||
                       !view_ok(backend, r->value_scales, YVEX_DTYPE_F32, r->key_value_heads))))
            return yvx_fail(err, YVEX_ERR_FORMAT, where, "pools, scales and block table do not hold the declared geometry");
        p.block_table = (const int *)r->block_table->data;
        p.block_tokens = (unsigned int)r->block_tokens;
        p.block_table_stride = (unsigned int)r->max_blocks_per_session;
        p.pool_blocks = (unsigned int)pages;
    } else {
        token_stride = r->kv_token_stride ? r->kv_token_stride : kv_width;
        head_stride = r->kv_head_stride ? r->kv_head_stride : r->head_dimension;
        outer_stride = r->kv_outer_stride;
        if (r->session_count > 1ull && !outer_stride)
            return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "kv_outer_stride is required for more than one contiguous session");
        extent = r->head_dimension;
        if (!extend(r->key_value_tokens, token_stride, &extent) || !extend(r->key_value_heads, head_stride, &extent) ||
            !extend(r->session_count, outer_stride, &extent))
            return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "key and value strides overflow");
        if (!view_ok(backend, r->key, kv_dtype, extent) || !view_ok(backend, r->value, kv_dtype, extent))
            return yvx_fail(err, YVEX_ERR_FORMAT, where, "key and value views do not hold the declared geometry");
    }
    p.query_row_stride = r->query_token_stride ? r->query_token_stride : query_width;
    extent = query_width;
    if (!extend(rows, p.query_row_stride, &extent) || !view_ok(backend, r->query, r->query->dtype, extent) ||
        !r->query->is_written || !yvx_u64_mul(rows, query_width, &elements) ||
        !view_ok(backend, r->output, r->output->dtype, elements) ||
        !view_ok(backend, r->kv_tokens, YVEX_DTYPE_I32, r->session_count) ||
        (r->query_start && !view_ok(backend, r->query_start, YVEX_DTYPE_I32, r->session_count)) ||
        (r->row_first && !view_ok(backend, r->row_first, YVEX_DTYPE_I32, rows)) ||
        (r->row_end && !view_ok(backend, r->row_end, YVEX_DTYPE_I32, rows)) ||
        (r->slopes && !view_ok(backend, r->slopes, YVEX_DTYPE_F32, r->query_heads)))
        return yvx_fail(err, YVEX_ERR_FORMAT, where, "bounded query, output, length, range and slope views are required");

    p.sessions = (unsigned int)r->session_count;
    p.query_rows = (unsigned int)r->query_tokens;
    p.query_heads = (unsigned int)r->query_heads;
    p.kv_heads = (unsigned int)r->key_value_heads;
    p.head_dim = (unsigned int)r->head_dimension;
    p.causal = r->causal != 0;
    p.scale = r->scale > 0.0f ? r->scale : 1.0f / sqrtf((float)r->head_dimension);
    p.cap = r->score_cap;
    p.window = (unsigned int)r->window;
    p.query_dtype = r->query->dtype;
    p.kv_dtype = kv_dtype;
    p.output_dtype = r->output->dtype;
    p.kv_code = r->kv_code;
    p.query = r->query->data;
    p.query_session_stride = p.query_row_stride * r->query_tokens;
    p.output = r->output->data;
    p.key = r->key->data;
    p.value = r->value->data;
    p.key_token_stride = p.value_token_stride = token_stride;
    p.key_head_stride = p.value_head_stride = head_stride;
    p.key_outer_stride = p.value_outer_stride = outer_stride;
    if (codes) {
        p.key_scales = (const float *)r->key_scales->data;
        p.value_scales = (const float *)r->value_scales->data;
    }
    p.kv_tokens = (const unsigned int *)r->kv_tokens->data;
    p.kv_tokens_max = (unsigned int)r->key_value_tokens;
    if (r->query_start)
        p.query_start = (const unsigned int *)r->query_start->data;
    else
        p.query_start_from_end = 1u;
    p.row_first = r->row_first ? (const int *)r->row_first->data : NULL;
    p.row_end = r->row_end ? (const int *)r->row_end->data : NULL;
    p.slopes = r->slopes ? (const float *)r->slopes->data : NULL;
    p.status = backend->status_device;
    yvx_cuda_scored_plan(&p, backend->sm_count);
    workspace = yvx_cuda_scored_workspace_bytes(&p);
    rc = yvx_backend_scratch(backend, workspace, &scratch, where, err);
    if (rc != YVEX_OK) return rc;
    p.workspace = scratch;
    p.workspace_bytes = workspace;
    rc = yvx_backend_status_join(backend, where, err);
    if (rc != YVEX_OK) return rc;
    rc = yvx_cuda_scored_attention(&p, backend->stream, &launches);
    if (rc != 0) return shim_failed(backend, rc, where, err);
    facts->activation_bytes = rows * p.query_row_stride * yvx_dtype_bytes(r->query->dtype) +
                              rows * query_width * yvx_dtype_bytes(r->output->dtype);
    rc = finish(backend, facts, launches, workspace, where, err);
    if (rc != YVEX_OK) return rc;
    r->output->is_written = 1;
    yvex_error_clear(err);
    return YVEX_OK;
}

int yvex_b200_attention_row_ranges(const unsigned long long *document_lengths, const unsigned long long *prefix_lengths,
                                   unsigned long long documents, unsigned long long query_start,
                                   unsigned long long rows, int *row_first, int *row_end)
{
    unsigned long long d, row = 0ull, start = 0ull, end, last;
    if ((documents && !document_lengths) || !rows || !row_first || !row_end ||
        !yvx_u64_add(query_start, rows, &last) || last > max_tokens)
        return 0;
    for (d = 0ull; d < documents; ++d) {
        unsigned long long prefix = prefix_lengths ? prefix_lengths[d] : 0ull;
        if (!yvx_u64_add(start, document_lengths[d], &end) || end > max_tokens) return 0;
        if (prefix > document_lengths[d]) prefix = document_lengths[d];
        for (; row < rows && query_start + row < end; ++row) {
            const unsigned long long seen = query_start + row + 1ull;
            row_first[row] = (int)start;
            row_end[row] = (int)(seen > start + prefix ? seen : start + prefix);
        }
        start = end;
    }
    for (; row < rows; ++row) row_first[row] = row_end[row] = 0;
    return 1;
}

int yvex_b200_kv8_append_execute(yvex_backend *backend, const yvex_b200_kv8_append_request *r,
                                 yvex_backend_operation_facts *facts, yvex_error *err)
{
    const char *where = "b200.kv8.append";
    unsigned long long kv_width, page_bytes, pages, elements, extent, last;
    const yvex_device_tensor *outputs[4];
    yvx_kv8_append_args a;
    int rc, i;
    if (!r || !facts || !r->key || !r->value || !r->block_table || !r->key_codes || !r->value_codes || !r->key_scales ||
        !r->value_scales)
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "new rows, codes, scales, block table and result facts are required");
    memset(facts, 0, sizeof(*facts));
    if (!r->session_count || !r->token_count || !r->key_value_heads || !r->head_dimension || !r->block_tokens ||
        !r->max_blocks_per_session || !yvx_u64_mul(r->key_value_heads, r->head_dimension, &kv_width) ||
        !yvx_u64_mul(r->block_tokens, kv_width, &page_bytes) || (r->token_stride && r->token_stride < kv_width))
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "sessions, rows, heads and pages must be consistent");
    if ((r->kv_code != YVX_KV_E4M3 && r->kv_code != YVX_KV_I8) || !float_type(r->key->dtype) ||
        r->value->dtype != r->key->dtype || r->head_dimension % 16ull || r->head_dimension > 256ull || r->block_tokens > 256ull)
        return yvx_fail(err, YVEX_ERR_UNSUPPORTED, where,
                        "e4m3 or integer codes, F32 or BF16 rows, head_dim a multiple of 16 up to 256, pages up to 256 tokens");
    if (r->session_count > 0xffffull || r->token_count > max_tokens || r->key_value_heads > 0x7fffull ||
        r->max_blocks_per_session > 0xffffffffull || !yvx_u64_add(r->max_kv_tokens, r->token_count, &last) ||
        last > max_tokens || (last + r->block_tokens - 1ull) / r->block_tokens > r->max_blocks_per_session)
        return yvx_fail(err, YVEX_ERR_BOUNDS, where, "new rows exceed the block table");
    rc = yvx_backend_admit(backend, where, err);
    if (rc != YVEX_OK) return rc;
    memset(&a, 0, sizeof(a));
    a.token_stride = r->token_stride ? r->token_stride : kv_width;
    if (!r->session_stride && !yvx_u64_mul(r->token_count, a.token_stride, &elements))
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "row strides overflow");
    a.session_stride = r->session_stride ? r->session_stride : elements;
    extent = kv_width;
    if (!extend(r->token_count, a.token_stride, &extent) || !extend(r->session_count, a.session_stride, &extent))
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "row strides overflow");
    outputs[0] = r->key_codes, outputs[1] = r->value_codes, outputs[2] = r->key_scales, outputs[3] = r->value_scales;
    pages = 0x7fffffffull;
    for (i = 0; i < 4; ++i) {
        const unsigned long long unit = i < 2 ? page_bytes : r->key_value_heads * sizeof(float);
        const unsigned long long held = outputs[i]->bytes / unit;
        if (!view_ok(backend, outputs[i], i < 2 ? YVEX_DTYPE_I8 : YVEX_DTYPE_F32, 1ull) || !held)
            return yvx_fail(err, YVEX_ERR_FORMAT, where, "I8 pages and F32 scales of this backend are required");
        if (held < pages) pages = held;
    }
    if (!view_ok(backend, r->key, r->key->dtype, extent) || !view_ok(backend, r->value, r->value->dtype, extent) ||
        !yvx_u64_mul(r->session_count, r->max_blocks_per_session, &elements) ||
        !view_ok(backend, r->block_table, YVEX_DTYPE_I32, elements) ||
        (r->kv_tokens && !view_ok(backend, r->kv_tokens, YVEX_DTYPE_I32, r->session_count)) ||
        (r->new_tokens && !view_ok(backend, r->new_tokens, YVEX_DTYPE_I32, r->session_count)))
        return yvx_fail(err, YVEX_ERR_FORMAT, where, "row, length and table views do not hold the declared geometry");
    a.sessions = (unsigned int)r->session_count;
    a.tokens = (unsigned int)r->token_count;
    a.kv_heads = (unsigned int)r->key_value_heads;
    a.head_dim = (unsigned int)r->head_dimension;
    a.code = r->kv_code;
    a.dtype = r->key->dtype;
    a.key = r->key->data;
    a.value = r->value->data;
    a.kv_tokens = r->kv_tokens ? (const unsigned int *)r->kv_tokens->data : NULL;
    a.kv_tokens_uniform = (unsigned int)r->max_kv_tokens;
    a.new_tokens = r->new_tokens ? (const unsigned int *)r->new_tokens->data : NULL;
    a.block_table = (const int *)r->block_table->data;
    a.block_tokens = (unsigned int)r->block_tokens;
    a.block_table_stride = (unsigned int)r->max_blocks_per_session;
    a.pool_blocks = (unsigned int)pages;
    a.key_codes = r->key_codes->data;
    a.value_codes = r->value_codes->data;
    a.code_token_stride = r->head_dimension;
    a.code_head_stride = r->block_tokens * r->head_dimension;
    a.code_block_stride = page_bytes;
    a.key_scales = (float *)r->key_scales->data;
    a.value_scales = (float *)r->value_scales->data;
    a.status = backend->status_device;
    rc = yvx_backend_status_join(backend, where, err);
    if (rc != YVEX_OK) return rc;
    rc = yvx_cuda_kv8_append(&a, backend->stream);
    if (rc != 0) return shim_failed(backend, rc, where, err);
    facts->state_bytes = 2ull * r->session_count * r->token_count * kv_width;
    facts->activation_bytes = facts->state_bytes * yvx_dtype_bytes(r->key->dtype);
    rc = finish(backend, facts, 1u, 0ull, where, err);
    if (rc != YVEX_OK) return rc;
    r->key_codes->is_written = r->value_codes->is_written = 1;
    r->key_scales->is_written = r->value_scales->is_written = 1;
    yvex_error_clear(err);
    return YVEX_OK;
}

int yvex_b200_kv_pages_copy_execute(yvex_backend *backend, const yvex_b200_kv_pages_pool *pools,
                                    unsigned int pool_count, const yvex_b200_kv_copy *copies,
                                    unsigned int copy_count, unsigned long long block_tokens,
                                    yvex_backend_operation_facts *facts, yvex_error *err)
{
    const char *where = "b200.kv.pages_copy";
    yvx_kv_page_pool *described;
    yvx_kv_pages_args a;
    unsigned int i, j, launches = 0u;
    int rc;
    if (!pools || !pool_count || (copy_count && !copies) || !facts || !block_tokens || block_tokens > 0xffffffffull)
        return yvx_fail(err, YVEX_ERR_INVALID_ARG, where, "pools, copies, the page length and result facts are required");
    memset(facts, 0, sizeof(*facts));
    rc = yvx_backend_admit(backend, where, err);
    if (rc != YVEX_OK) return rc;
    described = (yvx_kv_page_pool *)calloc(pool_count, sizeof(*described));
    if (!described) return yvx_fail(err, YVEX_ERR_NOMEM, where, "no memory for the pool list");
    for (i = 0; i < pool_count; ++i) {
        const yvex_device_tensor *t = pools[i].tensor;
        const unsigned long long segments = pools[i].whole ? 1ull : pools[i].segments;
        unsigned long long block, rows;
        if (!yvx_tensor_owned(backend, t) || !t->rank || !t->dims[0] || t->dims[0] > 0x7fffffffull || !segments ||
            segments > 0xffffffffull || t->bytes % t->dims[0]) {
            free(described);
            return yvx_fail(err, YVEX_ERR_FORMAT, where, "a pool tensor [block]... of this backend is required");
        }
        block = t->bytes / t->dims[0];
        if (!yvx_u64_mul(segments, block_tokens, &rows) || (!pools[i].whole && block % rows)) {
            free(described);
            return yvx_fail(err, YVEX_ERR_FORMAT, where, "a pool's blocks are not segments of block_tokens rows");
        }
        described[i].base = t->data;
        described[i].blocks = (unsigned int)t->dims[0];
        described[i].segments = (unsigned int)segments;
        described[i].block_stride = block;
        described[i].segment_stride = block / segments;
        described[i].row_bytes = pools[i].whole ? 0ull : block / rows;
        described[i].fixed_bytes = pools[i].whole ? block : 0ull;
        for (j = 0; j < copy_count; ++j)
            if (copies[j].needed)
                facts->d2d_bytes += pools[i].whole ? block : copies[j].rows * segments * described[i].row_bytes;
    }
    memset(&a, 0, sizeof(a));
    a.pools = described;
    a.copies = (const struct yvx_kv_page_copy *)(const void *)copies;
    a.pool_count = pool_count;
    a.copy_count = copy_count;
    a.block_tokens = (unsigned int)block_tokens;
    rc = yvx_backend_status_join(backend, where, err);
    if (rc == YVEX_OK) {
        rc = yvx_cuda_kv_pages_copy(&a, backend->stream, &launches);
        if (rc != 0) rc = shim_failed(backend, rc, where, err);
    }
    free(described);
    if (rc != YVEX_OK) return rc;
    rc = finish(backend, facts, launches, 0ull, where, err);
    if (rc != YVEX_OK) return rc;
    yvex_error_clear(err);
    return YVEX_OK;
}
