/* TEST INFRASTRUCTURE ONLY: a device in host memory for the operators of scored attention, the 8-bit cache
 * and page copies. Allocations are malloc, copies memcpy; the stand-ins of the kernels read the first and last
 * element of everything that the call lets a kernel read and write all that it lets it write, so that
 * AddressSanitizer sees a view which the host layer admitted although it is too small. None computes anything. */
#include "yvex_b200/abi.h"
#include "yvex_b200/cuda_shim.h"

#include <stddef.h>
#include <stdlib.h>
#include <string.h>

volatile unsigned int scored_host_seen;

int yvx_cuda_device_count(int *count) { *count = 1; return 0; }
int yvx_cuda_device_select(int device) { (void)device; return 0; }
int yvx_cuda_device_synchronize(void) { return 0; }
int yvx_cuda_device_properties(int device, int *sm, int *major, int *minor, unsigned long long *bytes, char *name, size_t cap)
{
    (void)device;
    *sm = 148, *major = 10, *minor = 0, *bytes = 1ull << 30;
    if (cap) name[0] = 0;
    return 0;
}
int yvx_cuda_malloc(void **out, unsigned long long bytes) { *out = malloc(bytes); return *out ? 0 : YVEX_ERR_NOMEM; }
int yvx_cuda_free(void *p) { free(p); return 0; }
int yvx_cuda_host_alloc(void **out, unsigned long long bytes) { return yvx_cuda_malloc(out, bytes); }
int yvx_cuda_host_free(void *p) { free(p); return 0; }
int yvx_cuda_memset_async(void *d, int v, unsigned long long n, void *s) { (void)s; memset(d, v, n); return 0; }
int yvx_cuda_upload_async(void *d, const void *h, unsigned long long n, void *s) { (void)s; memcpy(d, h, n); return 0; }
int yvx_cuda_download_async(void *h, const void *d, unsigned long long n, void *s) { (void)s; memcpy(h, d, n); return 0; }
int yvx_cuda_stream_create(void **s) { return yvx_cuda_malloc(s, 1ull); }
int yvx_cuda_stream_destroy(void *s) { free(s); return 0; }
int yvx_cuda_stream_synchronize(void *s) { (void)s; return 0; }

static void look(const void *base, unsigned long long from, unsigned long long bytes)
{
    if (!base || !bytes) return;
    scored_host_seen += ((const unsigned char *)base)[from] + ((const unsigned char *)base)[from + bytes - 1ull];
}

void yvx_cuda_scored_plan(yvx_scored_problem *p, int sm) { (void)sm; p->chunk_tokens = 64u, p->max_splits = 2u; }
unsigned long long yvx_cuda_scored_workspace_bytes(const yvx_scored_problem *p) { return 512ull * p->sessions; }

int yvx_cuda_scored_attention(const yvx_scored_problem *p, void *stream, unsigned int *launches)
{
    const unsigned long long element = p->kv_code ? 1ull : p->kv_dtype == YVEX_DTYPE_F32 ? 4ull : 2ull;
    const unsigned long long q_element = p->query_dtype == YVEX_DTYPE_F32 ? 4ull : 2ull;
    const unsigned long long o_element = p->output_dtype == YVEX_DTYPE_F32 ? 4ull : 2ull;
    const unsigned long long outer = p->block_table ? p->pool_blocks : p->sessions;
    const unsigned long long inner = p->block_table ? p->block_tokens : p->kv_tokens_max;
    const unsigned long long rows = (unsigned long long)p->sessions * p->query_rows;
    const unsigned long long last = (outer - 1ull) * p->key_outer_stride + (inner - 1ull) * p->key_token_stride +
                                    (p->kv_heads - 1ull) * p->key_head_stride + p->head_dim;
    (void)stream;
    look(p->key, 0ull, last * element);
    look(p->value, 0ull, last * element);
    look(p->query, 0ull, ((p->sessions - 1ull) * p->query_session_stride + (p->query_rows - 1ull) * p->query_row_stride +
                          (unsigned long long)p->query_heads * p->head_dim) * q_element);
    look(p->kv_tokens, 0ull, 4ull * p->sessions);
    look(p->query_start, 0ull, 4ull * p->sessions);
    look(p->row_first, 0ull, 4ull * rows);
    look(p->row_end, 0ull, 4ull * rows);
    look(p->slopes, 0ull, 4ull * p->query_heads);
    look(p->block_table, 0ull, 4ull * p->sessions * p->block_table_stride);
    look(p->key_scales, 0ull, 4ull * p->pool_blocks * p->kv_heads);
    look(p->value_scales, 0ull, 4ull * p->pool_blocks * p->kv_heads);
    memset(p->workspace, 1, p->workspace_bytes);
    memset(p->output, 0, rows * p->query_heads * p->head_dim * o_element);
    *p->status = 0;
    if (launches) *launches = 2u;
    return 0;
}

int yvx_cuda_kv8_append(const yvx_kv8_append_args *a, void *stream)
{
    const unsigned long long element = a->dtype == YVEX_DTYPE_F32 ? 4ull : 2ull;
    const unsigned long long bytes = ((a->sessions - 1ull) * a->session_stride + (a->tokens - 1ull) * a->token_stride +
                                      (unsigned long long)a->kv_heads * a->head_dim) * element;
    const unsigned long long codes = (a->pool_blocks - 1ull) * a->code_block_stride + (a->kv_heads - 1ull) * a->code_head_stride +
                                     (a->block_tokens - 1ull) * a->code_token_stride + a->head_dim;
    (void)stream;
    look(a->key, 0ull, bytes);
    look(a->value, 0ull, bytes);
    look(a->kv_tokens, 0ull, 4ull * a->sessions);
    look(a->new_tokens, 0ull, 4ull * a->sessions);
    look(a->block_table, 0ull, 4ull * a->sessions * a->block_table_stride);
    memset(a->key_codes, 1, codes);
    memset(a->value_codes, 1, codes);
    memset(a->key_scales, 0, 4ull * a->pool_blocks * a->kv_heads);
    memset(a->value_scales, 0, 4ull * a->pool_blocks * a->kv_heads);
    return 0;
}

int yvx_cuda_kv_pages_copy(const yvx_kv_pages_args *a, void *stream, unsigned int *launches)
{
    unsigned int i, j, s;
    (void)stream;
    for (i = 0; i < a->copy_count; ++i)
        for (j = 0; j < a->pool_count; ++j) {
            const yvx_kv_page_pool *pool = &a->pools[j];
            if (!a->copies[i].needed) continue;
            if (a->copies[i].source_block >= (int)pool->blocks || a->copies[i].destination_block >= (int)pool->blocks) return YVEX_ERR_INVALID_ARG;
            for (s = 0; s < pool->segments; ++s)
                memcpy((char *)pool->base + a->copies[i].destination_block * pool->block_stride + s * pool->segment_stride,
                       (char *)pool->base + a->copies[i].source_block * pool->block_stride + s * pool->segment_stride,
                       pool->fixed_bytes ? pool->fixed_bytes : a->copies[i].rows * pool->row_bytes);
        }
    if (launches) *launches = 1u;
    return 0;
}
