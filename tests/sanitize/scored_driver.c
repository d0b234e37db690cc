/* TEST INFRASTRUCTURE ONLY: drives the operators of scored attention, the 8-bit cache and page copies, and the
 * pool's truncation and compaction, over the host-memory device of scored_host.c. Random geometry meets views
 * that hold it, or one of which is a few elements short: the first have to be admitted and stay in bounds, the
 * second to be refused. Exits 0 when every check holds; a sanitizer report aborts the process. */
#include "yvex_b200/attention.h"
#include "yvex_b200/cuda_shim.h"

#include <stdio.h>
#include <string.h>

#define CHECK(cond) do { if (!(cond)) { fprintf(stderr, "check failed: %s (line %d): %s\n", #cond, __LINE__, err.message); return 1; } } while (0)

static unsigned long long state = 0x2545F4914F6CDD1Dull;
static unsigned int draw(unsigned int bound)
{
    state ^= state << 13; state ^= state >> 7; state ^= state << 17;
    return (unsigned int)(state % bound);
}

static yvex_error err;
static yvex_backend *backend;
static yvex_device_tensor *held[16];
static unsigned int count, short_one;      /* the tensor that lacks elements, or none */
static int cut;                            /* it was made */

static yvex_device_tensor *tensor(yvex_dtype dtype, unsigned long long elements, unsigned long long blocks)
{
    const unsigned long long size = dtype == YVEX_DTYPE_I8 ? 1ull : dtype == YVEX_DTYPE_BF16 ? 2ull : 4ull;
    yvex_backend_tensor_desc desc;
    memset(&desc, 0, sizeof(desc));
    if (count == short_one && elements > 1ull) --elements, cut = 1;
    desc.name = "t", desc.dtype = dtype, desc.rank = blocks ? 2u : 1u;
    desc.dims[0] = blocks ? blocks : elements, desc.dims[1] = blocks ? elements / blocks : 0ull;
    desc.bytes = elements * size;
    if (yvex_backend_tensor_alloc(backend, &desc, &held[count], &err) != YVEX_OK) return NULL;
    (void)yvex_backend_tensor_zero(backend, held[count], &err);
    return held[count++];
}

static void release(void)
{
    while (count) (void)yvex_backend_tensor_release(backend, &held[--count], &err);
    cut = 0;
}

static int attend(void)
{
    yvex_backend_operation_facts facts;
    unsigned int step, admitted = 0;
    for (step = 0; step < 4000u; ++step) {
        const int codes = (int)draw(3), paged = codes || draw(2);
        const unsigned long long sessions = 1u + draw(3), rows = 1u + draw(5), kv_heads = 1u + draw(3), group = 1u + draw(4);
        const unsigned long long hd = 1u + draw(256), tokens = 1u + draw(70), page = 1u + draw(40), pages = 1u + draw(6);
        const unsigned long long per = (tokens + page - 1ull) / page + draw(2), heads = kv_heads * group;
        const unsigned long long pad = draw(2) * draw(9), inner = paged ? page : tokens;
        const unsigned long long token = codes ? hd : kv_heads * hd + pad, head = codes ? page * hd : hd;
        const unsigned long long span = (inner - 1ull) * token + (kv_heads - 1ull) * head + hd, outer = span + draw(2) * draw(50);
        const yvex_dtype kv = codes ? YVEX_DTYPE_I8 : draw(2) ? YVEX_DTYPE_F32 : YVEX_DTYPE_BF16;
        const unsigned long long all = ((paged ? pages : sessions) - 1ull) * outer + (paged ? outer : span);
        yvex_b200_attention_scored_request r;
        int rc;
        memset(&r, 0, sizeof(r));
        short_one = draw(16);
        r.session_count = sessions, r.query_tokens = rows, r.query_heads = heads, r.key_value_heads = kv_heads;
        r.head_dimension = hd, r.key_value_tokens = tokens, r.causal = (int)draw(2), r.score_cap = (float)draw(2) * 30.0f;
        r.window = draw(2) * draw(9), r.kv_code = codes;
        r.kv_layout = paged ? YVEX_B200_KV_BLOCK_TABLE : YVEX_B200_KV_CONTIGUOUS;
        r.query_token_stride = heads * hd + pad, r.kv_token_stride = token, r.kv_head_stride = head, r.kv_outer_stride = outer;
        r.query = tensor(draw(2) ? YVEX_DTYPE_F32 : YVEX_DTYPE_BF16, (sessions * rows - 1ull) * r.query_token_stride + heads * hd, 0ull);
        r.output = tensor(draw(2) ? YVEX_DTYPE_F32 : YVEX_DTYPE_BF16, sessions * rows * heads * hd, 0ull);
        r.kv_tokens = tensor(YVEX_DTYPE_I32, sessions, 0ull);
        if (draw(2)) r.query_start = tensor(YVEX_DTYPE_I32, sessions, 0ull);
        if (draw(2)) r.row_first = tensor(YVEX_DTYPE_I32, sessions * rows, 0ull);
        if (draw(2)) r.row_end = tensor(YVEX_DTYPE_I32, sessions * rows, 0ull);
        if (draw(2)) r.slopes = tensor(YVEX_DTYPE_F32, heads, 0ull);
        if (paged) {
            r.block_table = tensor(YVEX_DTYPE_I32, sessions * per, 0ull);
            r.block_tokens = page, r.max_blocks_per_session = per;
        }
        if (paged) short_one = 16u;   /* a shorter pool is a pool of fewer pages: no fault */
        r.key = tensor(kv, all, 0ull);
        r.value = tensor(kv, all, 0ull);
        if (codes) {
            r.key_scales = tensor(YVEX_DTYPE_F32, pages * kv_heads, 0ull);
            r.value_scales = tensor(YVEX_DTYPE_F32, pages * kv_heads, 0ull);
        }
        rc = yvex_b200_attention_scored_execute(backend, &r, &facts, &err);
        if (cut) CHECK(rc == YVEX_ERR_FORMAT);
        else CHECK(rc == YVEX_OK && facts.kernel_launches == 2ull && r.output->is_written);
        admitted += rc == YVEX_OK;
        release();
    }
    CHECK(admitted > 1000u && admitted < 3900u);
    return 0;
}

static int append(void)
{
    yvex_backend_operation_facts facts;
    unsigned int step, admitted = 0;
    for (step = 0; step < 3000u; ++step) {
        const unsigned long long sessions = 1u + draw(3), fresh = 1u + draw(20), kv_heads = 1u + draw(3), hd = 16u * (1u + draw(8));
        const unsigned long long page = 1u + draw(33), present = draw(60), per = (present + fresh + page - 1ull) / page, pages = 1u + draw(5);
        const unsigned long long pad = draw(2) * draw(9);
        const yvex_dtype dtype = draw(2) ? YVEX_DTYPE_F32 : YVEX_DTYPE_BF16;
        yvex_b200_kv8_append_request r;
        int rc;
        memset(&r, 0, sizeof(r));
        short_one = draw(12);
        r.session_count = sessions, r.token_count = fresh, r.key_value_heads = kv_heads, r.head_dimension = hd;
        r.kv_code = 1 + (int)draw(2), r.token_stride = kv_heads * hd + pad, r.max_kv_tokens = present;
        r.key = tensor(dtype, (sessions * fresh - 1ull) * r.token_stride + kv_heads * hd, 0ull);
        r.value = tensor(dtype, (sessions * fresh - 1ull) * r.token_stride + kv_heads * hd, 0ull);
        r.block_table = tensor(YVEX_DTYPE_I32, sessions * per, 0ull);
        if (draw(2)) r.kv_tokens = tensor(YVEX_DTYPE_I32, sessions, 0ull);
        if (draw(2)) r.new_tokens = tensor(YVEX_DTYPE_I32, sessions, 0ull);
        r.block_tokens = page, r.max_blocks_per_session = per;
        short_one = cut ? short_one : 16u;
        r.key_codes = tensor(YVEX_DTYPE_I8, pages * page * kv_heads * hd, 0ull);
        r.value_codes = tensor(YVEX_DTYPE_I8, pages * page * kv_heads * hd, 0ull);
        r.key_scales = tensor(YVEX_DTYPE_F32, pages * kv_heads, 0ull);
        r.value_scales = tensor(YVEX_DTYPE_F32, (pages + draw(3)) * kv_heads, 0ull);
        rc = yvex_b200_kv8_append_execute(backend, &r, &facts, &err);
        if (cut) CHECK(rc == YVEX_ERR_FORMAT);
        else CHECK(rc == YVEX_OK && r.key_codes->is_written && r.value_scales->is_written);
        admitted += rc == YVEX_OK;
        release();
    }
    CHECK(admitted > 1000u && admitted < 2900u);
    return 0;
}

static int walk(void)
{
    enum { SESSIONS = 5, BLOCKS = 24, PAGE = 8, PER = 10, HEADS = 2, ROW = 16 };
    yvex_b200_kv_pool *pool = yvex_b200_kv_pool_create(BLOCKS, PAGE, SESSIONS, PER);
    yvex_backend_operation_facts facts;
    yvex_b200_kv_pages_pool pools[2];
    yvex_b200_kv_copy copies[BLOCKS];
    unsigned int open[SESSIONS], live = 0, moved = 0, step, i;
    memset(pools, 0, sizeof(pools));
    short_one = 16u;
    pools[0].tensor = tensor(YVEX_DTYPE_I8, BLOCKS * HEADS * PAGE * ROW, BLOCKS), pools[0].segments = HEADS;
    pools[1].tensor = tensor(YVEX_DTYPE_F32, BLOCKS * HEADS, BLOCKS), pools[1].whole = 1;
    CHECK(pool && pools[0].tensor && pools[1].tensor);
    for (step = 0; step < 20000u; ++step) {
        const unsigned int action = draw(8);
        const unsigned int id = live ? open[draw(live)] : 0u;
        unsigned int fresh;
        yvex_b200_kv_copy copy;
        if (action < 2u && live < SESSIONS) {
            const int rc = action && live ? yvex_b200_kv_pool_session_fork(pool, id, &fresh) : yvex_b200_kv_pool_session_open(pool, &fresh);
            CHECK(rc == YVEX_OK);
            open[live++] = fresh;
        } else if (action == 2u && live) {
            const unsigned int at = draw(live);
            CHECK(yvex_b200_kv_pool_session_close(pool, open[at]) == YVEX_OK);
            open[at] = open[--live];
        } else if (action == 3u && live) {
            const unsigned long long keep = draw(1u + (unsigned int)yvex_b200_kv_pool_committed(pool, id));
            CHECK(yvex_b200_kv_pool_session_truncate(pool, id, keep) == YVEX_OK && yvex_b200_kv_pool_committed(pool, id) == keep);
            CHECK(yvex_b200_kv_pool_session_truncate(pool, id, keep + 1ull) != YVEX_OK);
        } else if (action == 4u && draw(4) == 0u) {
            const unsigned int before = yvex_b200_kv_pool_free_blocks(pool);
            CHECK(yvex_b200_kv_pool_compact(pool, copies, BLOCKS, &moved) == YVEX_OK && yvex_b200_kv_pool_free_blocks(pool) == before);
            CHECK(yvex_b200_kv_pages_copy_execute(backend, pools, 2u, copies, moved, PAGE, &facts, &err) == YVEX_OK);
            for (i = 0; i < live; ++i) {
                unsigned long long r;
                for (r = 0; r < yvex_b200_kv_pool_committed(pool, open[i]); r += PAGE)
                    CHECK(yvex_b200_kv_pool_table(pool, open[i])[r / PAGE] < (int)(BLOCKS - before));
            }
        } else if (live) {
            const unsigned int rows = 1u + draw(12);
            if (yvex_b200_kv_pool_reserve(pool, id, rows, &copy) != YVEX_OK) continue;
            CHECK(yvex_b200_kv_pages_copy_execute(backend, pools, 2u, &copy, 1u, PAGE, &facts, &err) == YVEX_OK);
            CHECK(yvex_b200_kv_pool_commit(pool, id, draw(rows + 1u)) == YVEX_OK);
        }
    }
    while (live) CHECK(yvex_b200_kv_pool_session_close(pool, open[--live]) == YVEX_OK);
    CHECK(yvex_b200_kv_pool_free_blocks(pool) == BLOCKS);
    yvex_b200_kv_pool_destroy(pool);
    release();
    return 0;
}

static int ranges(void)
{
    const unsigned long long lengths[4] = {3ull, 0ull, 5ull, ~0ull}, prefixes[4] = {9ull, 1ull, 2ull, 0ull};
    int first[12], end[12];
    CHECK(yvex_b200_attention_row_ranges(lengths, prefixes, 3ull, 0ull, 12ull, first, end) && first[3] == 3 && end[3] == 5 && end[11] == 0);
    CHECK(!yvex_b200_attention_row_ranges(lengths, prefixes, 4ull, 0ull, 12ull, first, end));
    CHECK(!yvex_b200_attention_row_ranges(lengths, prefixes, 3ull, ~0ull, 12ull, first, end));
    CHECK(!yvex_b200_attention_row_ranges(NULL, NULL, 1ull, 0ull, 12ull, first, end));
    return 0;
}

int main(void)
{
    yvex_backend_options options = {YVEX_BACKEND_KIND_CUDA, "0", 0ull};
    CHECK(yvex_backend_open(&backend, &options, &err) == YVEX_OK);
    if (attend() || append() || walk() || ranges()) return 1;
    CHECK(yvex_backend_close_checked(&backend, &err) == YVEX_OK);
    puts("scored operators clean under the sanitizers");
    return 0;
}
