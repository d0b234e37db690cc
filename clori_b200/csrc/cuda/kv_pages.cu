// Copies of pages in every layer's pool, one launch for up to 512 copies and 128 pools.
//
// The lists travel as kernel parameters: no upload, no buffer that has to outlive the call, and a
// captured graph carries them. A CTA moves 16 KB of one (copy, pool) pair, four 16-byte loads of a
// thread in flight before the first store. Bound by HBM: every byte is read once and written once.
// Measured: 700 whole pages in 16 pools 228 us (6.4 TB/s of reads and writes), 32 partly filled pages in 64 pools
// 20.5 us; one fork's page a launch.
#include "common.cuh"

#include <stdlib.h>

namespace yvx {

constexpr unsigned int kPgCopies = 512, kPgPools = 128, kPgThreads = 256, kPgBatch = 4;

struct PagesBatch {
    yvx_kv_page_pool pools[kPgPools];
    int source[kPgCopies], destination[kPgCopies];
    unsigned int rows[kPgCopies];
};
static_assert(sizeof(PagesBatch) <= 32000, "the lists have to fit the kernel parameters");

// grid: x = piece of the pair's bytes, y = copy, z = pool
template <typename Unit>
__global__ void __launch_bounds__(kPgThreads) kv_pages_copy_kernel(const __grid_constant__ PagesBatch batch)
{
    const yvx_kv_page_pool &pool = batch.pools[blockIdx.z];
    const unsigned long long segment_bytes =
        pool.fixed_bytes ? pool.fixed_bytes : (unsigned long long)batch.rows[blockIdx.y] * pool.row_bytes;
    const unsigned long long units = segment_bytes / sizeof(Unit), total = units * pool.segments;
    const unsigned char *from = reinterpret_cast<const unsigned char *>(pool.base) +
                                (unsigned long long)batch.source[blockIdx.y] * pool.block_stride;
    unsigned char *to = reinterpret_cast<unsigned char *>(pool.base) +
                        (unsigned long long)batch.destination[blockIdx.y] * pool.block_stride;
    Unit value[kPgBatch];
    unsigned long long offset[kPgBatch];
    const unsigned long long first = (unsigned long long)blockIdx.x * kPgThreads * kPgBatch + threadIdx.x;
#pragma unroll
    for (int i = 0; i < (int)kPgBatch; ++i) {
        const unsigned long long at = first + (unsigned long long)i * kPgThreads;
        if (at < total) {
            const unsigned long long segment = pool.segments == 1u ? 0ull : at / units;
            offset[i] = segment * pool.segment_stride + (at - segment * units) * sizeof(Unit);
            value[i] = *reinterpret_cast<const Unit *>(from + offset[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < (int)kPgBatch; ++i)
        if (first + (unsigned long long)i * kPgThreads < total) *reinterpret_cast<Unit *>(to + offset[i]) = value[i];
}

static int pages_refuse(int code, const char *text)
{
    yvx_cuda_set_error_text(text);
    return code;
}

static int pages_check(const yvx_kv_pages_args *a)
{
    if (!a || !a->pools || !a->pool_count || !a->block_tokens || (a->copy_count && !a->copies))
        return pages_refuse(YVEX_ERR_INVALID_ARG, "kv pages: pools, copies and the page length are required");
    unsigned int blocks = 0xffffffffu;
    for (unsigned int i = 0; i < a->pool_count; ++i) {
        const yvx_kv_page_pool &p = a->pools[i];
        // sizes bounded one by one, so that no product below leaves 64 bits
        const unsigned long long most = 0xffffffffffull;
        const bool bounded = p.base && p.blocks && p.blocks <= 0x7fffffffu && p.segments && p.row_bytes <= most && p.fixed_bytes <= most &&
                             p.segment_stride <= most && p.block_stride <= (1ull << 62) / p.blocks;
        const unsigned long long segment = !bounded ? 0ull : p.fixed_bytes ? p.fixed_bytes : p.row_bytes * a->block_tokens;
        if (!segment || segment > most || (p.segments > 1u && p.segment_stride < segment) || p.block_stride < segment ||
            (p.segments > 1u && p.segment_stride > (p.block_stride - segment) / (p.segments - 1ull)))
            return pages_refuse(YVEX_ERR_INVALID_ARG, "kv pages: a pool's strides do not hold its pages");
        if (p.blocks < blocks) blocks = p.blocks;
    }
    unsigned char *role = (unsigned char *)calloc(blocks, 1);  // 1: a source, 2: a destination
    if (!role) return pages_refuse(YVEX_ERR_NOMEM, "kv pages: no memory to check the copies");
    const char *wrong = nullptr;
    for (unsigned int i = 0; i < a->copy_count && !wrong; ++i) {
        const yvx_kv_page_copy &c = a->copies[i];
        if (!c.needed) continue;
        if (c.source_block < 0 || c.destination_block < 0 || (unsigned int)c.source_block >= blocks ||
            (unsigned int)c.destination_block >= blocks || c.rows > a->block_tokens)
            wrong = "kv pages: a copy names a page outside a pool, or more rows than a page has";
        else if (role[c.destination_block] || role[c.source_block] == 2 || c.source_block == c.destination_block)
            wrong = "kv pages: a destination is also a source or the destination of another copy";
        else {
            role[c.source_block] = 1;
            role[c.destination_block] = 2;
        }
    }
    free(role);
    return wrong ? pages_refuse(YVEX_ERR_INVALID_ARG, wrong) : 0;
}

}  // namespace yvx

extern "C" int yvx_cuda_kv_pages_copy(const yvx_kv_pages_args *a, void *stream, unsigned int *launches)
{
    using namespace yvx;
    if (launches) *launches = 0u;
    const int rc = pages_check(a);
    if (rc != 0) return rc;
    PagesBatch batch;
    unsigned int count = 0u;
    for (unsigned int p0 = 0; p0 < a->pool_count; p0 += kPgPools) {
        const unsigned int pools = a->pool_count - p0 < kPgPools ? a->pool_count - p0 : kPgPools;
        unsigned long long bits = 0ull;
        for (unsigned int i = 0; i < pools; ++i) {
            const yvx_kv_page_pool &p = batch.pools[i] = a->pools[p0 + i];
            bits |= reinterpret_cast<uintptr_t>(p.base) | p.block_stride | (p.fixed_bytes ? p.fixed_bytes : p.row_bytes) |
                    (p.segments > 1u ? p.segment_stride : 0ull);
        }
        for (unsigned int c0 = 0; c0 < a->copy_count;) {
            unsigned int copies = 0u, rows = 0u;
            for (; c0 < a->copy_count && copies < kPgCopies; ++c0) {
                const yvx_kv_page_copy &c = a->copies[c0];
                if (!c.needed) continue;
                batch.source[copies] = c.source_block;
                batch.destination[copies] = c.destination_block;
                batch.rows[copies++] = c.rows;
                if (c.rows > rows) rows = c.rows;
            }
            unsigned long long most = 0ull;
            for (unsigned int i = 0; i < pools; ++i) {
                const yvx_kv_page_pool &p = batch.pools[i];
                const unsigned long long bytes = p.segments * (p.fixed_bytes ? p.fixed_bytes : rows * p.row_bytes);
                if (bytes > most) most = bytes;
            }
            if (!copies || !most) continue;
            const unsigned long long unit = !(bits & 15ull) ? 16ull : !(bits & 3ull) ? 4ull : 1ull;
            const unsigned long long pieces = (most / unit + kPgThreads * kPgBatch - 1ull) / (kPgThreads * kPgBatch);
            if (pieces > 0x7fffffffull) return pages_refuse(YVEX_ERR_BOUNDS, "kv pages: a page is too large for one grid");
            const dim3 grid((unsigned int)pieces, copies, pools);
            cudaStream_t s = (cudaStream_t)stream;
            if (unit == 16ull)
                kv_pages_copy_kernel<uint4><<<grid, kPgThreads, 0, s>>>(batch);
            else if (unit == 4ull)
                kv_pages_copy_kernel<unsigned int><<<grid, kPgThreads, 0, s>>>(batch);
            else
                kv_pages_copy_kernel<unsigned char><<<grid, kPgThreads, 0, s>>>(batch);
            const int launched = yvx_cuda_check(cudaGetLastError(), "kv_pages_copy_kernel");
            if (launched != 0) return launched;
            ++count;
        }
    }
    if (launches) *launches = count;
    return 0;
}
