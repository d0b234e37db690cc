// What the scored-attention kernels share: the visible run of a query row, the score rule and
// the split-KV partials.
#pragma once

#include "pipeline.cuh"

namespace yvx {

constexpr float kScoredLog2e = 1.4426950408889634f;

// Tokens [first, end), and where the distance bias counts from: the row's own position, or the end of the run that is
// nearest to it. A row's logits may all move alike, and distances of millions would take their last bits along.
struct ScoredRange {
    int first, end, position;
};

__device__ __forceinline__ long long scored_query_start(const yvx_scored_problem &p, unsigned int b,
                                                        unsigned int kv_tokens)
{
    if (p.query_start) return (long long)p.query_start[b];
    if (p.query_start_from_end) return (long long)kv_tokens - (long long)p.query_rows;
    return (long long)p.query_start_uniform;
}

__device__ __forceinline__ ScoredRange scored_range(const yvx_scored_problem &p, unsigned int b, unsigned int row,
                                                    unsigned int kv_tokens, long long query_start)
{
    ScoredRange r;
    const long long position = query_start + (long long)row;
    const unsigned long long at = (unsigned long long)b * p.query_rows + row;
    long long first = p.row_first ? (long long)p.row_first[at] : 0;
    if (p.window) first = max(first, position + 1 - (long long)p.window);
    long long end = p.row_end ? (long long)p.row_end[at] : (p.causal ? position + 1 : (long long)kv_tokens);
    end = min(max(end, 0ll), (long long)kv_tokens);
    first = min(max(first, 0ll), end);
    r.first = (int)first;
    r.end = (int)end;
    r.position = (int)max(min(position, end - 1), first);
    return r;
}

// Query heads that share a 128-row tile of the prompt kernel: a KV head's group, so that few query rows fill a
// tile too. One where a tile does not hold a group.
__host__ __device__ __forceinline__ unsigned int scored_packed_heads(const yvx_scored_problem &p)
{
    const unsigned int group = p.query_heads / p.kv_heads;
    return group <= 128u ? group : 1u;
}

// A session's staged rows: all that its rows can see, which a causal window bounds (the same tokens on both sides: from
// the first row's window on, rounded down to a tile of 128).
__host__ __device__ __forceinline__ bool scored_stage_windowed(const yvx_scored_problem &p)
{
    return p.window && p.causal && !p.row_end &&
           (unsigned long long)p.window + p.query_rows + 126ull < (unsigned long long)p.kv_tokens_max;
}
__host__ __device__ __forceinline__ unsigned long long scored_stage_tokens(const yvx_scored_problem &p)
{
    const unsigned long long seen = scored_stage_windowed(p) ? (unsigned long long)p.window + p.query_rows + 126ull : p.kv_tokens_max;
    return (seen + 63ull) / 64ull * 64ull;
}
__device__ __forceinline__ int scored_stage_first(const yvx_scored_problem &p, unsigned int kv_tokens, long long query_start)
{
    if (!scored_stage_windowed(p)) return 0;
    return (int)min(max(query_start + 1 - (long long)p.window, 0ll), (long long)kv_tokens) & ~127;
}

// The run of tokens that some row of [row0, row1) sees (first == end: none does); all 32 lanes.
__device__ __forceinline__ void scored_hull(const yvx_scored_problem &p, unsigned int b, unsigned int row0,
                                            unsigned int row1, unsigned int kv_tokens, long long query_start,
                                            int &first, int &end)
{
    int lo = 0x7fffffff, hi = 0;
    for (unsigned int row = row0 + (threadIdx.x & 31u); row < row1; row += 32u) {
        const ScoredRange r = scored_range(p, b, row, kv_tokens, query_start);
        if (r.first < r.end) {
            lo = min(lo, r.first);
            hi = max(hi, r.end);
        }
    }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    first = hi > 0 ? lo : 0;
    end = hi;
}

// Splits count tokens from the hull's first 64-token boundary.
__device__ __forceinline__ void scored_split(const yvx_scored_problem &p, unsigned int split, int hull_first,
                                             int hull_end, int &t0, int &t1)
{
    const long long base = (long long)(hull_first & ~63) + (long long)split * (long long)p.chunk_tokens;
    t0 = (int)min(base, (long long)hull_end);
    t1 = (int)min(base + (long long)p.chunk_tokens, (long long)hull_end);
}

// A page of the pool, or -1 (recorded as a contract failure) when the table names none.
__device__ __forceinline__ int scored_page(const yvx_scored_problem &p, unsigned int b, unsigned int index)
{
    const int page = p.block_table[(unsigned long long)b * p.block_table_stride + index];
    if (page >= 0 && (unsigned int)page < p.pool_blocks) return page;
    atomicCAS(p.status, 0, YVX_STATUS_CONTRACT);
    return -1;
}

// Partials of a split: [item][split][head_dim + 4] floats (o, maximum, sum, two unused: rows stay on
// 16-byte boundaries), an item being (session, row, query head); o is not normalised, the maximum
// is in log2 units, a split that saw nothing has sum 0.
__device__ __forceinline__ float *scored_partial(const yvx_scored_problem &p, unsigned long long item,
                                                 unsigned int split)
{
    return reinterpret_cast<float *>(p.workspace) + (item * p.max_splits + split) * (p.head_dim + 4ull);
}

__device__ __forceinline__ void scored_store_empty(const yvx_scored_problem &p, unsigned long long item,
                                                   unsigned int split, unsigned int lane, unsigned int lanes)
{
    if (p.max_splits > 1u) {
        if (lane == 0) {
            float *part = scored_partial(p, item, split);
            part[p.head_dim] = -INFINITY;
            part[p.head_dim + 1] = 0.0f;
        }
        return;
    }
    for (unsigned int d = lane; d < p.head_dim; d += lanes) store_output(p.output, p.output_dtype, item * p.head_dim + d, 0.0f);
}

int scored_general_launch(const yvx_scored_problem &p, cudaStream_t stream);
// `staged`: K and V are staged rows; scored_stage_tokens of a session, from scored_stage_first on.
int scored_prompt_launch(const yvx_scored_problem &p, bool staged, cudaStream_t stream);
unsigned long long scored_stage_bytes(const yvx_scored_problem &p);
unsigned int scored_stage_sessions(const yvx_scored_problem &p);
int scored_stage_launch(const yvx_scored_problem &p, void *rows, yvx_scored_problem *staged, cudaStream_t stream);
int scored_decode_launch(const yvx_scored_problem &p, cudaStream_t stream);
int scored_combine_launch(const yvx_scored_problem &p, cudaStream_t stream);

}  // namespace yvx
