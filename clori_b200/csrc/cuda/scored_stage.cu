// Pages of codes (or small pages of bf16) laid out as bf16 rows [session][kv_head][token][128] for the
// prompt-sized attention kernel. Values of a power-of-two scale are exact in bf16; others are rounded once.
// Memory bound: 1 byte read and 2 written per lane, 150 us for 131072 tokens of 8 KV heads (5.4 TB/s): a small part of a
// long prompt's attention, more than half of a call of 17 rows.
#include "scored.cuh"

namespace yvx {

constexpr int kStThreads = 256;

// Staged rows of at most this many bytes at a time (or one session's): calls of more go through groups of sessions, one after
// the other in the same workspace. 64 sessions of 512 to 32768 tokens, 17 rows of 32 heads in groups of 4: all together
// (8.6 GB) 1994 us, in two groups 2090, in four (2 GiB) 2471, whose ends no longer fill the machine.
constexpr unsigned long long kStBytes = 4ull << 30;

// grid: x = 32 tokens, y = kv_head, z = session. A thread moves 16 lanes of a token's K, then of its V.
template <int CODE>
__global__ void __launch_bounds__(kStThreads)
scored_stage_kernel(const yvx_scored_problem p, unsigned short *key, unsigned short *value, const unsigned long long tokens)
{
    const unsigned int b = blockIdx.z, kv_head = blockIdx.y;
    const unsigned int kv_tokens = admitted_kv_tokens(p.kv_tokens, b, p.kv_tokens_uniform, p.kv_tokens_max, p.status);
    // Only what the rows see is looked up: pages in front of it may be gone. Without row runs both ends move
    // with the row, so the first and the last row bound them.
    __shared__ int run[3];
    if (threadIdx.x < 32u) {
        const long long query_start = scored_query_start(p, b, kv_tokens);
        int first, end;
        if (p.row_first || p.row_end) {
            scored_hull(p, b, 0u, p.query_rows, kv_tokens, query_start, first, end);
        } else {
            first = scored_range(p, b, 0u, kv_tokens, query_start).first;
            end = scored_range(p, b, p.query_rows - 1u, kv_tokens, query_start).end;
        }
        if (threadIdx.x == 0) run[0] = first, run[1] = end, run[2] = scored_stage_first(p, kv_tokens, query_start);
    }
    __syncthreads();
    const unsigned int at = blockIdx.x * 32u + (threadIdx.x >> 3), token = (unsigned int)run[2] + at, d = (threadIdx.x & 7u) * 16u;
    if (token < (unsigned int)run[0] || token >= (unsigned int)run[1]) return;
    const int named = scored_page(p, b, token / p.block_tokens);
    const unsigned long long page = (unsigned long long)(named < 0 ? 0 : named), slot = token % p.block_tokens;
    const unsigned long long to = (((unsigned long long)b * p.kv_heads + kv_head) * tokens + at) * 128ull + d;
#pragma unroll
    for (int operand = 0; operand < 2; ++operand) {
        const unsigned long long from = page * (operand ? p.value_outer_stride : p.key_outer_stride) +
                                        slot * (operand ? p.value_token_stride : p.key_token_stride) +
                                        kv_head * (operand ? p.value_head_stride : p.key_head_stride) + d;
        const void *base = operand ? p.value : p.key;
        uint4 *dst = reinterpret_cast<uint4 *>((operand ? value : key) + to);
        if (CODE == YVX_KV_PLAIN) {
            const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned short *>(base) + from);
            dst[0] = src[0];
            dst[1] = src[1];
            continue;
        }
        const float scale = (operand ? p.value_scales : p.key_scales)[page * (p.scale_block_stride ? p.scale_block_stride : p.kv_heads) + kv_head];
        const uint4 raw = *reinterpret_cast<const uint4 *>(reinterpret_cast<const unsigned char *>(base) + from);
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t out[8];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float x[4];
            if (CODE == YVX_KV_E4M3) {
                uint32_t lo, hi;
                asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
                    "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
                    : "=r"(lo), "=r"(hi)
                    : "r"(words[w]));
                const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
                const float2 c = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
                x[0] = a.x, x[1] = a.y, x[2] = c.x, x[3] = c.y;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (float)(signed char)((words[w] >> (8 * e)) & 0xffu);
            }
            out[2 * w] = pack_bf16(x[0] * scale, x[1] * scale);
            out[2 * w + 1] = pack_bf16(x[2] * scale, x[3] * scale);
        }
        dst[0] = make_uint4(out[0], out[1], out[2], out[3]);
        dst[1] = make_uint4(out[4], out[5], out[6], out[7]);
    }
}

// Sessions of a group, and the bytes of its staged rows.
unsigned int scored_stage_sessions(const yvx_scored_problem &p)
{
    const unsigned long long fit = kStBytes / (2ull * p.kv_heads * scored_stage_tokens(p) * 128ull * 2ull);
    return fit < 1ull ? 1u : fit < p.sessions ? (unsigned int)fit : p.sessions;
}

unsigned long long scored_stage_bytes(const yvx_scored_problem &p)
{
    return 2ull * scored_stage_sessions(p) * p.kv_heads * scored_stage_tokens(p) * 128ull * 2ull;
}

// Enqueues the staging into `rows` and describes the staged rows.
int scored_stage_launch(const yvx_scored_problem &p, void *rows, yvx_scored_problem *staged, cudaStream_t stream)
{
    const unsigned long long tokens = scored_stage_tokens(p);
    unsigned short *key = reinterpret_cast<unsigned short *>(rows);
    unsigned short *value = key + (unsigned long long)p.sessions * p.kv_heads * tokens * 128ull;
    const dim3 grid((unsigned int)(tokens / 32ull), p.kv_heads, p.sessions);
    if (p.kv_code == YVX_KV_E4M3)
        scored_stage_kernel<YVX_KV_E4M3><<<grid, kStThreads, 0, stream>>>(p, key, value, tokens);
    else if (p.kv_code == YVX_KV_I8)
        scored_stage_kernel<YVX_KV_I8><<<grid, kStThreads, 0, stream>>>(p, key, value, tokens);
    else
        scored_stage_kernel<YVX_KV_PLAIN><<<grid, kStThreads, 0, stream>>>(p, key, value, tokens);
    *staged = p;
    staged->kv_code = YVX_KV_PLAIN;
    staged->kv_dtype = YVEX_DTYPE_BF16;
    staged->key = key;
    staged->value = value;
    staged->block_table = nullptr;
    staged->key_token_stride = staged->value_token_stride = 128ull;
    staged->key_head_stride = staged->value_head_stride = tokens * 128ull;
    staged->key_outer_stride = staged->value_outer_stride = (unsigned long long)p.kv_heads * tokens * 128ull;
    return yvx_cuda_check(cudaGetLastError(), "scored_stage_kernel");
}

}  // namespace yvx
