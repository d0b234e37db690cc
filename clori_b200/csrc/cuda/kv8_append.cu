// New K and V rows into pages of 8-bit codes with one power-of-two scale per (page, KV head).
//
// One CTA per (page that the new rows touch, KV head, K or V, session). It takes the largest
// magnitude of the page's new rows, chooses the scale, brings codes that the page already holds
// to it when it grew, and writes the new rows' codes. Scales are powers of two, so every division
// is exact and a lane is rounded once when it is stored (again only if its page's scale grows;
// e4m3 codes then lose nothing above the subnormal range). Memory bound: an element is read once
// (2 or 4 bytes) and one byte is written; a thread owns 16 adjacent lanes of a row, so both sides
// move in 16-byte pieces.
#include "common.cuh"

namespace yvx {

constexpr int kA8Threads = 128;

template <bool E4M3>
__device__ __forceinline__ float a8_decode(unsigned int byte)
{
    if (!E4M3) return (float)(signed char)byte;
    uint32_t pair;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(pair) : "h"((unsigned short)byte));
    return __half2float(__ushort_as_half((unsigned short)(pair & 0xffffu)));
}

template <bool E4M3>
__device__ __forceinline__ unsigned int a8_encode4(const float (&x)[4])
{
    if (E4M3) {
        unsigned short lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1]), "f"(x[0]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3]), "f"(x[2]));
        return (unsigned int)lo | ((unsigned int)hi << 16);
    }
    unsigned int packed = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) packed |= ((unsigned int)__float2int_rn(x[i]) & 0xffu) << (8 * i);
    return packed;
}

// 16 adjacent lanes of a row. `aligned`: rows lie on 16-byte boundaries.
__device__ __forceinline__ void a8_load16(const void *base, int dtype, unsigned long long at, bool aligned, float (&x)[16])
{
    if (dtype == YVEX_DTYPE_BF16) {
        const unsigned short *src = reinterpret_cast<const unsigned short *>(base) + at;
        if (aligned) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 raw = reinterpret_cast<const uint4 *>(src)[i];
                const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    x[8 * i + 2 * w] = __uint_as_float(words[w] << 16);
                    x[8 * i + 2 * w + 1] = __uint_as_float(words[w] & 0xffff0000u);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = __uint_as_float((uint32_t)src[i] << 16);
        }
    } else {
        const float *src = reinterpret_cast<const float *>(base) + at;
        if (aligned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 raw = reinterpret_cast<const float4 *>(src)[i];
                x[4 * i] = raw.x, x[4 * i + 1] = raw.y, x[4 * i + 2] = raw.z, x[4 * i + 3] = raw.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = src[i];
        }
    }
}

// The smallest power of two s >= 2^-126 with amax <= limit * s; limit = (1 + fraction) * 2^shift.
__device__ __forceinline__ float a8_scale(float amax, float limit, int shift)
{
    const int exponent = (int)(__float_as_uint(amax) >> 23) - shift;
    const float s = __uint_as_float((unsigned int)max(exponent, 1) << 23);
    return amax > limit * s ? 2.0f * s : s;
}

// grid: x = touched page of the session, y = 2 * kv_head + (0: K, 1: V), z = session
template <bool E4M3>
__global__ void __launch_bounds__(kA8Threads) kv8_append_kernel(const yvx_kv8_append_args a, const int aligned)
{
    __shared__ float warp_top[kA8Threads / 32];
    const unsigned int b = blockIdx.z, kv_head = blockIdx.y >> 1, is_value = blockIdx.y & 1u;
    const unsigned long long present = a.kv_tokens ? a.kv_tokens[b] : a.kv_tokens_uniform;
    const unsigned long long fresh = a.new_tokens ? a.new_tokens[b] : a.tokens;
    // Lengths live in device memory: more rows than the launch was made for, or rows behind the
    // session's table row, are recorded and nothing of the session is written.
    if (fresh > a.tokens || present + fresh > (unsigned long long)a.block_table_stride * a.block_tokens) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, YVX_STATUS_CONTRACT);
        return;
    }
    const unsigned long long index = present / a.block_tokens + blockIdx.x;
    const unsigned long long page_start = index * a.block_tokens;
    if (page_start >= present + fresh) return;
    const int page = a.block_table[(unsigned long long)b * a.block_table_stride + index];
    if (page < 0 || (unsigned int)page >= a.pool_blocks) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, YVX_STATUS_CONTRACT);
        return;
    }
    const unsigned long long from = present > page_start ? present : page_start;
    const unsigned long long until = min(present + fresh, page_start + a.block_tokens);
    const unsigned int kept = (unsigned int)(from - page_start), rows = (unsigned int)(until - from);
    const unsigned int chunks = a.head_dim / 16u;
    const void *source = is_value ? a.value : a.key;
    const unsigned long long origin = (unsigned long long)b * a.session_stride + (from - present) * a.token_stride +
                                      (unsigned long long)kv_head * a.head_dim;
    unsigned char *codes = reinterpret_cast<unsigned char *>(is_value ? a.value_codes : a.key_codes) +
                           (unsigned long long)page * a.code_block_stride + (unsigned long long)kv_head * a.code_head_stride;
    float *scale_slot = (is_value ? a.value_scales : a.key_scales) +
                        (unsigned long long)page * (a.scale_block_stride ? a.scale_block_stride : a.kv_heads) + kv_head;

    float top = 0.0f;
    bool finite = true;
    for (unsigned int i = threadIdx.x; i < rows * chunks; i += kA8Threads) {
        float x[16];
        a8_load16(source, a.dtype, origin + (unsigned long long)(i / chunks) * a.token_stride + 16u * (i % chunks), aligned, x);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const bool ok = fabsf(x[e]) < INFINITY;
            finite = finite && ok;
            top = ok ? fmaxf(top, fabsf(x[e])) : top;
        }
    }
    if (!finite) atomicCAS(a.status, 0, YVX_STATUS_NONFINITE);
    top = warp_max(top);
    if ((threadIdx.x & 31u) == 0) warp_top[threadIdx.x >> 5] = top;
    const float held = kept ? *scale_slot : 0.0f;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kA8Threads / 32; ++w) top = fmaxf(top, warp_top[w]);
    const float wanted = E4M3 ? a8_scale(top, 448.0f, 8) : a8_scale(top, 127.0f, 6);
    const float scale = fmaxf(held, wanted);
    if (scale > held && kept) {
        const float ratio = held / scale;
        for (unsigned int i = threadIdx.x; i < kept * chunks; i += kA8Threads) {
            uint4 *slot = reinterpret_cast<uint4 *>(codes + (i / chunks) * a.code_token_stride + 16u * (i % chunks));
            uint4 raw = *slot;
            uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = a8_decode<E4M3>((words[w] >> (8 * e)) & 0xffu) * ratio;
                words[w] = a8_encode4<E4M3>(x);
            }
            *slot = make_uint4(words[0], words[1], words[2], words[3]);
        }
    }
    const float inverse = 1.0f / scale;
    for (unsigned int i = threadIdx.x; i < rows * chunks; i += kA8Threads) {
        const unsigned int row = i / chunks, chunk = i % chunks;
        float x[16];
        a8_load16(source, a.dtype, origin + (unsigned long long)row * a.token_stride + 16u * chunk, aligned, x);
        uint32_t words[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fabsf(x[4 * w + e]) < INFINITY ? x[4 * w + e] * inverse : 0.0f;
            words[w] = a8_encode4<E4M3>(y);
        }
        *reinterpret_cast<uint4 *>(codes + (unsigned long long)(kept + row) * a.code_token_stride + 16u * chunk) =
            make_uint4(words[0], words[1], words[2], words[3]);
    }
    if (threadIdx.x == 0 && scale != held) *scale_slot = scale;
}

static int a8_refuse(int code, const char *text)
{
    yvx_cuda_set_error_text(text);
    return code;
}

}  // namespace yvx

extern "C" int yvx_cuda_kv8_append(const yvx_kv8_append_args *a, void *stream)
{
    using namespace yvx;
    if (!a || !a->key || !a->value || !a->block_table || !a->key_codes || !a->value_codes || !a->key_scales ||
        !a->value_scales || !a->status || !a->sessions || !a->tokens || !a->kv_heads || !a->head_dim || !a->block_tokens ||
        !a->block_table_stride || !a->pool_blocks || a->pool_blocks > 0x7fffffffu)
        return a8_refuse(YVEX_ERR_INVALID_ARG, "kv8 append: rows, codes, scales, table and geometry are required");
    if ((a->code != YVX_KV_E4M3 && a->code != YVX_KV_I8) || (a->dtype != YVEX_DTYPE_F32 && a->dtype != YVEX_DTYPE_BF16) ||
        a->head_dim % 16u || a->head_dim > 256u || a->block_tokens > 256u)
        return a8_refuse(YVEX_ERR_UNSUPPORTED,
                         "kv8 append: e4m3 or integer codes, F32 or BF16 rows, head_dim a multiple of 16 up to 256, pages up to 256 tokens");
    if ((reinterpret_cast<uintptr_t>(a->key_codes) & 15u) || (reinterpret_cast<uintptr_t>(a->value_codes) & 15u) ||
        (a->code_token_stride & 15ull) || (a->code_head_stride & 15ull) || (a->code_block_stride & 15ull) ||
        a->code_token_stride < a->head_dim || !a->code_head_stride || !a->code_block_stride)
        return a8_refuse(YVEX_ERR_INVALID_ARG, "kv8 append: codes and their strides lie on 16-byte boundaries");
    const unsigned long long pages = ((unsigned long long)a->tokens + 2ull * a->block_tokens - 2ull) / a->block_tokens;
    if (a->sessions > 65535u || a->kv_heads > 32767u || pages > 0x7fffffffull)
        return a8_refuse(YVEX_ERR_BOUNDS, "kv8 append: at most 65535 sessions and 32767 heads");
    const unsigned long long unit = a->dtype == YVEX_DTYPE_BF16 ? 8ull : 4ull;
    const int aligned = !(reinterpret_cast<uintptr_t>(a->key) & 15u) && !(reinterpret_cast<uintptr_t>(a->value) & 15u) &&
                        a->token_stride % unit == 0ull && a->session_stride % unit == 0ull;
    const dim3 grid((unsigned int)pages, 2u * a->kv_heads, a->sessions);
    if (a->code == YVX_KV_E4M3)
        kv8_append_kernel<true><<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(*a, aligned);
    else
        kv8_append_kernel<false><<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(*a, aligned);
    return yvx_cuda_check(cudaGetLastError(), "kv8_append_kernel");
}
