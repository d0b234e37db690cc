// New K and V rows into pages of 8-bit codes with one power-of-two scale per (page, KV head).
//
// One CTA per (page that the new rows touch, KV head, K or V, session). It takes the largest
// magnitude of the page's new rows, chooses the scale, brings codes that the page already holds
// to it when it grew, and writes the new rows' codes. Scales are powers of two, so every division
// is exact and a lane is rounded once when it is stored (again only if its page's scale grows;
// e4m3 codes then lose nothing above the subnormal range). Memory bound: an element is read once
// (2 or 4 bytes) and one byte is written; a thread owns 16 adjacent lanes of a row, so both sides
// move in 16-byte pieces; the new rows of a page of up to 64 tokens of 128 bf16 lanes (32 tokens of F32
// lanes; the others are read again) stay in registers between the two passes. Measured, replayed in a
// graph (a call adds 3 us): 4 x 4093 rows of 8 KV heads of 128 bf16 lanes 21.2 us (4.8 TB/s of reads and
// writes; 28.8 us when the second pass read the rows again, 27.9 without the bound on registers, which
// let half as many blocks be resident); 64 sessions of one row each 3.2 us, a launch.
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
    if constexpr (E4M3) {
        unsigned short lo, hi;
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(x[1]), "f"(x[0]));
        asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(x[3]), "f"(x[2]));
        return (unsigned int)lo | ((unsigned int)hi << 16);
    } else {
        // |x| <= 127: adding 1.5 * 2^23 rounds to nearest even and leaves the integer in the low byte
        uint32_t b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(x[i] + 12582912.0f);
        return __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
}

// 16 adjacent lanes of a row as they lie in memory: bf16 pairs or floats. `aligned`: rows lie on 16-byte boundaries.
struct A8Bf16 {
    uint32_t words[8];
};
struct A8Float {
    float lanes[16];
};
__device__ __forceinline__ void a8_load16(const void *base, unsigned long long at, bool aligned, A8Bf16 &raw)
{
    const unsigned short *src = reinterpret_cast<const unsigned short *>(base) + at;
    if (aligned) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src) + i);
            raw.words[4 * i] = v.x, raw.words[4 * i + 1] = v.y, raw.words[4 * i + 2] = v.z, raw.words[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw.words[i] = (uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16);
    }
}
__device__ __forceinline__ void a8_load16(const void *base, unsigned long long at, bool aligned, A8Float &raw)
{
    const float *src = reinterpret_cast<const float *>(base) + at;
    if (aligned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(src) + i);
            raw.lanes[4 * i] = v.x, raw.lanes[4 * i + 1] = v.y, raw.lanes[4 * i + 2] = v.z, raw.lanes[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) raw.lanes[i] = src[i];
    }
}
__device__ __forceinline__ void a8_floats(const A8Bf16 &raw, float (&x)[16])
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[2 * i] = __uint_as_float(raw.words[i] << 16);
        x[2 * i + 1] = __uint_as_float(raw.words[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void a8_floats(const A8Float &raw, float (&x)[16])
{
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = raw.lanes[i];
}

// The largest magnitude as the bits of a float; at least 0x7f800000 when a lane is not finite.
__device__ __forceinline__ uint32_t a8_top(const A8Bf16 &raw)
{
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = __vmaxu2(top, raw.words[i] & 0x7fff7fffu);
    return max(top << 16, top & 0x7fff0000u);
}
__device__ __forceinline__ uint32_t a8_top(const A8Float &raw)
{
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(raw.lanes[i]) & 0x7fffffffu);
    return top;
}
// The largest finite magnitude.
template <typename Raw>
__device__ __forceinline__ uint32_t a8_finite_top(const Raw &raw)
{
    float x[16], top = 0.0f;
    a8_floats(raw, x);
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fabsf(x[i]) < INFINITY ? fmaxf(top, fabsf(x[i])) : top;
    return __float_as_uint(top);
}

// The smallest power of two s >= 2^-126 with amax <= limit * s; limit = (1 + fraction) * 2^shift.
__device__ __forceinline__ float a8_scale(float amax, float limit, int shift)
{
    const int exponent = (int)(__float_as_uint(amax) >> 23) - shift;
    const float s = __uint_as_float((unsigned int)max(exponent, 1) << 23);
    return amax > limit * s ? 2.0f * s : s;
}

constexpr int kA8Resident = 8;   // blocks of an SM: 64 registers a thread

// grid: x = touched page of the session, y = 2 * kv_head + (0: K, 1: V), z = session
template <bool E4M3, typename Raw>
__global__ void __launch_bounds__(kA8Threads, kA8Resident) kv8_append_kernel(const yvx_kv8_append_args a, const int aligned)
{
    constexpr int kA8Held = sizeof(Raw) == sizeof(A8Bf16) ? 4 : 2;
    __shared__ uint32_t warp_top[2][kA8Threads / 32];
    const unsigned int b = blockIdx.z, kv_head = blockIdx.y >> 1, is_value = blockIdx.y & 1u;
    const unsigned long long present = a.kv_tokens ? a.kv_tokens[b] : a.kv_tokens_uniform;
    const unsigned long long fresh = a.new_tokens ? a.new_tokens[b] : a.tokens;
    // Lengths live in device memory: more rows than the launch was made for, or rows behind the
    // session's table row, are recorded and nothing of the session is written.
    if (fresh > a.tokens || present + fresh > (unsigned long long)a.block_table_stride * a.block_tokens) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, YVX_STATUS_CONTRACT);
        return;
    }
    if (!fresh) return;   // its pages are neither looked up nor touched: the slot may be idle, its last page shared
    const unsigned long long index = present / a.block_tokens + blockIdx.x;
    const unsigned long long page_start = index * a.block_tokens;
    if (page_start >= present + fresh) return;
    const int page = a.block_table[(unsigned long long)b * a.block_table_stride + index];   // checked below
    const unsigned long long from = present > page_start ? present : page_start;
    const unsigned long long until = min(present + fresh, page_start + a.block_tokens);
    const unsigned int kept = (unsigned int)(from - page_start), rows = (unsigned int)(until - from);
    const unsigned int chunks = a.head_dim / 16u;
    const void *source = is_value ? a.value : a.key;
    const unsigned long long origin = (unsigned long long)b * a.session_stride + (from - present) * a.token_stride +
                                      (unsigned long long)kv_head * a.head_dim;
    // Up to kA8Held pieces of 16 lanes of a thread stay in registers between the two passes (a whole page of 64
    // tokens of 128 bf16 lanes, half of one of F32 lanes), all loads in flight at once and beside the table's; what is more is read again.
    const unsigned int pieces = rows * chunks;
    auto piece_at = [&](unsigned int piece) {
        return origin + (unsigned long long)(piece / chunks) * a.token_stride + 16u * (piece % chunks);
    };
    Raw raw[kA8Held];
#pragma unroll
    for (int i = 0; i < kA8Held; ++i)
        if (threadIdx.x + i * kA8Threads < pieces) a8_load16(source, piece_at(threadIdx.x + i * kA8Threads), aligned, raw[i]);
    if (page < 0 || (unsigned int)page >= a.pool_blocks) {
        if (threadIdx.x == 0) atomicCAS(a.status, 0, YVX_STATUS_CONTRACT);
        return;
    }
    unsigned char *codes = reinterpret_cast<unsigned char *>(is_value ? a.value_codes : a.key_codes) +
                           (unsigned long long)page * a.code_block_stride + (unsigned long long)kv_head * a.code_head_stride;
    float *scale_slot = (is_value ? a.value_scales : a.key_scales) +
                        (unsigned long long)page * (a.scale_block_stride ? a.scale_block_stride : a.kv_heads) + kv_head;

    const float held = kept ? *scale_slot : 0.0f;
    auto largest = [&](auto of, uint32_t *slots) {
        uint32_t mine = 0u;
#pragma unroll
        for (int i = 0; i < kA8Held; ++i)
            if (threadIdx.x + i * kA8Threads < pieces) mine = max(mine, of(raw[i]));
        for (unsigned int piece = threadIdx.x + kA8Held * kA8Threads; piece < pieces; piece += kA8Threads) {
            Raw more;
            a8_load16(source, piece_at(piece), aligned, more);
            mine = max(mine, of(more));
        }
        mine = __reduce_max_sync(0xffffffffu, mine);
        if ((threadIdx.x & 31u) == 0) slots[threadIdx.x >> 5] = mine;
        __syncthreads();
        uint32_t all = 0u;
#pragma unroll
        for (int w = 0; w < kA8Threads / 32; ++w) all = max(all, slots[w]);
        return all;
    };
    uint32_t top_bits = largest([](const Raw &piece) { return a8_top(piece); }, warp_top[0]);
    const bool finite = top_bits < 0x7f800000u;
    if (!finite) top_bits = largest([](const Raw &piece) { return a8_finite_top(piece); }, warp_top[1]);
    if (!finite && threadIdx.x == 0) atomicCAS(a.status, 0, YVX_STATUS_NONFINITE);
    const float top = __uint_as_float(top_bits);
    const float wanted = E4M3 ? a8_scale(top, 448.0f, 8) : a8_scale(top, 127.0f, 6);
    const float scale = fmaxf(held, wanted);
    if (scale > held && kept) {
        const float ratio = held / scale;
        for (unsigned int i = threadIdx.x; i < kept * chunks; i += kA8Threads) {
            uint4 *slot = reinterpret_cast<uint4 *>(codes + (i / chunks) * a.code_token_stride + 16u * (i % chunks));
            const uint4 was = *slot;
            uint32_t words[4] = {was.x, was.y, was.z, was.w};
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
    auto store = [&](const float (&x)[16], unsigned int piece) {
        uint32_t words[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = finite || fabsf(x[4 * w + e]) < INFINITY ? x[4 * w + e] * inverse : 0.0f;
            words[w] = a8_encode4<E4M3>(y);
        }
        *reinterpret_cast<uint4 *>(codes + (unsigned long long)(kept + piece / chunks) * a.code_token_stride + 16u * (piece % chunks)) =
            make_uint4(words[0], words[1], words[2], words[3]);
    };
#pragma unroll
    for (int i = 0; i < kA8Held; ++i)
        if (threadIdx.x + i * kA8Threads < pieces) {
            float x[16];
            a8_floats(raw[i], x);
            store(x, threadIdx.x + i * kA8Threads);
        }
    for (unsigned int piece = threadIdx.x + kA8Held * kA8Threads; piece < pieces; piece += kA8Threads) {
        Raw more;
        float x[16];
        a8_load16(source, piece_at(piece), aligned, more);
        a8_floats(more, x);
        store(x, piece);
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
    const bool bf16 = a->dtype == YVEX_DTYPE_BF16;
    void (*const kernels[4])(const yvx_kv8_append_args, const int) = {
        kv8_append_kernel<false, A8Float>, kv8_append_kernel<true, A8Float>, kv8_append_kernel<false, A8Bf16>,
        kv8_append_kernel<true, A8Bf16>};
    kernels[(bf16 ? 2 : 0) + (a->code == YVX_KV_E4M3 ? 1 : 0)]<<<grid, kA8Threads, 0, (cudaStream_t)stream>>>(*a, aligned);
    return yvx_cuda_check(cudaGetLastError(), "kv8_append_kernel");
}
