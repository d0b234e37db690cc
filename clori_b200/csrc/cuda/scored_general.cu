// Scored attention for every admitted shape, in F32 throughout: any head_dim up to 256, F32 or
// bf16 rows at any strides, pages of any size, codes of both kinds; and the fold of its splits.
//
// A CTA owns 16 vectors (query rows x heads of one KV head), so a K or V element fetched once is
// used 16 times, and walks its split in tiles of 32 tokens: K and V are decoded into shared
// memory as floats, a thread computes the scores of one token against four vectors, a warp runs
// the softmax of four vectors, a thread accumulates one or two head dimensions of all 16. Bound
// by the FMA pipe and shared-memory reads: 64 sessions of 512 to 32768 tokens of e4m3 codes 8.3 ms (22 times the decode
// kernel), 4 x 1531 rows 10.4 ms (61 times the prompt kernel). It is the kernel of the F32 contract, of head
// dimensions other than 128 and of layouts that the tiled copies cannot describe.
#include "scored.cuh"

#include <cuda_fp8.h>

namespace yvx {

constexpr int kSgVectors = 16, kSgTokens = 32, kSgThreads = 128;

template <int KV>
struct SgElement {
    typedef float type;
};
template <>
struct SgElement<1> {
    typedef __nv_bfloat16 type;
};
template <>
struct SgElement<2> {
    typedef unsigned char type;
};
template <>
struct SgElement<3> {
    typedef signed char type;
};

__device__ __forceinline__ float sg_value(float x) { return x; }
__device__ __forceinline__ float sg_value(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float sg_value(signed char x) { return (float)x; }
__device__ __forceinline__ float sg_value(unsigned char x)
{
    __nv_fp8_e4m3 code;
    code.__x = x;
    return (float)code;
}

// KV: 0 F32, 1 bf16, 2 e4m3 codes, 3 integer codes. grid: x = kv_head * row_tiles + row_tile,
// y = split, z = session.
template <int KV>
__global__ void __launch_bounds__(kSgThreads) scored_general_kernel(const yvx_scored_problem p)
{
    typedef typename SgElement<KV>::type Element;
    extern __shared__ float sg_smem[];
    const unsigned int hd = p.head_dim, kpitch = hd + 1u;
    float *q_smem = sg_smem;                          // [16][hd]
    float *k_smem = q_smem + kSgVectors * hd;         // [32][hd + 1]: a token per thread, no conflicts
    float *v_smem = k_smem + kSgTokens * kpitch;      // [32][hd]
    float *s_smem = v_smem + kSgTokens * hd;          // [16][32]
    float *keep_smem = s_smem + kSgVectors * kSgTokens;
    float *l_smem = keep_smem + kSgVectors, *m_smem = l_smem + kSgVectors;

    const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const unsigned int group = p.query_heads / p.kv_heads;
    const unsigned long long vectors = (unsigned long long)p.query_rows * group;
    const unsigned int row_tiles = (unsigned int)((vectors + kSgVectors - 1u) / kSgVectors);
    const unsigned int kv_head = blockIdx.x / row_tiles, row_tile = blockIdx.x % row_tiles;
    const unsigned int b = blockIdx.z, split = blockIdx.y;
    const unsigned int kv_tokens = admitted_kv_tokens(p.kv_tokens, b, p.kv_tokens_uniform, p.kv_tokens_max, p.status);
    const long long query_start = scored_query_start(p, b, kv_tokens);
    const unsigned long long vector_base = (unsigned long long)row_tile * kSgVectors;
    const unsigned int live = (unsigned int)min((unsigned long long)kSgVectors, vectors - vector_base);
    int hull_first, hull_end, t0, t1;
    scored_hull(p, b, (unsigned int)(vector_base / group), (unsigned int)((vector_base + live - 1u) / group) + 1u,
                kv_tokens, query_start, hull_first, hull_end);
    scored_split(p, split, hull_first, hull_end, t0, t1);

    auto item_of = [&](unsigned int i) {
        const unsigned long long v = vector_base + i;
        return ((unsigned long long)b * p.query_rows + v / group) * p.query_heads + kv_head * group + v % group;
    };
    if (t0 >= t1) {
        for (unsigned int i = warp; i < live; i += kSgThreads / 32) scored_store_empty(p, item_of(i), split, lane, 32u);
        return;
    }
    const unsigned long long head_stride = p.query_head_stride ? p.query_head_stride : hd;
    for (unsigned int i = threadIdx.x; i < kSgVectors * hd; i += kSgThreads) {
        const unsigned int vi = i / hd, d = i % hd;
        float x = 0.0f;
        if (vi < live) {
            const unsigned long long v = vector_base + vi;
            const unsigned long long at = (unsigned long long)b * p.query_session_stride + (v / group) * p.query_row_stride +
                                          (kv_head * group + v % group) * head_stride + d;
            x = p.query_dtype == YVEX_DTYPE_BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p.query)[at])
                                                 : reinterpret_cast<const float *>(p.query)[at];
        }
        q_smem[i] = x;
    }
    // the vectors whose scores this thread computes: 4 * warp .. + 3
    ScoredRange range[4];
    float slope[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned int vi = 4u * warp + i;
        range[i].first = range[i].end = 0;
        range[i].position = 0;
        slope[i] = 0.0f;
        if (vi < live) {
            const unsigned long long v = vector_base + vi;
            range[i] = scored_range(p, b, (unsigned int)(v / group), kv_tokens, query_start);
            if (p.slopes) slope[i] = p.slopes[kv_head * group + v % group];
        }
    }
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.0f;
    float acc[2][kSgVectors];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < kSgVectors; ++i) acc[h][i] = 0.0f;

    for (int tile = t0; tile < t1; tile += kSgTokens) {
        __syncthreads();
        for (unsigned int token = warp; token < kSgTokens; token += kSgThreads / 32) {
            const int t = tile + (int)token;
            const Element *key = nullptr, *value = nullptr;
            float key_scale = 1.0f, value_scale = 1.0f;
            if (t < t1 && t >= hull_first) {  // pages in front of the first visible token may be gone
                unsigned long long outer = b, inner = (unsigned long long)t;
                if (p.block_table) {
                    const int page = scored_page(p, b, (unsigned int)t / p.block_tokens);
                    outer = (unsigned long long)(page < 0 ? 0 : page);
                    inner = (unsigned int)t % p.block_tokens;
                    if (KV >= 2) {
                        const unsigned long long at = outer * (p.scale_block_stride ? p.scale_block_stride : p.kv_heads) + kv_head;
                        key_scale = p.key_scales[at];
                        value_scale = p.value_scales[at];
                    }
                }
                key = reinterpret_cast<const Element *>(p.key) + outer * p.key_outer_stride + inner * p.key_token_stride +
                      kv_head * p.key_head_stride;
                value = reinterpret_cast<const Element *>(p.value) + outer * p.value_outer_stride +
                        inner * p.value_token_stride + kv_head * p.value_head_stride;
            }
            for (unsigned int d = lane; d < hd; d += 32u) {
                k_smem[token * kpitch + d] = key ? sg_value(key[d]) * key_scale : 0.0f;
                v_smem[token * hd + d] = value ? sg_value(value[d]) * value_scale : 0.0f;
            }
        }
        __syncthreads();
        // scores of token `lane` against this warp's four vectors
        float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const float *k_row = k_smem + lane * kpitch, *q_rows = q_smem + 4u * warp * hd;
        for (unsigned int d = 0; d < hd; ++d) {
            const float k = k_row[d];
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = fmaf(q_rows[i * hd + d], k, z[i]);
        }
        const int t = tile + (int)lane;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float s = z[i] * p.scale;
            if (p.cap > 0.0f) s = p.cap * tanhf(s / p.cap);
            if (p.slopes) s -= slope[i] * (float)abs(range[i].position - t);
            s = t >= range[i].first && t < range[i].end ? s * kScoredLog2e : -INFINITY;
            // a NaN that a row sees has to reach its result: max() alone would drop it
            const float top = warp_max(s != s ? INFINITY : s);
            const float fresh = fmaxf(m[i], top);
            const float base = fresh == -INFINITY ? 0.0f : fresh;
            const float keep = m[i] == -INFINITY ? 0.0f : exp2f(m[i] - base);
            const float weight = exp2f(s - base);
            l[i] = l[i] * keep + warp_sum(weight);
            m[i] = fresh;
            s_smem[(4u * warp + i) * kSgTokens + lane] = weight;
            if (lane == 0) keep_smem[4u * warp + i] = keep;
        }
        __syncthreads();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned int d = threadIdx.x + h * kSgThreads;
            if (d >= hd) continue;
#pragma unroll
            for (int i = 0; i < kSgVectors; ++i) acc[h][i] *= keep_smem[i];
            for (unsigned int token = 0; token < kSgTokens; ++token) {
                const float v = v_smem[token * hd + d];
#pragma unroll
                for (int i = 0; i < kSgVectors; ++i) {
                    // a weight of zero takes nothing, whatever lies in the row behind the mask
                    const float weight = s_smem[i * kSgTokens + token];
                    acc[h][i] = weight != 0.0f ? fmaf(weight, v, acc[h][i]) : acc[h][i];
                }
            }
        }
    }
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            l_smem[4u * warp + i] = l[i];
            m_smem[4u * warp + i] = m[i];
        }
    }
    __syncthreads();
    for (unsigned int i = 0; i < live; ++i) {
        const unsigned long long item = item_of(i);
        const float sum = l_smem[i];
        float *part = p.max_splits > 1u ? scored_partial(p, item, split) : nullptr;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned int d = threadIdx.x + h * kSgThreads;
            if (d >= hd) continue;
            float x = 0.0f;
#pragma unroll
            for (int j = 0; j < kSgVectors; ++j) x = j == (int)i ? acc[h][j] : x;
            if (part) {
                part[d] = x;
                continue;
            }
            x = sum == 0.0f ? 0.0f : x / sum;
            if (!isfinite(x)) atomicCAS(p.status, 0, YVX_STATUS_NONFINITE);
            store_output(p.output, p.output_dtype, item * hd + d, x);
        }
        if (part && threadIdx.x == 0) {
            part[hd] = m_smem[i];
            part[hd + 1] = sum;
        }
    }
}

// What a split's weight is taken from: its maximum; -inf when it saw nothing. A sum that is NaN (a row saw a NaN) stands
// above every maximum, which a NaN may not have moved, so that no fold leaves it out: its weight becomes inf - inf.
__device__ __forceinline__ float scored_split_height(float m, float l)
{
    return l == 0.0f ? -INFINITY : l != l ? INFINITY : m;
}

// One CTA per item. The splits' weights go to shared memory once; then eight warps share the splits, a lane
// owns four adjacent dims at a time and the rows of four splits are in flight together. Warps are added in
// order: the result depends on the inputs alone.
constexpr int kScThreads = 256, kScWarps = kScThreads / 32, kScBatch = 4;

__global__ void __launch_bounds__(kScThreads) scored_combine_kernel(const yvx_scored_problem p)
{
    extern __shared__ float weight[];               // [max_splits]
    __shared__ float total[kScWarps][256 + 4];
    __shared__ float warp_top[kScWarps], warp_sum_of[kScWarps];
    const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, hd = p.head_dim;
    const unsigned long long item = blockIdx.x;
    pdl_wait();
    const float *parts = scored_partial(p, item, 0u);
    const unsigned long long pitch = hd + 4ull;
    float top = -INFINITY;
    for (unsigned int j = threadIdx.x; j < p.max_splits; j += kScThreads) {
        const float m = parts[j * pitch + hd], l = parts[j * pitch + hd + 1];
        const float height = scored_split_height(m, l);
        weight[j] = height;
        top = fmaxf(top, height);
    }
    top = warp_max(top);
    if (lane == 0) warp_top[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kScWarps; ++w) top = fmaxf(top, warp_top[w]);
    float sum = 0.0f;
    for (unsigned int j = threadIdx.x; j < p.max_splits; j += kScThreads) {
        const float m = weight[j], w = m == -INFINITY ? 0.0f : exp2f(m - top);
        weight[j] = w;
        if (w != 0.0f) sum += parts[j * pitch + hd + 1] * w;
    }
    sum = warp_sum(sum);
    if (lane == 0) warp_sum_of[warp] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kScWarps; ++w) sum += warp_sum_of[w];
    for (unsigned int d0 = 0; d0 < hd; d0 += 128u) {
        const unsigned int d = d0 + 4u * lane;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (hd % 4u == 0u ? d < hd : false) {
            for (unsigned int j0 = warp; j0 < p.max_splits; j0 += kScWarps * kScBatch) {
                float4 o[kScBatch];
                float w[kScBatch];
#pragma unroll
                for (int u = 0; u < kScBatch; ++u) {
                    const unsigned int j = j0 + u * kScWarps;
                    w[u] = j < p.max_splits ? weight[j] : 0.0f;
                    if (w[u] != 0.0f) o[u] = *reinterpret_cast<const float4 *>(parts + j * pitch + d);  // rows of weight 0 hold anything
                }
#pragma unroll
                for (int u = 0; u < kScBatch; ++u)
                    if (w[u] != 0.0f) {
                        acc[0] = fmaf(o[u].x, w[u], acc[0]);
                        acc[1] = fmaf(o[u].y, w[u], acc[1]);
                        acc[2] = fmaf(o[u].z, w[u], acc[2]);
                        acc[3] = fmaf(o[u].w, w[u], acc[3]);
                    }
            }
        } else {
            for (unsigned int j = warp; j < p.max_splits; j += kScWarps)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d + i < hd && weight[j] != 0.0f) acc[i] = fmaf(parts[j * pitch + d + i], weight[j], acc[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (d + i < hd) total[warp][d + i] = acc[i];
    }
    __syncthreads();
    for (unsigned int d = threadIdx.x; d < hd; d += kScThreads) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < kScWarps; ++w) x += total[w][d];
        x = sum == 0.0f ? 0.0f : x / sum;
        if (!isfinite(x)) atomicCAS(p.status, 0, YVX_STATUS_NONFINITE);
        store_output(p.output, p.output_dtype, item * hd + d, x);
    }
}

// The same with a warp for each item, for up to 32 splits: a lane holds one split's weight, then four adjacent dims.
__global__ void __launch_bounds__(kScThreads) scored_combine_warp_kernel(const yvx_scored_problem p, const unsigned int items)
{
    const unsigned int lane = threadIdx.x & 31u, item = blockIdx.x * kScWarps + (threadIdx.x >> 5), hd = p.head_dim;
    if (item >= items) return;   // uniform over the warp; whole warps have nothing to wait for
    pdl_wait();
    const float *parts = scored_partial(p, item, 0u);
    const unsigned int pitch = hd + 4u;
    const float l = lane < p.max_splits ? parts[lane * pitch + hd + 1] : 0.0f;
    const float m = l == 0.0f ? -INFINITY : scored_split_height(parts[lane * pitch + hd], l);
    const float top = warp_max(m), weight = m == -INFINITY ? 0.0f : exp2f(m - top), sum = warp_sum(l * weight);
    for (unsigned int d0 = 0; d0 < hd; d0 += 128u) {
        const unsigned int d = d0 + 4u * lane;
        const bool wide = hd % 4u == 0u && d < hd;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (unsigned int j0 = 0; j0 < p.max_splits; j0 += kScBatch) {
            float o[kScBatch][4];
            float w[kScBatch];
#pragma unroll
            for (int u = 0; u < kScBatch; ++u) {
                const unsigned int j = j0 + u;
                w[u] = __shfl_sync(0xffffffffu, weight, j & 31u);
                if (j >= p.max_splits) w[u] = 0.0f;
                const float *row = parts + j * pitch + d;
#pragma unroll
                for (int i = 0; i < 4; ++i) o[u][i] = 0.0f;
                if (w[u] != 0.0f) {   // rows of weight 0 hold anything
                    if (wide) *reinterpret_cast<float4 *>(o[u]) = *reinterpret_cast<const float4 *>(row);
                    else
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (d + i < hd) o[u][i] = row[i];
                }
            }
#pragma unroll
            for (int u = 0; u < kScBatch; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = fmaf(o[u][i], w[u], acc[i]);
        }
        bool finite = true;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (d + i >= hd) continue;
            const float x = sum == 0.0f ? 0.0f : acc[i] / sum;
            finite = finite && isfinite(x);
            store_output(p.output, p.output_dtype, (unsigned long long)item * hd + d + i, x);
        }
        if (!finite) atomicCAS(p.status, 0, YVX_STATUS_NONFINITE);
    }
}

int scored_combine_launch(const yvx_scored_problem &p, cudaStream_t stream)
{
    const unsigned long long items = (unsigned long long)p.sessions * p.query_rows * p.query_heads;
    // A block for an item has more loads in flight, a warp for an item wastes no threads: 32 items of 32 splits 10.1 us
    // (whole call) against 13.9, 640 of 18 102.1 / 103.7; 2560 of 4 388 / 381, 9600 of 7 209 / 190, 16384 of 2 180 / 143.
    const bool warps = p.max_splits <= 32u && items >= 2048ull;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned int)(warps ? (items + kScWarps - 1) / kScWarps : items), 1, 1);
    config.blockDim = dim3(kScThreads, 1, 1);
    config.dynamicSmemBytes = warps ? 0 : p.max_splits * sizeof(float);  // the plan keeps them within 8192
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    if (warps)
        return yvx_cuda_check(cudaLaunchKernelEx(&config, scored_combine_warp_kernel, p, (unsigned int)items), "scored_combine_warp_kernel");
    return yvx_cuda_check(cudaLaunchKernelEx(&config, scored_combine_kernel, p), "scored_combine_kernel");
}

int scored_general_launch(const yvx_scored_problem &p, cudaStream_t stream)
{
    const unsigned long long vectors = (unsigned long long)p.query_rows * (p.query_heads / p.kv_heads);
    const unsigned long long tiles = (vectors + kSgVectors - 1ull) / kSgVectors * p.kv_heads;
    const unsigned int hd = p.head_dim;
    const int smem = (int)(sizeof(float) * (kSgVectors * hd + kSgTokens * (hd + 1u) + kSgTokens * hd +
                                            kSgVectors * kSgTokens + 3 * kSgVectors));
    const int kind = p.kv_code == YVX_KV_E4M3 ? 2 : p.kv_code == YVX_KV_I8 ? 3 : p.kv_dtype == YVEX_DTYPE_BF16 ? 1 : 0;
    void (*const kernels[4])(const yvx_scored_problem) = {scored_general_kernel<0>, scored_general_kernel<1>,
                                                          scored_general_kernel<2>, scored_general_kernel<3>};
    YVX_CUDA_TRY(cudaFuncSetAttribute((const void *)kernels[kind], cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    kernels[kind]<<<dim3((unsigned int)tiles, p.max_splits, p.sessions), kSgThreads, smem, stream>>>(p);
    return yvx_cuda_check(cudaGetLastError(), "scored_general_kernel");
}

}  // namespace yvx
