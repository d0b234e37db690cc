// Scored attention for few query rows over long caches: decode and verify, head_dim 128, bf16
// queries, K and V as bf16 rows or 8-bit codes, contiguous or in pages of 16, 32 or 64 n tokens.
//
// Bandwidth-shaped split-KV kernel. A CTA owns up to 16 vectors (query rows x heads of one KV
// head) and one split; a producer warp streams 64-token tiles of K and V into a ring with tiled
// copies (one per page and operand; 128-byte swizzle, so every shared-memory read below is free of
// bank conflicts) together with the pages' scales, and four consumer warps own 16 tokens of each
// tile: S = Q K^T and O += P V as mma.sync m16n8k16 with the vectors in M. M is at most 16, so the
// 5th-generation tensor cores have nothing to win: the memory system is the bound.
//
// Codes. A lane of 8 bits becomes an exact f16. A page's K scale multiplies the scores; its V scale
// multiplies the weights. Each row has a reference of its own for these products, as lazy as the maximum of
// the scores: the operand of P V stays inside f16 however far the V scales of the pages that different rows
// see lie apart, and the arithmetic of a code costs one conversion and nothing else. Queries are brought to f16 by a power of two per vector
// (exact but for lanes below 2^-29 of the vector's largest). The order of head dimensions inside a
// k-step is free, so a thread takes 32 adjacent dims of its token with two 16-byte reads.
// Weights: the maximum is lazy, it moves when a score exceeds it by 2^4 (codes) or 2^8, and the
// weights of codes carry a factor 2^11 (at most 2^15): one rounding to 11 bits, full precision down
// to 2^-25 of the largest. bf16 caches carry a weight as head + tail, 16 bits.
//
// Measured, a call between events (replayed in a graph): 64 sessions of 512 to 32768 tokens, 8 KV heads, groups of 5, e4m3
// 433 us (390) for 2.16 GB, the same copies without the arithmetic 327 in a graph. 131072 tokens of int8 codes, 16 vectors,
// capped: 78 us (76) for 268 MB, its copies alone 55. 64 sessions behind a window of 4096, bf16 rows, capped: 163 us (152)
// for 1.0 GB. One session of 4096 tokens, e4m3: 12.3 us (10.2), of which the two launches and their first loads are most.
// A row's own reference for weights times V scales costs 1.5 to 3 % (426 -> 433, 75.7 -> 78). A pass waits for its matrix
// instructions and conversions (an SM issues in 40 % of its cycles), which two tiles of codes a pass hide in part;
// with 8 warps an SM has no others to turn to.
#include "scored.cuh"

namespace yvx {

constexpr int kSdTokens = 64, kSdDim = 128, kSdWarps = 4, kSdThreads = (kSdWarps + 1) * 32;
constexpr int kSdQRowBytes = kSdDim * 2 + 16;          // padded rows
constexpr int kSdMergeFloats = kSdDim + 4;
constexpr int kSdRingBytes = 96 * 1024;

struct SdMaps {
    CUtensorMap key, value;
};

template <int CODE>
struct SdShape {
    static constexpr int operand_bytes = kSdTokens * kSdDim * (CODE ? 1 : 2);  // one K or V tile
    static constexpr int stages = kSdRingBytes / (2 * operand_bytes);
    static constexpr int pair = CODE ? 2 : 1;
};
constexpr int kSdMaxStages = SdShape<1>::stages;
constexpr int kSdSmemBytes = kSdRingBytes + 16 * kSdQRowBytes + kSdMaxStages * kSdWarps * 8 + kSdMaxStages * 16 + 64 + 64 + 1024;

// 16 bits of code (two lanes) -> f16x2, four lanes -> two of them.
template <int CODE>
__device__ __forceinline__ void sd_codes(uint32_t word, uint32_t &lo, uint32_t &hi)
{
    if (CODE == YVX_KV_E4M3) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
            "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(word));
    } else {
        // a byte u under the exponent 0x64 reads 1024 + u; u = lane + 128
        uint32_t a, b;
        const uint32_t biased = word ^ 0x80808080u;
        asm("prmt.b32 %0, %1, %2, 0x4140;" : "=r"(a) : "r"(biased), "r"(0x64646464u));
        asm("prmt.b32 %0, %1, %2, 0x4342;" : "=r"(b) : "r"(biased), "r"(0x64646464u));
        asm("sub.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
        asm("sub.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
    }
}

// Above this cap the exponential's error, a few 2^-23 of the cap, would count: a few 2^-17 there, as much as the
// rounding of a bf16 call's weights.
constexpr float kSdWideCap = 64.0f;

// tanh(x) / x of x^2 for |x| <= 0.6, fitted for this kernel: relative error at most 1.7e-7.
__device__ __forceinline__ float sd_tanh_ratio(float square)
{
    float r = 0.015475619f;
    r = fmaf(r, square, -0.05210145f);
    r = fmaf(r, square, 0.13310167f);
    r = fmaf(r, square, -0.33332309f);
    return fmaf(r, square, 0.99999994f);
}

// grid: x = split, y = kv_head * row_tiles + row_tile, z = session. `unit`: tokens of one tiled copy
// (a page or 64). `head_inner`: the maps order their middle dimensions (head, token). WIDE: the cap is above kSdWideCap.
template <int CODE, bool WIDE>
__global__ void __launch_bounds__(kSdThreads, 2)
scored_decode_kernel(const yvx_scored_problem p, const __grid_constant__ SdMaps maps, const int unit, const int head_inner)
{
    typedef SdShape<CODE> Shape;
    constexpr int kStages = Shape::stages, kOperand = Shape::operand_bytes;
    extern __shared__ unsigned char sd_raw[];
    // the 128-byte swizzle is a function of address bits 4..9
    unsigned char *ring = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(sd_raw) + 1023u) & ~uintptr_t(1023));
    unsigned char *q_smem = ring + kSdRingBytes;
    float2 *scale_smem = reinterpret_cast<float2 *>(q_smem + 16 * kSdQRowBytes);   // [stage][warp]: K, V
    uint64_t *full = reinterpret_cast<uint64_t *>(scale_smem + kSdMaxStages * kSdWarps);
    uint64_t *empty = full + kSdMaxStages;
    float *q_unscale = reinterpret_cast<float *>(empty + kSdMaxStages);            // [16]

    const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const unsigned int group = p.query_heads / p.kv_heads, vectors = p.query_rows * group;
    const unsigned int row_tiles = (vectors + 15u) / 16u;
    const unsigned int kv_head = blockIdx.y / row_tiles, row_tile = blockIdx.y % row_tiles;
    const unsigned int b = blockIdx.z, split = blockIdx.x;
    const unsigned int kv_tokens = admitted_kv_tokens(p.kv_tokens, b, p.kv_tokens_uniform, p.kv_tokens_max, p.status);
    const long long query_start = scored_query_start(p, b, kv_tokens);
    const unsigned int vector_base = row_tile * 16u, live = min(16u, vectors - vector_base);
    int hull_first, hull_end, t0, t1;
    scored_hull(p, b, vector_base / group, (vector_base + live - 1u) / group + 1u, kv_tokens, query_start, hull_first, hull_end);
    scored_split(p, split, hull_first, hull_end, t0, t1);
    auto item_of = [&](unsigned int i) {
        const unsigned int v = vector_base + i;
        return ((unsigned long long)b * p.query_rows + v / group) * p.query_heads + kv_head * group + v % group;
    };
    if (t0 >= t1) {
        for (unsigned int i = warp; i < live; i += kSdThreads / 32) scored_store_empty(p, item_of(i), split, lane, 32u);
        return;
    }
    const unsigned int tiles = (unsigned int)(t1 - t0 + kSdTokens - 1) / kSdTokens;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kSdWarps);
        }
        fence_barrier_init();
    }
    __syncthreads();

    if (warp == kSdWarps) {
        // ---- producer: 32 table entries (and scales) at a time, a lane each ----------------------
        const unsigned int per_tile = (unsigned int)(kSdTokens / unit), batch_tiles = 32u / per_tile;
        int page = 0, inner = 0;
        float key_scale = 0.0f, value_scale = 0.0f;
        for (unsigned int i = 0; i < tiles; ++i) {
            const unsigned int slot = i % batch_tiles;
            if (slot == 0u) {
                const int token = t0 + (int)(i * kSdTokens) + (int)lane * unit;
                page = -1;
                // pages in front of the first visible token may be gone: not looked up, not loaded
                if (token < t1 && token + unit > hull_first) {
                    if (p.block_table) {
                        page = scored_page(p, b, (unsigned int)token / p.block_tokens);
                        if (page < 0) page = 0;
                        inner = (int)((unsigned int)token % p.block_tokens);
                        if (CODE) {
                            const unsigned long long at =
                                (unsigned long long)page * (p.scale_block_stride ? p.scale_block_stride : p.kv_heads) + kv_head;
                            key_scale = p.key_scales[at];
                            value_scale = p.value_scales[at];
                        }
                    } else {
                        page = (int)b;
                        inner = token;
                    }
                }
            }
            const unsigned int stage = i % kStages;
            if (i >= (unsigned int)kStages && !__all_sync(0xffffffffu, mbar_wait(&empty[stage], ((i / kStages) - 1u) & 1u))) {
                if (lane == 0) atomicCAS(p.status, 0, YVX_STATUS_TIMEOUT);
                return;
            }
            const unsigned int mine = slot * per_tile + min(lane, per_tile - 1u);
            const int unit_page = __shfl_sync(0xffffffffu, page, mine), unit_inner = __shfl_sync(0xffffffffu, inner, mine);
            const unsigned int loaded = __ballot_sync(0xffffffffu, lane < per_tile && unit_page >= 0);
            unsigned char *k_dst = ring + stage * 2 * kOperand, *v_dst = k_dst + kOperand;
            if (lane < per_tile && unit_page >= 0) {
                const int c1 = head_inner ? (int)kv_head : unit_inner, c2 = head_inner ? unit_inner : (int)kv_head;
                const uint32_t at = lane * (uint32_t)unit * 128u;
                tma_load_4d(k_dst + at, &maps.key, &full[stage], 0, c1, c2, unit_page);
                if (!CODE) tma_load_4d(k_dst + kOperand / 2 + at, &maps.key, &full[stage], 64, c1, c2, unit_page);
                tma_load_4d(v_dst + at, &maps.value, &full[stage], 0, c1, c2, unit_page);
                if (!CODE) tma_load_4d(v_dst + kOperand / 2 + at, &maps.value, &full[stage], 64, c1, c2, unit_page);
            }
            if (CODE) {
                // meanwhile the scales of the 16 tokens of consumer warp `lane`; a unit that is not loaded: 0
                const unsigned int of_warp = slot * per_tile + (16u * min(lane, 3u)) / (unsigned int)unit;
                const float ks = __shfl_sync(0xffffffffu, key_scale, of_warp), vs = __shfl_sync(0xffffffffu, value_scale, of_warp);
                const int there = __shfl_sync(0xffffffffu, page, of_warp);
                if (lane < (unsigned int)kSdWarps)
                    scale_smem[stage * kSdWarps + lane] = there >= 0 ? make_float2(ks, vs) : make_float2(0.0f, 0.0f);
            }
            // the phase ends with this arrival, the bytes may have landed before
            __syncwarp();
            if (lane == 0) mbar_expect_tx(&full[stage], (uint32_t)__popc(loaded) * (uint32_t)unit * kSdDim * 2u * (CODE ? 1u : 2u));
        }
        return;
    }

    // ---- consumers ------------------------------------------------------------------------------
    const unsigned int g = lane >> 2, c = lane & 3u;
    // queries into shared memory: bf16 as they are, or f16 after a power of two that brings the vector's
    // largest lane to [2^14, 2^15); a warp per row, 4 dims per lane
    for (unsigned int row = warp; row < 16u; row += kSdWarps) {
        uint2 raw = make_uint2(0u, 0u);
        if (row < live) {
            const unsigned int v = vector_base + row;
            raw = *reinterpret_cast<const uint2 *>(
                reinterpret_cast<const __nv_bfloat16 *>(p.query) + (unsigned long long)b * p.query_session_stride +
                (unsigned long long)(v / group) * p.query_row_stride +
                (unsigned long long)(kv_head * group + v % group) * (p.query_head_stride ? p.query_head_stride : kSdDim) + 4u * lane);
        }
        if (CODE) {
            const float x0 = __uint_as_float(raw.x << 16), x1 = __uint_as_float(raw.x & 0xffff0000u);
            const float x2 = __uint_as_float(raw.y << 16), x3 = __uint_as_float(raw.y & 0xffff0000u);
            const float top = warp_max(fmaxf(fmaxf(fabsf(x0), fabsf(x1)), fmaxf(fabsf(x2), fabsf(x3))));
            // exponent field of the largest lane, kept where the factor and its inverse are normal numbers
            const int e = min(max((int)(__float_as_uint(top) >> 23), 16), 254);
            const float up = __uint_as_float((unsigned int)min(127 + 14 + 127 - e, 254) << 23);
            raw.x = pack_f16(x0 * up, x1 * up);
            raw.y = pack_f16(x2 * up, x3 * up);
            if (lane == 0) q_unscale[row] = 1.0f / up;
        }
        *reinterpret_cast<uint2 *>(q_smem + row * kSdQRowBytes + 8u * lane) = raw;
    }
    named_barrier(1, kSdWarps * 32);
    uint32_t qa[8][4];
    float mul[2] = {p.scale, p.scale};    // raw product -> logit (natural units)
    if (CODE) {
        // dims 32c .. 32c+31 of rows g and g + 8; k-step s takes the four at 32c + 4s
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint4 a = *reinterpret_cast<const uint4 *>(q_smem + g * kSdQRowBytes + 64u * c + 16u * i);
            const uint4 d = *reinterpret_cast<const uint4 *>(q_smem + (g + 8u) * kSdQRowBytes + 64u * c + 16u * i);
            qa[2 * i][0] = a.x, qa[2 * i][2] = a.y, qa[2 * i + 1][0] = a.z, qa[2 * i + 1][2] = a.w;
            qa[2 * i][1] = d.x, qa[2 * i][3] = d.y, qa[2 * i + 1][1] = d.z, qa[2 * i + 1][3] = d.w;
        }
        mul[0] *= q_unscale[g];
        mul[1] *= q_unscale[g + 8u];
    } else {
        const unsigned int j = lane >> 3, i = lane & 7u;
        const uint32_t base = smem_u32(q_smem) + (8u * (j & 1u) + i) * kSdQRowBytes + 16u * (j >> 1);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) ldmatrix_x4(qa[ks], base + ks * 32u);
    }
    // this thread's rows, and the tokens that every live row of the CTA sees
    int first[2], end[2], position[2];
    float slope[2];
    int inner_first = 0, inner_end = 0x7fffffff;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned int row = g + 8u * h;
        first[h] = 0x7fffffff, end[h] = 0, position[h] = 0, slope[h] = 0.0f;
        if (row < live) {
            const unsigned int v = vector_base + row;
            const ScoredRange r = scored_range(p, b, v / group, kv_tokens, query_start);
            first[h] = r.first, end[h] = r.end, position[h] = r.position;
            if (p.slopes) slope[h] = p.slopes[kv_head * group + v % group];
            inner_first = max(inner_first, r.first);
            inner_end = min(inner_end, r.end);
        }
    }
    inner_first = __reduce_max_sync(0xffffffffu, inner_first);
    inner_end = __reduce_min_sync(0xffffffffu, inner_end);

    constexpr float kSlack = CODE ? 4.0f : 8.0f, kLift = CODE ? 11.0f : 0.0f;
    const bool capped = p.cap > 0.0f, biased = p.slopes != nullptr;
    const float inverse_cap = capped ? 1.0f / p.cap : 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    // codes: a row's accumulators count in 2^(v_ref - kLift), and its weights are multiplied by v_unit = 2^(m - v_ref) and
    // the page's V scale on their way to f16
    float v_ref[2] = {-INFINITY, -INFINITY}, v_unit[2] = {0.0f, 0.0f};
    float o[16][4];
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.0f;

    // kPair tiles per pass: their scores and weights are independent, which hides the latency of the matrix
    // and conversion chains (a warp's issue slots are 40 % busy with one tile of codes at a time)
    constexpr int kPair = Shape::pair, kCols = 2 * kPair;
    for (unsigned int i = 0; i < tiles; i += kPair) {
        unsigned int stage[kPair];
        bool there[kPair], ok = true;
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
            there[u] = i + u < tiles;
            stage[u] = (i + u) % kStages;
            if (there[u]) ok = ok && mbar_wait(&full[stage[u]], ((i + u) / kStages) & 1u);
        }
        if (!ok) {
            atomicCAS(p.status, 0, YVX_STATUS_TIMEOUT);
            break;
        }
        const int token0 = t0 + (int)(i * kSdTokens) + 16 * (int)warp;   // tile u: + 64 u
        float2 scales[kPair];
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
            scales[u] = make_float2(0.0f, 0.0f);
            if (CODE && there[u]) scales[u] = scale_smem[stage[u] * kSdWarps + warp];
        }

        // ---- S = Q K^T over 16 tokens of a tile: column 8 n + j of tile u is its token 8 n + j ------
        float sc[kCols][4];
#pragma unroll
        for (int n = 0; n < kCols; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] = 0.0f;
        // (consecutive matrix instructions go to different accumulators: each of them has a long latency)
        if (CODE) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint4 kq[kCols];
#pragma unroll
                for (int n = 0; n < kCols; ++n) {
                    // a tile behind the split's end stands in for itself with the first one; it is masked below
                    const unsigned char *k_tile = ring + stage[there[n >> 1] ? n >> 1 : 0] * 2 * kOperand;
                    const unsigned int row = 16u * warp + 8u * (n & 1) + g;
                    kq[n] = *reinterpret_cast<const uint4 *>(k_tile + row * 128u + (((2u * c + half) ^ (row & 7u)) << 4));
                }
#pragma unroll
                for (int w = 0; w < 4; ++w)
#pragma unroll
                    for (int n = 0; n < kCols; ++n) {
                        const uint32_t words[4] = {kq[n].x, kq[n].y, kq[n].z, kq[n].w};
                        uint32_t b0, b1;
                        sd_codes<CODE>(words[w], b0, b1);
                        mma_f16(sc[n], qa[4 * half + w], b0, b1);
                    }
            }
        } else {
            const uint32_t k_base = smem_u32(ring + stage[0] * 2 * kOperand);
            const unsigned int j = lane >> 3, r = lane & 7u;
            const unsigned int token = 16u * warp + 8u * (j >> 1) + r;
            float odd[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) odd[n][e] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < 8; ks += 2) {
                uint32_t kb[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const unsigned int chunk = 2u * ((ks + i) & 3) + (j & 1u);
                    ldmatrix_x4(kb[i], k_base + (ks >> 2) * (kOperand / 2) + token * 128u + ((chunk ^ (token & 7u)) << 4));
                }
                mma_bf16(sc[0], qa[ks], kb[0][0], kb[0][1]);
                mma_bf16(sc[1], qa[ks], kb[0][2], kb[0][3]);
                mma_bf16(odd[0], qa[ks + 1], kb[1][0], kb[1][1]);
                mma_bf16(odd[1], qa[ks + 1], kb[1][2], kb[1][3]);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] += odd[n][e];
        }
        // ---- the score rule, in log2 units --------------------------------------------------------
        if (capped || biased) {
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float z = sc[n][e] * (mul[e >> 1] * (CODE ? scales[n >> 1].x : 1.0f));
                    if (capped) {
                        // tanh from one exponential: 1 - 2 / (e^2x + 1), absolute error a few 2^-23
                        const float x = z * inverse_cap, t = exp2_approx(x * (2.0f * kScoredLog2e));
                        const float curve = fmaf(-2.0f * p.cap, rcp_approx(t + 1.0f), p.cap);
                        z = WIDE && fabsf(x) <= 0.6f ? z * sd_tanh_ratio(x * x) : curve;
                    }
                    if (biased) {
                        const int distance = position[e >> 1] - (token0 + 64 * (n >> 1) + 8 * (n & 1) + 2 * (int)c + (e & 1));
                        z = fmaf(-slope[e >> 1], fabsf((float)distance), z);
                    }
                    sc[n][e] = z * kScoredLog2e;
                }
        } else {
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] *= mul[e >> 1] * kScoredLog2e * (CODE ? scales[n >> 1].x : 1.0f);
        }
        // ---- visibility: tokens that no row of the CTA sees may hold anything in V ----------------
        uint32_t keep_lo[kPair], keep_hi[kPair];
#pragma unroll
        for (int u = 0; u < kPair; ++u) keep_lo[u] = keep_hi[u] = 0xffffffffu;
        const bool cut = token0 < inner_first || token0 + 64 * (kPair - 1) + 16 > inner_end || !there[kPair - 1];
        if (cut) {
            uint32_t seen = 0u;
#pragma unroll
            for (int n = 0; n < kCols; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int token = token0 + 64 * (n >> 1) + 8 * (n & 1) + 2 * (int)c + (e & 1);
                    const bool visible = there[n >> 1] && token >= first[e >> 1] && token < end[e >> 1];
                    if (!visible) sc[n][e] = -INFINITY;
                    seen |= (visible ? 1u : 0u) << (2 * n + (e & 1));
                }
#pragma unroll
            for (int offset = 4; offset < 32; offset <<= 1) seen |= __shfl_xor_sync(0xffffffffu, seen, offset);
#pragma unroll
            for (int u = 0; u < kPair; ++u) {
                const uint32_t bits = seen >> (4 * u);
                keep_lo[u] = (bits & 1u ? 0x0000ffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
                keep_hi[u] = (bits & 4u ? 0x0000ffffu : 0u) | (bits & 8u ? 0xffff0000u : 0u);
            }
            if (CODE) {
                // 16 tokens that no row sees may lie in a page that was never written: its scales count as zero
                const uint32_t some = __reduce_or_sync(0xffffffffu, seen);
#pragma unroll
                for (int u = 0; u < kPair; ++u)
                    if (!(some >> (4 * u) & 15u)) scales[u] = make_float2(0.0f, 0.0f);
            }
        }
        // ---- online softmax with a lazy maximum ----------------------------------------------------
        float top[2], of[kPair][2], v_log[kPair];   // the largest score, of each tile; log2 of the tile's V scale
        bool grow = false;
#pragma unroll
        for (int u = 0; u < kPair; ++u) v_log[u] = CODE ? log2_approx(fabsf(scales[u].y)) : 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            top[h] = -INFINITY;
#pragma unroll
            for (int u = 0; u < kPair; ++u) {
                of[u][h] = max3(fmaxf(sc[2 * u][2 * h], sc[2 * u][2 * h + 1]), sc[2 * u + 1][2 * h], sc[2 * u + 1][2 * h + 1]);
                top[h] = u ? fmaxf(top[h], of[u][h]) : of[u][h];
                if (CODE) grow = grow || of[u][h] > v_ref[h] + kSlack - v_log[u];
            }
            grow = grow || top[h] > m[h] + kSlack;   // m is -inf while the row has seen nothing
        }
        if (__any_sync(0xffffffffu, grow)) {
            float keep[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
                const float fresh = fmaxf(m[h], top[h]);
                keep[h] = fresh == -INFINITY ? 1.0f : exp2_approx(m[h] - fresh);
                m[h] = fresh;
                l[h] *= keep[h];
                if (CODE) {
                    float heavy = -INFINITY;
#pragma unroll
                    for (int u = 0; u < kPair; ++u) heavy = fmaxf(heavy, of[u][h] + v_log[u]);
                    heavy = fmaxf(heavy, __shfl_xor_sync(0xffffffffu, heavy, 1));
                    heavy = fmaxf(heavy, __shfl_xor_sync(0xffffffffu, heavy, 2));
                    const float next = fmaxf(v_ref[h], heavy);
                    keep[h] = next == -INFINITY ? 1.0f : exp2_approx(v_ref[h] - next);
                    v_ref[h] = next;
                    // (a page of scale 0 may hold the largest score)
                    v_unit[h] = next == -INFINITY ? 0.0f : exp2_approx(fminf(m[h] - next, 126.0f));
                }
            }
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                o[n][0] *= keep[0];
                o[n][1] *= keep[0];
                o[n][2] *= keep[1];
                o[n][3] *= keep[1];
            }
        }
        float offset[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) offset[h] = m[h] == -INFINITY ? 0.0f : kLift - m[h];
        uint32_t p_head[kPair][4], p_tail[kPair][4];
#pragma unroll
        for (int n = 0; n < kCols; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float p0 = exp2_approx(sc[n][2 * h] + offset[h]), p1 = exp2_approx(sc[n][2 * h + 1] + offset[h]);
                l[h] += p0 + p1;
                if (CODE) {
                    const float times = min_nan(scales[n >> 1].y * v_unit[h], 1e36f);   // weights of 0 stay 0
                    p_head[n >> 1][2 * (n & 1) + h] = pack_f16(p0 * times, p1 * times);
                } else {
                    const uint32_t head = pack_bf16(p0, p1);
                    p_head[n >> 1][2 * (n & 1) + h] = head;
                    p_tail[n >> 1][2 * (n & 1) + h] = pack_bf16(p0 - __uint_as_float(head << 16), p1 - __uint_as_float(head & 0xffff0000u));
                }
            }
        // ---- O += P V -------------------------------------------------------------------------------
        const unsigned int j = lane >> 3, r = lane & 7u;
        const unsigned int token = 16u * warp + 8u * (j & 1u) + r;
#pragma unroll
        for (int u = 0; u < kPair; ++u) {
            if (!there[u]) continue;
            const uint32_t v_base = smem_u32(ring + stage[u] * 2 * kOperand + kOperand);
            if (CODE) {
                // A transposed 8x8 block of 16-bit pairs gives a thread two tokens of two adjacent dims; columns
                // of the accumulator tile 2 ch + parity are the dims 16 ch + 2 g + parity.
#pragma unroll
                for (int np = 0; np < 4; ++np) {
                    uint32_t raw[4];
                    ldmatrix_x4_trans(raw, v_base + token * 128u + (((2u * np + (j >> 1)) ^ (token & 7u)) << 4));
                    if (cut) {   // both dims' codes of a token are 16 bits of the register
#pragma unroll
                        for (int ch = 0; ch < 2; ++ch) raw[2 * ch] &= keep_lo[u], raw[2 * ch + 1] &= keep_hi[u];
                    }
#pragma unroll
                    for (int ch = 0; ch < 2; ++ch) {
                        uint32_t lo, hi, lo_even, lo_odd, hi_even, hi_odd;
                        asm("prmt.b32 %0, %1, 0, 0x3120;" : "=r"(lo) : "r"(raw[2 * ch]));
                        asm("prmt.b32 %0, %1, 0, 0x3120;" : "=r"(hi) : "r"(raw[2 * ch + 1]));
                        sd_codes<CODE>(lo, lo_even, lo_odd);
                        sd_codes<CODE>(hi, hi_even, hi_odd);
                        mma_f16(o[4 * np + 2 * ch], p_head[u], lo_even, hi_even);
                        mma_f16(o[4 * np + 2 * ch + 1], p_head[u], lo_odd, hi_odd);
                    }
                }
            } else {
#pragma unroll
                for (int np = 0; np < 8; ++np) {
                    const unsigned int chunk = 2u * (np & 3) + (j >> 1);
                    uint32_t vb[4];
                    ldmatrix_x4_trans(vb, v_base + (np >> 2) * (kOperand / 2) + token * 128u + ((chunk ^ (token & 7u)) << 4));
                    if (cut) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) vb[i] &= i & 1 ? keep_hi[u] : keep_lo[u];
                    }
                    mma_bf16(o[2 * np], p_head[u], vb[0], vb[1]);
                    mma_bf16(o[2 * np + 1], p_head[u], vb[2], vb[3]);
                    mma_bf16(o[2 * np], p_tail[u], vb[0], vb[1]);
                    mma_bf16(o[2 * np + 1], p_tail[u], vb[2], vb[3]);
                }
            }
        }
        __syncwarp();
#pragma unroll
        for (int u = 0; u < kPair; ++u)
            if (lane == 0 && there[u]) mbar_arrive(&empty[stage[u]]);
    }

    // ---- merge the four warps and publish ------------------------------------------------------------
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
    pdl_launch_dependents();
    named_barrier(1, kSdWarps * 32);   // every warp is done reading the ring
    float *merge_o = reinterpret_cast<float *>(ring);                      // [4][16][132]
    float *merge_m = merge_o + kSdWarps * 16 * kSdMergeFloats;             // [4][16]
    float *merge_l = merge_m + kSdWarps * 16;                              // [4][16]
    float *merge_r = CODE ? merge_l + kSdWarps * 16 : merge_m;             // [4][16]: what o counts in
#pragma unroll
    for (int n = 0; n < 16; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float *row = merge_o + (warp * 16u + g + 8u * h) * kSdMergeFloats;
            if (CODE) {
                row[16 * (n >> 1) + 4 * c + (n & 1)] = o[n][2 * h];
                row[16 * (n >> 1) + 4 * c + 2 + (n & 1)] = o[n][2 * h + 1];
            } else {
                *reinterpret_cast<float2 *>(row + 8 * n + 2 * c) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
            }
        }
    if (c == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            merge_m[warp * 16u + g + 8u * h] = m[h] - kLift;
            merge_l[warp * 16u + g + 8u * h] = l[h];
            if (CODE) merge_r[warp * 16u + g + 8u * h] = v_ref[h] - kLift;
        }
    }
    named_barrier(1, kSdWarps * 32);
    const unsigned int d = threadIdx.x;  // one head dimension per consumer thread
    for (unsigned int row = 0; row < live; ++row) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kSdWarps; ++w) top = fmaxf(top, merge_m[w * 16 + row]);
        float sum = 0.0f, acc = 0.0f;
#pragma unroll
        for (int w = 0; w < kSdWarps; ++w) {
            const float mw = merge_m[w * 16 + row];
            const float weight = mw == -INFINITY ? 0.0f : exp2_approx(mw - top);
            sum += merge_l[w * 16 + row] * weight;
            const float rw = CODE ? merge_r[w * 16 + row] : mw, of_o = !CODE ? weight : rw == -INFINITY ? 0.0f : exp2_approx(rw - top);
            acc += merge_o[(w * 16 + row) * kSdMergeFloats + d] * of_o;
        }
        const unsigned long long item = item_of(row);
        if (p.max_splits > 1u) {
            float *part = scored_partial(p, item, split);
            part[d] = acc;
            if (d == 0) {
                part[kSdDim] = top;
                part[kSdDim + 1] = sum;
            }
        } else {
            const float value = sum == 0.0f ? 0.0f : acc / sum;
            if (!isfinite(value)) atomicCAS(p.status, 0, YVX_STATUS_NONFINITE);
            store_output(p.output, p.output_dtype, item * kSdDim + d, value);
        }
    }
}

// ---- host side ------------------------------------------------------------------------------------------

typedef CUresult (*ScoredEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static ScoredEncodeFn scored_encode_entry()
{
    static ScoredEncodeFn entry = [] {
        void *symbol = nullptr;
        cudaDriverEntryPointQueryResult query;
        const bool found = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &symbol, cudaEnableDefault, &query) == cudaSuccess &&
                           query == cudaDriverEntryPointSuccess;
        return found ? reinterpret_cast<ScoredEncodeFn>(symbol) : nullptr;
    }();
    return entry;
}

// {128 lanes, two middle dimensions by ascending stride, outer}; the box is 128 bytes of `box_tokens` rows.
// Returns false when tiled copies cannot describe the layout.
bool scored_encode_rows(CUtensorMap *map, const void *base, int element_bytes, unsigned long long token_stride,
                        unsigned long long head_stride, unsigned long long outer_stride, unsigned long long tokens,
                        unsigned long long heads, unsigned long long outer, bool head_inner, unsigned int box_tokens,
                        unsigned int box_heads)
{
    ScoredEncodeFn encode = scored_encode_entry();
    const unsigned long long tb = token_stride * element_bytes, hb = head_stride * element_bytes;
    unsigned long long ob = outer_stride * element_bytes;
    if (outer == 1ull) ob = ((head_inner ? tb * tokens : hb * heads) + 15ull) & ~15ull;
    if (!encode || (reinterpret_cast<uintptr_t>(base) & 15u) || (tb & 15ull) || (hb & 15ull) || (ob & 15ull) || !tb || !hb ||
        !ob || tb >= (1ull << 40) || hb >= (1ull << 40) || ob >= (1ull << 40))
        return false;
    const cuuint64_t dims[4] = {kSdDim, head_inner ? heads : tokens, head_inner ? tokens : heads, outer};
    const cuuint64_t strides[3] = {head_inner ? hb : tb, head_inner ? tb : hb, ob};
    const cuuint32_t box[4] = {128u / (unsigned int)element_bytes, head_inner ? box_heads : box_tokens,
                               head_inner ? box_tokens : box_heads, 1u};
    const cuuint32_t steps[4] = {1, 1, 1, 1};
    return encode(map, element_bytes == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                  const_cast<void *>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 1: launched, 0: not this kernel's shape, negative: an error.
int scored_decode_launch(const yvx_scored_problem &p, cudaStream_t stream)
{
    const int element_bytes = p.kv_code == YVX_KV_PLAIN ? 2 : 1;
    const unsigned long long vectors = (unsigned long long)p.query_rows * (p.query_heads / p.kv_heads);
    const unsigned long long head_stride = p.query_head_stride ? p.query_head_stride : kSdDim;
    if (p.head_dim != (unsigned)kSdDim || p.query_dtype != YVEX_DTYPE_BF16 ||
        (p.kv_code == YVX_KV_PLAIN && p.kv_dtype != YVEX_DTYPE_BF16) || (reinterpret_cast<uintptr_t>(p.query) & 7u) ||
        (p.query_row_stride & 3ull) || (p.query_session_stride & 3ull) || (head_stride & 3ull) ||
        (vectors + 15ull) / 16ull * p.kv_heads > 65535ull)
        return 0;
    unsigned int unit = kSdTokens;
    if (p.block_table && p.block_tokens % kSdTokens) {
        if (p.block_tokens != 16u && p.block_tokens != 32u) return 0;
        unit = p.block_tokens;
    }
    const bool head_inner = p.key_head_stride < p.key_token_stride;
    if ((p.value_head_stride < p.value_token_stride) != head_inner) return 0;
    const unsigned long long tokens = p.block_table ? p.block_tokens : p.kv_tokens_max;
    const unsigned long long outer = p.block_table ? p.pool_blocks : p.sessions;
    SdMaps maps;
    if (!scored_encode_rows(&maps.key, p.key, element_bytes, p.key_token_stride, p.key_head_stride, p.key_outer_stride, tokens,
                            p.kv_heads, outer, head_inner, unit, 1u) ||
        !scored_encode_rows(&maps.value, p.value, element_bytes, p.value_token_stride, p.value_head_stride,
                            p.value_outer_stride, tokens, p.kv_heads, outer, head_inner, unit, 1u))
        return 0;
    // (in one kernel for both, the choice costs 4 rows over 131072 tokens of codes under a cap 78 -> 82 us)
    void (*const kernels[6])(const yvx_scored_problem, const SdMaps, const int, const int) = {
        scored_decode_kernel<YVX_KV_PLAIN, false>, scored_decode_kernel<YVX_KV_E4M3, false>, scored_decode_kernel<YVX_KV_I8, false>,
        scored_decode_kernel<YVX_KV_PLAIN, true>,  scored_decode_kernel<YVX_KV_E4M3, true>,  scored_decode_kernel<YVX_KV_I8, true>};
    const auto kernel = kernels[p.kv_code + (p.cap > kSdWideCap ? 3 : 0)];
    YVX_CUDA_TRY(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSdSmemBytes));
    const dim3 grid(p.max_splits, p.kv_heads * (unsigned int)((vectors + 15ull) / 16ull), p.sessions);
    kernel<<<grid, kSdThreads, kSdSmemBytes, stream>>>(p, maps, (int)unit, head_inner ? 1 : 0);
    const int rc = yvx_cuda_check(cudaGetLastError(), "scored_decode_kernel");
    return rc != 0 ? rc : 1;
}

}  // namespace yvx
