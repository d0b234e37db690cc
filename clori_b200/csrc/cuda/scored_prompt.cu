// Scored attention for prompt-sized calls on the 5th-generation tensor cores: bf16 Q / K / V,
// head_dim 128, contiguous rows or pages of 64 n tokens, any rule and any visible runs.
//
// A CTA owns two tiles (A, B) of 128 rows, a row being a (query row, head of the KV head's group) pair: a tile of
// a group of 4 is 32 query rows, which see fewer tokens in vain than 128 do, and few rows fill it (17 rows of 32
// heads over 131072 tokens: 306 us with a head for each tile, 102 so). While one tile is in its softmax the other is
// in its matrix products. Warp 8 brings K and V in tiles of 128 tokens (tiled copies, 128-byte swizzle, two stages
// each), warp 9 issues S = Q K^T (both operands in shared memory) into one score buffer that is free again as soon
// as it is read, warp 10 O += P V (P in tensor memory), warps 0-3 and 4-7 run the softmax of A and B, a thread per
// row, and warp 11 fetches the CTA's next piece of work: the grid has a block for every piece, and a block that
// is done takes the work of one that has not started (cluster launch control), so loads and first products of a
// piece run beside the last tiles of the one before (4 x 1531 rows with a prefix: 260 us -> 242). Registers: 224 a
// thread for the softmax and 56 for the others, of the 168 at launch. A tile walks only the token tiles that some
// row of it sees, the last one first: with a bias against distance, and often without, the largest weights come
// early. With few pieces of work the KV sequence is split and folded.
//
// A thread takes its row's 128 products into registers, and P V of the first 64 starts while the others are
// exponentiated. The score rule runs two lanes at a time (f32x2 instructions):
//   cap    tanh(x) = x p(x^2) with p of degree 3 while every |x| of the warp's tile is at most 5/8, of degree 6 up to
//          11/8, beyond 1 - 2 / (e^2x + 1) from the exponential unit, which is as loaded as the tensor cores. What
//          decides on the form bounds the logits as well: while the bound is at most 2^32 above the row's reference, no
//          maximum is looked for.
//   bias   slope * (s - position) is linear in the token inside a tile: one multiply-add per score and one
//          constant per row and tile; tokens behind the row's position (prefixes) take |.| in full.
// Weights are rounded to bf16 (the tensor cores' operand; at most 2^-8 of each), sums and the accumulator are F32.
//
// Measured, calls between events with the L2 flushed before: 37 heads x 1024 rows x 4096 tokens, nothing masked, 82 us
// (75 in a loop: 1.06 PFLOP/s), with a cap of 50 92, with a bias 100; two prompts of 8192 capped rows 1.56 ms, 1531-row prompts with a prefix and a cap 190 us
// (4 of 40 heads), 16384 rows of packed documents with a bias 485 us (32 heads). A pair of tiles takes about 3300 cycles without a cap;
// the products need 2048, the exponential unit 2048. With the softmax's arithmetic taken out the same loop still takes
// 2800: the one score buffer goes back and forth (products, read, free, products), and tensor memory has no room
// for a second beside O and P. A piece of work costs about 10000 cycles besides its tiles: its first and last tile
// have no partner and run masks, rows leave, all of it code that the instruction cache has lost since the last piece.
#include "scored.cuh"
#include "tcgen05.cuh"

namespace yvx {

constexpr int kSpM = 128, kSpN = 128, kSpD = 128, kSpStages = 2, kSpThreads = 384;
constexpr int kSpHalfBytes = kSpM * 64 * 2;        // [128][64] bf16, swizzled
constexpr int kSpTileBytes = 2 * kSpHalfBytes;     // 32 KB
constexpr int kSpOutBytes = 32 * 64;               // a warp's rows on their way out, 64 bytes of each at a time
constexpr int kSpSharedBytes = 8 * 1024;
constexpr int kSpSmemBytes = (2 + 2 * kSpStages) * kSpTileBytes + 8 * kSpOutBytes + 1024 + kSpSharedBytes;
constexpr float kSpWideCap = 2048.0f;              // the exponential unit's tanh is off by some 2^-22 of the cap: 5e-4 here
constexpr float kSpRescale = 8.0f;                 // log2 units the maximum may lag behind
// The same where a bound of the tile's logits stands for the maximum: values up to 1e23 stay in F32's range over 131072
// tokens. Two prompts of 8192 rows under a cap of 50: 1800 us with 16, 1587 with 24, 1557 with 32, 1556 with 48.
constexpr float kSpNear = 32.0f;
constexpr uint32_t kSpTmemColumns = 512;           // S 128 | P_A 64 | P_B 64 | O_A 128 | O_B 128
constexpr int kSpReaders = 11;                     // warps that read a piece of work
constexpr uint32_t kSpPColumn = 128, kSpOColumn = 256;

struct SpMaps {
    CUtensorMap query, key, value;
};

// One piece of work: two row tiles and what they see. Warp 11 fills it.
struct SpWork {
    int first[2 * kSpM], end[2 * kSpM];   // visible run of each query row; rows that do not exist see nothing
    int position[2 * kSpM];               // where its bias counts from
    int hull_first, hull_end;             // of all of them
    int staged_first;                     // the token that staged rows begin with
    int solid_end;                        // every token of [hull_first, solid_end) is seen by some row
    int from[2], until[2];                // token tiles [from[x], until[x]) of the two row tiles
    unsigned int q0, head, b, split;      // first query row, first query head
    int valid;                            // 0: nothing is left
};

struct SpShared {
    uint4 next_block;                     // the answer to a request for another block's work
    uint64_t next_full, work_full[2], work_empty[2], ask;
    uint64_t q_full, q_empty;
    uint64_t k_full[kSpStages], k_empty[kSpStages], v_full[kSpStages], v_empty[kSpStages];
    uint64_t s_full[2], s_free, p_half[2][2], pv_done[2];
    uint32_t tmem_base;
    unsigned int where[kSpM];             // a tile's row: its query row | its head << 16, or ~0 when it is not used
    SpWork work[2];
};
static_assert(sizeof(SpShared) <= kSpSharedBytes, "the barrier block outgrew its slot");

// Asks the hardware for a block of the grid that has not started: its index, or "none is left", arrives in *slot.
__device__ __forceinline__ void sp_ask_block(uint4 *slot, uint64_t *bar)
{
    mbar_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
                 :: "r"(smem_u32(slot)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool sp_block_given(const uint4 *slot, unsigned int &block)
{
    uint32_t given;
    asm volatile(
        "{\n\t.reg .b128 r;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
        "ld.shared.b128 r, [%2];\n\t"
        "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "mov.u32 %1, 0;\n\t"
        "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, r;\n\t}"
        : "=r"(given), "=r"(block) : "r"(smem_u32(slot)) : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the slot may be written again
    return given != 0u;
}

// ---- two floats at a time -----------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long f2_pack(float lo, float hi)
{
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void f2_unpack(unsigned long long v, float &lo, float &hi)
{
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long f2_fma(unsigned long long a, unsigned long long b, unsigned long long c)
{
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long f2_mul(unsigned long long a, unsigned long long b)
{
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ unsigned long long f2_add(unsigned long long a, unsigned long long b)
{
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ unsigned long long f2_load(const uint32_t (&s)[32], int c)
{
    return f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1]));
}
__device__ __forceinline__ void f2_store(unsigned long long v, uint32_t (&s)[32], int c)
{
    float lo, hi;
    f2_unpack(v, lo, hi);
    s[c] = __float_as_uint(lo);
    s[c + 1] = __float_as_uint(hi);
}

// tanh(x) = x (a0 + a1 x^2 + ..) for |x| <= 5/8 and |x| <= 11/8, fitted for this kernel: the largest absolute errors
// are 8.3e-7 and 8.2e-7.
__device__ constexpr float kSpTanhTiny[4] = {0.999987904734053f, -0.33290581616016607f, 0.1292045463446343f, -0.03864439123986797f};
__device__ constexpr float kSpTanhSmall[7] = {0.9999906071821962f,  -0.3331309371709024f,   0.13205654305843492f, -0.050316830005499996f,
                                              0.016203115118873665f, -0.0035891439879808845f, 0.00038086217121292696f};

// grid: one dimension, the split of the KV sequence slowest. (session, head) lanes in groups whose K and V fit the L2 together; inside a group the
// pair of row tiles varies slowest, last rows first, and the lane fastest.
// WIDE: a cap above kSpWideCap, under which a logit that is small beside the cap keeps its accuracy whatever its tile holds.
template <bool CAP, bool BIAS, bool SPLIT, bool WIDE>
__global__ void __launch_bounds__(kSpThreads, 1)
scored_prompt_kernel(const yvx_scored_problem p, const __grid_constant__ SpMaps maps, const int head_inner,
                     const unsigned int lane_group, const int staged)
{
    extern __shared__ unsigned char sp_raw[];
    unsigned char *smem = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(sp_raw) + 1023u) & ~uintptr_t(1023));
    unsigned char *q_smem = smem;                                  // tile A, then tile B
    unsigned char *k_smem = smem + 2 * kSpTileBytes;
    unsigned char *v_smem = k_smem + kSpStages * kSpTileBytes;
    unsigned char *out_smem = v_smem + kSpStages * kSpTileBytes;
    SpShared *sh = reinterpret_cast<SpShared *>(out_smem + 8 * kSpOutBytes);

    const unsigned int warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    // A tile holds `pack` query heads of `tile_rows` query rows each, the heads of a row side by side.
    const unsigned int pack = scored_packed_heads(p), tile_rows = kSpM / pack, used = tile_rows * pack;
    if (threadIdx.x < (unsigned int)kSpM)
        sh->where[threadIdx.x] = threadIdx.x < used ? threadIdx.x / pack | (threadIdx.x % pack) << 16 : ~0u;
    // rows of Q behind the used ones stay zero
    for (unsigned int i = threadIdx.x; i < 2u * 2u * (kSpM - used) * 8u; i += kSpThreads)
        *reinterpret_cast<uint4 *>(q_smem + i / ((kSpM - used) * 8u) * kSpHalfBytes + used * 128u + i % ((kSpM - used) * 8u) * 16u) =
            make_uint4(0u, 0u, 0u, 0u);
    fence_proxy_async();
    if (threadIdx.x == 0) {
        mbar_init(&sh->next_full, 1);
        mbar_init(&sh->ask, 1);
        mbar_init(&sh->q_full, 1);
        mbar_init(&sh->q_empty, 1);
        mbar_init(&sh->s_free, kSpM);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->work_full[i], 1);
            mbar_init(&sh->work_empty[i], kSpReaders);
        }
        for (int i = 0; i < kSpStages; ++i) {
            mbar_init(&sh->k_full[i], 1);
            mbar_init(&sh->k_empty[i], 1);
            mbar_init(&sh->v_full[i], 1);
            mbar_init(&sh->v_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh->s_full[i], 1);
            mbar_init(&sh->p_half[i][0], kSpM);
            mbar_init(&sh->p_half[i][1], kSpM);
            mbar_init(&sh->pv_done[i], 1);
        }
        fence_barrier_init();
    }
    if (warp == 9) {
        tmem_alloc(&sh->tmem_base, kSpTmemColumns);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sh->tmem_base;
    auto fail = [&]() { atomicCAS(p.status, 0, YVX_STATUS_TIMEOUT); };
    auto waited = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity)) != 0; };
    // The turn-th piece of work, or null when none is left (or a wait gave up).
    auto take = [&](unsigned int turn) -> const SpWork * {
        const SpWork *w = &sh->work[turn & 1u];
        if (!waited(&sh->work_full[turn & 1u], (turn >> 1) & 1u)) {
            if (lane == 0) fail();
            return nullptr;
        }
        return w->valid ? w : nullptr;
    };
    auto give_back = [&](unsigned int turn) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->work_empty[turn & 1u]);
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            // ------------------------------ tiled copies ----------------------------------------------
            unsigned int tiles = 0u, pieces = 0u;   // so far: token tiles, pieces of work with any
            bool ok = true;
            for (unsigned int turn = 0; ok; ++turn) {
                const SpWork *const w = take(turn);
                if (w == nullptr) break;
                const int hull_first = w->hull_first, hull_end = w->hull_end, start = hull_first / kSpN, staged_first = w->staged_first;
                const int stop = (hull_end + kSpN - 1) / kSpN;
                const unsigned int b = w->b, kv_head = w->head / (p.query_heads / p.kv_heads);
                if (lane == 0) {
                    if (stop > start) {
                        if (pieces) ok = mbar_wait(&sh->q_empty, (pieces - 1u) & 1u);
                        if (ok) {
                            mbar_expect_tx(&sh->q_full, 2u * 2u * used * 128u);
                            for (int x = 0; x < 2; ++x)
                                for (int h = 0; h < 2; ++h)
                                    tma_load_4d(q_smem + x * kSpTileBytes + h * kSpHalfBytes, &maps.query, &sh->q_full, 64 * h,
                                                (int)w->head, (int)(w->q0 + x * tile_rows), (int)b);
                        }
                    }
                    for (int j = stop - 1; ok && j >= start; --j) {
                        const unsigned int n = tiles + (unsigned int)(stop - 1 - j), stage = n % kSpStages;
                        const uint32_t parity = ((n / kSpStages) - 1u) & 1u;
                        // two runs of 64 tokens (a page may end between them); one behind the hull is not loaded
                        int outer[2], inner[2], runs = 0;
                        for (int r = 0; r < 2; ++r) {
                            const int token = j * kSpN + 64 * r;
                            if (token >= hull_end) break;
                            outer[r] = (int)b, inner[r] = token - staged_first;
                            if (p.block_table) {
                                const int page = token + 64 > hull_first ? scored_page(p, b, (unsigned int)token / p.block_tokens) : 0;
                                outer[r] = page < 0 ? 0 : page;
                                inner[r] = (int)((unsigned int)token % p.block_tokens);
                            }
                            ++runs;
                        }
                        for (int operand = 0; ok && operand < 2; ++operand) {
                            uint64_t *full = operand ? &sh->v_full[stage] : &sh->k_full[stage];
                            uint64_t *empty = operand ? &sh->v_empty[stage] : &sh->k_empty[stage];
                            unsigned char *dst = (operand ? v_smem : k_smem) + stage * kSpTileBytes;
                            const CUtensorMap *map = operand ? &maps.value : &maps.key;
                            if (n >= (unsigned int)kSpStages) ok = mbar_wait(empty, parity);
                            if (!ok) break;
                            mbar_expect_tx(full, (uint32_t)runs * (kSpTileBytes / 2));
                            for (int r = 0; r < runs; ++r) {
                                const int c1 = head_inner ? (int)kv_head : inner[r], c2 = head_inner ? inner[r] : (int)kv_head;
                                tma_load_4d(dst + r * 64 * 128, map, full, 0, c1, c2, outer[r]);
                                tma_load_4d(dst + kSpHalfBytes + r * 64 * 128, map, full, 64, c1, c2, outer[r]);
                            }
                        }
                    }
                    if (!ok) fail();
                    mbar_arrive(&sh->ask);   // all loads are under way: time to look for the next piece
                }
                ok = __all_sync(0xffffffffu, ok);
                tiles += (unsigned int)(stop - start);
                pieces += stop > start ? 1u : 0u;
                give_back(turn);
            }
        } else if (warp == 9) {
            // ------------------------------ S = Q K^T, A and B in turn ------------------------------
            // all 32 lanes run converged, one elected lane issues
            constexpr uint32_t idesc = idesc_bf16_f32(kSpM, kSpN, false);
            const uint32_t q_addr = smem_u32(q_smem), k_addr = smem_u32(k_smem);
            unsigned int issued = 0u, tiles = 0u, pieces = 0u;
            bool ok = true;
            for (unsigned int turn = 0; ok; ++turn) {
                const SpWork *const w = take(turn);
                if (w == nullptr) break;
                const int start = w->hull_first / kSpN, stop = (w->hull_end + kSpN - 1) / kSpN;
                const int from[2] = {w->from[0], w->from[1]}, until[2] = {w->until[0], w->until[1]};
                give_back(turn);
                if (stop <= start) continue;
                ok = waited(&sh->q_full, pieces & 1u);
                for (int j = stop - 1; ok && j >= start; --j) {
                    const unsigned int n = tiles + (unsigned int)(stop - 1 - j), stage = n % kSpStages;
                    ok = waited(&sh->k_full[stage], (n / kSpStages) & 1u);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (!ok || j < from[x] || j >= until[x]) continue;
                        if (issued) ok = waited(&sh->s_free, (issued - 1u) & 1u);   // the previous products have been read
                        if (!ok) break;
                        tc_fence_after_sync();
                        ++issued;
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks) {
                            const uint32_t off = (ks >> 2) * kSpHalfBytes + (ks & 3) * 32;
                            tc_mma_ss_elect(tmem, smem_desc_sw128(q_addr + x * kSpTileBytes + off, 16, 1024),
                                            smem_desc_sw128(k_addr + stage * kSpTileBytes + off, 16, 1024), idesc, ks ? 1u : 0u);
                        }
                        tc_commit_elect(&sh->s_full[x]);
                    }
                    if (ok) tc_commit_elect(&sh->k_empty[stage]);
                }
                if (ok) tc_commit_elect(&sh->q_empty);
                if (!ok && lane == 0) fail();
                tiles += (unsigned int)(stop - start);
                ++pieces;
            }
        } else if (warp == 10) {
            // ------------------------------ O += P V ------------------------------------------------
            constexpr uint32_t idesc = idesc_bf16_f32(kSpM, kSpD, true);
            const uint32_t v_addr = smem_u32(v_smem);
            unsigned int tiles = 0u, counts[2] = {0u, 0u};
            bool ok = true;
            for (unsigned int turn = 0; ok; ++turn) {
                const SpWork *const w = take(turn);
                if (w == nullptr) break;
                const int start = w->hull_first / kSpN, stop = (w->hull_end + kSpN - 1) / kSpN;
                const int from[2] = {w->from[0], w->from[1]}, until[2] = {w->until[0], w->until[1]};
                give_back(turn);
                for (int j = stop - 1; ok && j >= start; --j) {
                    const unsigned int n = tiles + (unsigned int)(stop - 1 - j), stage = n % kSpStages;
                    ok = waited(&sh->v_full[stage], (n / kSpStages) & 1u);
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        if (!ok || j < from[x] || j >= until[x]) continue;
                        const uint32_t later = j < until[x] - 1 ? 1u : 0u;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            ok = ok && waited(&sh->p_half[x][h], counts[x] & 1u);
                            if (!ok) break;
                            tc_fence_after_sync();
#pragma unroll
                            for (int kk = 4 * h; kk < 4 * h + 4; ++kk)
                                tc_mma_ts_elect(tmem + kSpOColumn + x * kSpD, tmem + kSpPColumn + x * 64 + kk * 8,
                                                smem_desc_sw128(v_addr + stage * kSpTileBytes + kk * 2048, kSpHalfBytes, 1024), idesc,
                                                kk ? 1u : later);
                        }
                        if (ok) tc_commit_elect(&sh->pv_done[x]);
                        ++counts[x];
                    }
                    if (ok) tc_commit_elect(&sh->v_empty[stage]);
                }
                if (!ok && lane == 0) fail();
                tiles += (unsigned int)(stop - start);
            }
        } else {
            // ------------------------------ pieces of work ------------------------------------------
            // The block's own first, then those of blocks that have not started, as long as there are any.
            const unsigned int pairs = (p.query_rows + 2u * tile_rows - 1u) / (2u * tile_rows), lanes = p.query_heads / pack * p.sessions;
            const unsigned int per_group = pairs * lane_group;   // the grid holds it: below 2^31
            const unsigned int per_split = (lanes + lane_group - 1u) / lane_group * per_group;
            unsigned int block = blockIdx.x, asked = 0u;
            bool ok = true, more = true;
            for (unsigned int turn = 0; ok && more; ++turn) {
                SpWork *const w = &sh->work[turn & 1u];
                if (turn >= 2u) ok = waited(&sh->work_empty[turn & 1u], ((turn >> 1) - 1u) & 1u);
                unsigned int work_lane = 0u, within = 0u, split = 0u;
                auto given = [&]() {
                    split = SPLIT ? block / per_split : 0u;
                    const unsigned int rest = SPLIT ? block % per_split : block;
                    within = rest % per_group;
                    work_lane = rest / per_group * lane_group + within % lane_group;
                    return work_lane < lanes;   // the last group may be short
                };
                bool look = turn > 0u || !given();
                while (ok && look) {
                    if (lane == 0) sp_ask_block(&sh->next_block, &sh->next_full);
                    ok = waited(&sh->next_full, asked & 1u);
                    ++asked;
                    more = ok && sp_block_given(&sh->next_block, block);
                    __syncwarp();
                    look = more && !given();
                }
                if (!ok) {
                    if (lane == 0) fail();
                    break;   // who waits for the piece gives up as well
                }
                int tiles = 0;
                if (more) {
                    const unsigned int q0 = (pairs - 1u - within / lane_group) * 2u * tile_rows;
                    const unsigned int head = work_lane % (p.query_heads / pack) * pack, b = work_lane / (p.query_heads / pack);
                    const unsigned int kv_tokens = admitted_kv_tokens(p.kv_tokens, b, p.kv_tokens_uniform, p.kv_tokens_max, p.status);
                    const long long query_start = scored_query_start(p, b, kv_tokens);
                    int hull_first, hull_end;
                    auto look_at_rows = [&](int t0, int t1) {   // as far as they see tokens [t0, t1)
                        hull_first = 0x7fffffff, hull_end = 0;
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            int lo = 0x7fffffff, hi = 0;
                            for (unsigned int at = x * tile_rows + lane; at < (x + 1) * tile_rows; at += 32u) {
                                ScoredRange range = {0, 0, 0};
                                if (q0 + at < p.query_rows) range = scored_range(p, b, q0 + at, kv_tokens, query_start);
                                if (SPLIT) {
                                    range.first = max(range.first, t0), range.end = min(range.end, t1);
                                    if (range.first >= range.end) range.first = range.end = 0;
                                }
                                w->first[at] = range.first, w->end[at] = range.end;
                                if (BIAS) w->position[at] = range.position;
                                if (range.first < range.end) lo = min(lo, range.first), hi = max(hi, range.end);
                            }
                            lo = __reduce_min_sync(0xffffffffu, lo);
                            hi = __reduce_max_sync(0xffffffffu, hi);
                            if (lane == 0) w->from[x] = hi > 0 ? lo / kSpN : 0, w->until[x] = (hi + kSpN - 1) / kSpN;
                            hull_first = min(hull_first, lo);
                            hull_end = max(hull_end, hi);
                        }
                    };
                    look_at_rows(0, 0x7fffffff);
                    if (SPLIT && hull_end > 0) {
                        // a split takes its part of the pair's own hull, from the hull's first boundary of 128 tokens; the
                        // last one takes what is left
                        const long long t0 = (hull_first & ~(kSpN - 1)) + (long long)split * p.chunk_tokens;
                        look_at_rows((int)min(t0, (long long)hull_end),
                                     split + 1u < p.max_splits ? (int)min(t0 + p.chunk_tokens, (long long)hull_end) : hull_end);
                    }
                    if (hull_end == 0) hull_first = 0;
                    // Runs of the rows may leave gaps. Every pass goes on to the last token that a run reaches from where
                    // the pass before ended; it ends at the first gap.
                    int solid_end = hull_end;
                    if (p.row_first || p.row_end) {
                        __syncwarp();
                        int reach = hull_first;
                        do {
                            solid_end = reach;
                            for (unsigned int at = lane; at < 2u * tile_rows; at += 32u)
                                if (w->first[at] <= solid_end) reach = max(reach, w->end[at]);
                            reach = __reduce_max_sync(0xffffffffu, reach);
                        } while (reach > solid_end);
                    }
                    if (lane == 0)
                        w->staged_first = staged ? scored_stage_first(p, kv_tokens, query_start) : 0, w->solid_end = solid_end, w->hull_first = hull_first, w->hull_end = hull_end, w->q0 = q0, w->head = head, w->b = b, w->split = split;
                    tiles = (hull_end + kSpN - 1) / kSpN - hull_first / kSpN;
                }
                if (lane == 0) w->valid = more;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->work_full[turn & 1u]);
                // the next one when this one's loads are all under way: a piece taken earlier might start later here
                // than elsewhere. A wait's limit is meant for one tile.
                ok = !more;
                for (int i = 0; !ok && i <= tiles; ++i) ok = waited(&sh->ask, turn & 1u);
                if (!ok && lane == 0) fail();
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ------------------------------ softmax ----------------------------------------------------
        const int x = (int)(warp >> 2);
        const uint32_t lane_base = tmem + (((warp & 3u) * 32u) << 16);
        const uint32_t p_col = lane_base + kSpPColumn + x * 64u, o_col = lane_base + kSpOColumn + x * kSpD;
        const unsigned int tile_row = threadIdx.x & 127u;
        // Raw products become exponents (log2 units): s * mul, or mul * tanh(s * to_unit) with
        // tanh(x) = x (a0 + a1 x^2 + ..).
        const float mul = (CAP ? p.cap : p.scale) * kScoredLog2e;
        const float to_unit = CAP ? p.scale / p.cap : 0.0f;
        const float inside_small = CAP ? 1.375f / to_unit : 0.0f, unit3 = to_unit * to_unit * to_unit;
        const float last = mul * to_unit * unit3 * unit3;   // what the short polynomial's last coefficient is folded with
        const float inside_tiny = CAP && last >= 1e-34f && last <= 1e30f ? 0.625f / to_unit : -1.0f;
        unsigned int tiles = 0u, count = 0u;   // so far: token tiles of the block, of this row tile
        bool ok = true;
        for (unsigned int turn = 0; ok; ++turn) {
        const SpWork *const w = take(turn);
        if (w == nullptr) break;
        ScoredRange range;
        bool exists;
        float slope2 = 0.0f;
        {
            const unsigned int place = sh->where[tile_row], at = place == ~0u ? 0u : place & 0xffffu;
            const unsigned int row = w->q0 + x * tile_rows + at;
            exists = place != ~0u && row < p.query_rows;
            range = {exists ? w->first[x * tile_rows + at] : 0, exists ? w->end[x * tile_rows + at] : 0,
                     BIAS ? w->position[x * tile_rows + at] : 0};
            if (BIAS) slope2 = p.slopes[w->head + (exists ? place >> 16 : 0u)] * kScoredLog2e;
        }
        const int hull_first = w->hull_first, solid_end = w->solid_end, my_from = w->from[x], my_until = w->until[x];
        const int stop = (w->hull_end + kSpN - 1) / kSpN, start = hull_first / kSpN;
        const float slope_held = BIAS ? (CAP ? slope2 : slope2 / mul) : 0.0f;
        float m = -INFINITY, l = 0.0f;
        for (int j = my_until - 1; ok && j >= my_from; --j) {   // (a wait that gave up is the last one)
            const uint32_t parity = count & 1u;
            ++count;
            const int k0 = j * kSpN;
            if (!waited(&sh->s_full[x], parity)) ok = false;
            tc_fence_after_sync();
            uint32_t s[4][32];
#pragma unroll
            for (int q = 0; q < 4; ++q) tmem_ld32(lane_base + 32 * q, s[q]);
            tmem_wait_ld();
            tc_fence_before_sync();
            mbar_arrive(&sh->s_free);   // the other tile's products may come
            if (k0 < hull_first || k0 + kSpN > solid_end) {
                // tokens that no row of the CTA sees: their rows of V may hold anything and become zero
                const unsigned int n = tiles + (unsigned int)(stop - 1 - j), stage = n % kSpStages;
                if (!waited(&sh->v_full[stage], (n / kSpStages) & 1u)) ok = false;
                const int token = k0 + (int)tile_row, warp_token = token - (int)lane;
                bool unseen = token < hull_first || token >= solid_end;
                if (warp_token < w->hull_end && warp_token + 32 > solid_end) {
                    // behind a gap: a lane looks which of the warp's 32 tokens some of the rows see
                    uint32_t some = 0u;
                    for (unsigned int at = lane; at < 2u * tile_rows; at += 32u) {
                        const int lo = max(w->first[at] - warp_token, 0), hi = min(w->end[at] - warp_token, 32);
                        if (lo < hi) some |= (0xffffffffu >> (32 - hi)) & (0xffffffffu << lo);
                    }
                    some = __reduce_or_sync(0xffffffffu, some);
                    unseen = !(some >> lane & 1u);
                }
                if (unseen) {
                    unsigned char *v_row = v_smem + stage * kSpTileBytes + tile_row * 128u;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        // eight rows write to eight different groups of banks
                        const unsigned int at = 16u * (i ^ (tile_row & 7u));
                        *reinterpret_cast<uint4 *>(v_row + at) = make_uint4(0u, 0u, 0u, 0u);
                        *reinterpret_cast<uint4 *>(v_row + kSpHalfBytes + at) = make_uint4(0u, 0u, 0u, 0u);
                    }
                }
                fence_proxy_async();
            }
            // rows that do not exist (their Q is zero, nothing is stored) ask for no mask
            const int lo = exists ? range.first - k0 : 0, hi = exists ? range.end - k0 : kSpN;
            bool cut[2];   // tokens 64 h .. 64 h + 63: some row of the warp does not see all of them
#pragma unroll
            for (int h = 0; h < 2; ++h) cut[h] = __any_sync(0xffffffffu, lo > 64 * h || hi < 64 * h + 64);
            // a value inside the run [lo, hi) against two ramps: at least kHuge / 2 inside, at most -kHuge / 2 outside,
            // and the smallest of the three hides what stands there (min passes over a NaN)
            constexpr float kHuge = 1e30f;
            const float up = kHuge * (0.5f - (float)max(lo, -kSpN)), down = kHuge * ((float)min(max(hi, -1), 2 * kSpN) - 0.5f);
            auto hide = [&](float value, int c) { return min3(value, fmaf((float)c, kHuge, up), fmaf((float)c, -kHuge, down)); };
            // the bias of column c: slope * (ahead + c), or -slope * |ahead + c| where a row sees tokens behind itself
            const int ahead = BIAS ? k0 - range.position : 0;
            const bool linear = !BIAS || __all_sync(0xffffffffu, !exists || min(range.end, k0 + kSpN) <= range.position + 1);
            const float ahead_f = BIAS && linear ? (float)ahead : 0.0f;
            // The reference m follows the maximum when it lags by more than 2^8. P of the previous tile is overwritten
            // afterwards, and O may be touched: its P V has to have landed.
            auto landed = [&]() {
                if (j < my_until - 1 && !waited(&sh->pv_done[x], parity ^ 1u)) ok = false;
            };
            auto agree = [&](float found) {
                landed();
                const bool grow = found > m + kSpRescale || (m == -INFINITY && found > -INFINITY);
                if (__any_sync(0xffffffffu, grow)) {
                    const float fresh = grow ? found : m, factor = m == -INFINITY ? 1.0f : exp2_approx(m - fresh);
                    m = fresh;
                    l *= factor;
                    if (j < my_until - 1) {
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int i = 0; i < 8; ++i) {
                            uint32_t o[16];
                            tmem_ld16(o_col + 16 * i, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * factor);
                            tmem_st16(o_col + 16 * i, o);
                        }
                        tmem_wait_st();
                    }
                }
                return m == -INFINITY ? 0.0f : fmaf(slope2, ahead_f, -m);
            };
            auto hand_over = [&](const uint32_t (&packed)[32], int h) {
                tmem_st32(p_col + 32 * h, packed);
                tmem_wait_st();
                tc_fence_before_sync();
                mbar_arrive(&sh->p_half[x][h]);      // weights of tokens 64 h .. 64 h + 63
            };
            unsigned long long sum2[2] = {0ull, 0ull};
            // ---- a cap: how large the products are decides on the form of tanh ---------------------------------------
            bool done = false, small = false;   // (a cap without a bias: also, whether a maximum is needed)
            if (CAP) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (cut[h]) {   // columns that a row does not see may hold anything
#pragma unroll
                        for (int c = 64 * h; c < 64 * h + 64; ++c)
                            if (c < lo || c >= hi) s[c >> 5][c & 31] = 0u;
                    }
                float top[2] = {0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 128; i += 2)
                    top[(i >> 1) & 1] = max3_abs(top[(i >> 1) & 1], __uint_as_float(s[i >> 5][i & 31]), __uint_as_float(s[i >> 5][(i & 31) + 1]));
                const float largest = fmaxf(top[0], top[1]);
                small = __all_sync(0xffffffffu, largest <= inside_small);
                // x p(x^2), the exponential, sum and rounding of both halves as one straight run of instructions (a branch
                // between the halves costs the common tile 13 %). The short polynomial takes the products as they are,
                // to_unit folded into its coefficients; the long one, whose coefficients would leave F32's range, x itself.
                auto weights = [&](const auto &a) {
                    constexpr int kTerms = sizeof(a) / sizeof(a[0]);
                    constexpr bool kFolded = kTerms == 4;
                    unsigned long long poly2[kTerms];   // each coefficient twice
                    float power = mul * (kFolded ? to_unit : 1.0f);
#pragma unroll
                    for (int i = 0; i < kTerms; ++i) {
                        poly2[i] = f2_pack(a[i] * power, a[i] * power);
                        if (kFolded) power *= to_unit * to_unit;
                    }
                    const unsigned long long unit2 = f2_pack(to_unit, to_unit);
                    const unsigned long long minus_m2 = f2_pack(-m, -m);
                    landed();
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t packed[32];
#pragma unroll
                        for (int i = 0; i < 64; i += 2) {
                            unsigned long long v = f2_load(s[2 * h + (i >> 5)], i & 31);
                            if (!kFolded) {
                                asm volatile("" : "+l"(v));   // or what both forms share is drawn in front of their branch
                                v = f2_mul(v, unit2);
                            }
                            const unsigned long long w2 = f2_mul(v, v);
                            unsigned long long r = poly2[kTerms - 1];
#pragma unroll
                            for (int k = kTerms - 2; k >= 0; --k) r = f2_fma(r, w2, poly2[k]);
                            float e0, e1;
                            f2_unpack(f2_fma(v, r, minus_m2), e0, e1);
                            e0 = exp2_approx(e0);
                            e1 = exp2_approx(e1);
                            sum2[(i >> 1) & 1] = f2_add(sum2[(i >> 1) & 1], f2_pack(e0, e1));
                            packed[i >> 1] = pack_bf16(e0, e1);
                        }
                        hand_over(packed, h);
                    }
                };
                // |cap tanh x| <= |cap x| bounds every logit of the tile: the reference that the row has will do
                if (!BIAS && small && !cut[0] && !cut[1] && __all_sync(0xffffffffu, largest * (mul * to_unit) <= m + kSpNear)) {
                    if (__all_sync(0xffffffffu, largest <= inside_tiny)) weights(kSpTanhTiny);
                    else weights(kSpTanhSmall);
                    done = true;
                }
            }
            if (!done) {
                // ---- without a cap: raw products, the bias in their units; with one: logits in log2 units. Then the mask,
                // the maximum and the weights are the same for all.
                if (CAP) {
                    const float to_exp = to_unit * (2.0f * kScoredLog2e);
                    if (small) {
                        const unsigned long long unit2 = f2_pack(to_unit, to_unit);
#pragma unroll
                        for (int i = 0; i < 128; i += 2) {
                            const unsigned long long v = f2_mul(f2_load(s[i >> 5], i & 31), unit2), w2 = f2_mul(v, v);
                            unsigned long long r = f2_pack(kSpTanhSmall[6] * mul, kSpTanhSmall[6] * mul);
#pragma unroll
                            for (int k = 5; k >= 0; --k) r = f2_fma(r, w2, f2_pack(kSpTanhSmall[k] * mul, kSpTanhSmall[k] * mul));
                            f2_store(f2_mul(v, r), s[i >> 5], i & 31);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < 128; ++c) {
                            const float value = __uint_as_float(s[c >> 5][c & 31]), x = value * to_unit;
                            const float curve = fmaf(-2.0f * mul, rcp_approx(exp2_approx(value * to_exp) + 1.0f), mul);
                            float r = kSpTanhSmall[6];
#pragma unroll
                            for (int k = 5; k >= 0; --k) r = fmaf(r, x * x, kSpTanhSmall[k]);
                            s[c >> 5][c & 31] = __float_as_uint(WIDE && fabsf(x) <= 1.375f ? x * mul * r : curve);
                        }
                    }
                }
                if (BIAS) {
                    if (linear) {
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            s[c >> 5][c & 31] = __float_as_uint(fmaf((float)c, slope_held, __uint_as_float(s[c >> 5][c & 31])));
                    } else {
#pragma unroll
                        for (int c = 0; c < 128; ++c)
                            s[c >> 5][c & 31] =
                                __float_as_uint(fmaf(-slope_held, fabsf((float)(ahead + c)), __uint_as_float(s[c >> 5][c & 31])));
                    }
                }
                if (cut[0] || cut[1]) {
#pragma unroll
                    for (int c = 0; c < 128; ++c)
                        s[c >> 5][c & 31] = __float_as_uint(hide(__uint_as_float(s[c >> 5][c & 31]), c));
                }
                const float held = CAP ? 1.0f : mul;
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 128; i += 2)
                    top[(i >> 1) & 1] = max3(top[(i >> 1) & 1], __uint_as_float(s[i >> 5][i & 31]), __uint_as_float(s[i >> 5][(i & 31) + 1]));
                const float found = fmaxf(top[0], top[1]);
                float offset = agree(found < -1e29f ? -INFINITY : fmaf(found, held, slope2 * ahead_f));
                if (found > 1e29f) offset = __int_as_float(0x7fffffff);   // a NaN (or infinity) inside the run: not lost in the mask
                const unsigned long long offset2 = f2_pack(offset, offset), held2 = f2_pack(held, held);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t packed[32];
#pragma unroll
                    for (int i = 0; i < 64; i += 2) {
                        float e0, e1;
                        f2_unpack(f2_fma(f2_load(s[2 * h + (i >> 5)], i & 31), held2, offset2), e0, e1);
                        e0 = exp2_approx(e0);
                        e1 = exp2_approx(e1);
                        sum2[(i >> 1) & 1] = f2_add(sum2[(i >> 1) & 1], f2_pack(e0, e1));
                        packed[i >> 1] = pack_bf16(e0, e1);
                    }
                    hand_over(packed, h);
                }
            }
            float sum_lo, sum_hi;
            f2_unpack(f2_add(sum2[0], sum2[1]), sum_lo, sum_hi);
            l += sum_lo + sum_hi;
        }
        // ------------------------------ epilogue ----------------------------------------------------
        const bool any = my_until > my_from;
        tiles += (unsigned int)(stop - start);
        if (any && !waited(&sh->pv_done[x], (count - 1u) & 1u)) ok = false;
        if (!ok) {
            fail();
        } else {
            tc_fence_after_sync();
            const float inverse = SPLIT ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            // A thread holds a row, a store wants lanes side by side: 64 bytes of each row (32 bf16 or 16 F32 lanes) at a
            // time go through shared memory, their four 16-byte pieces in an order that spreads them over the banks.
            unsigned char *const out = out_smem + warp * kSpOutBytes;
            const bool narrow = !SPLIT && p.output_dtype == YVEX_DTYPE_BF16, sees = range.first < range.end;
            const unsigned int q0 = w->q0 + x * tile_rows, head = w->head, b = w->b, split = w->split;
            const unsigned int out_lane = lane >> 2, width = narrow ? 2u : 4u;
            const unsigned long long item0 = ((unsigned long long)b * p.query_rows + q0) * p.query_heads + head;
            unsigned char *dst[4];   // of the rows that this thread stores, null where there is none
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const unsigned int place = sh->where[(warp & 3u) * 32u + 8u * i + out_lane];
                const unsigned long long item = item0 + (unsigned long long)(place & 0xffffu) * p.query_heads + (place >> 16);
                dst[i] = place == ~0u || q0 + (place & 0xffffu) >= p.query_rows ? nullptr
                         : 16u * (lane & 3u) + (SPLIT ? reinterpret_cast<unsigned char *>(scored_partial(p, item, split))
                                                      : reinterpret_cast<unsigned char *>(p.output) + item * kSpD * width);
            }
            // NaN once a lane is not finite, or when all that the row sees fell below the mask's range
            float check = sees && l == 0.0f ? __int_as_float(0x7fffffff) : l * 0.0f;
            uint4 staged[4];
            auto send = [&](int chunk) {
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4 *>(out + lane * 64u + 16u * (i ^ ((lane >> 1) & 3u))) = staged[i];
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const unsigned int r = 8u * i + out_lane;
                    const uint4 piece = *reinterpret_cast<const uint4 *>(out + r * 64u + 16u * ((lane & 3u) ^ ((r >> 1) & 3u)));
                    if (dst[i]) *reinterpret_cast<uint4 *>(dst[i] + 64 * chunk) = piece;
                }
                __syncwarp();
            };
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                uint32_t o[32];
#pragma unroll
                for (int c = 0; c < 32; ++c) o[c] = 0u;
                if (any) {
                    tmem_ld32(o_col + 32 * i, o);
                    tmem_wait_ld();
                }
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    const float v = sees ? __uint_as_float(o[c]) * inverse : 0.0f;
                    check = fmaf(v, 0.0f, check);
                    o[c] = __float_as_uint(v);
                }
                if (narrow) {
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        (&staged[c >> 2].x)[c & 3] = pack_bf16(__uint_as_float(o[2 * c]), __uint_as_float(o[2 * c + 1]));
                    send(i);
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int c = 0; c < 16; ++c) (&staged[c >> 2].x)[c & 3] = o[16 * h + c];
                        send(2 * i + h);
                    }
                }
            }
            if (exists) {
                const unsigned int mine = sh->where[tile_row];
                if (SPLIT) {
                    float *part = scored_partial(p, item0 + (unsigned long long)(mine & 0xffffu) * p.query_heads + (mine >> 16), split);
                    part[kSpD] = m, part[kSpD + 1] = l;
                }
                if (check != 0.0f) atomicCAS(p.status, 0, YVX_STATUS_NONFINITE);
            }
        }
        give_back(turn);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 9) tmem_dealloc(tmem, kSpTmemColumns);
}

bool scored_encode_rows(CUtensorMap *map, const void *base, int element_bytes, unsigned long long token_stride,
                        unsigned long long head_stride, unsigned long long outer_stride, unsigned long long tokens,
                        unsigned long long heads, unsigned long long outer, bool head_inner, unsigned int box_tokens,
                        unsigned int box_heads);

// 1: launched, 0: not this kernel's shape, negative: an error.
int scored_prompt_launch(const yvx_scored_problem &p, bool staged, cudaStream_t stream)
{
    const unsigned long long head_stride = p.query_head_stride ? p.query_head_stride : kSpD;
    if (p.head_dim != (unsigned)kSpD || p.query_dtype != YVEX_DTYPE_BF16 || p.kv_code != YVX_KV_PLAIN ||
        p.kv_dtype != YVEX_DTYPE_BF16 || (reinterpret_cast<uintptr_t>(p.output) & 15u) ||
        (p.block_table && p.block_tokens % 64u) || head_stride > p.query_row_stride)
        return 0;
    const bool head_inner = p.key_head_stride < p.key_token_stride;
    const unsigned int pack = scored_packed_heads(p), pair_rows = 2u * (kSpM / pack);
    if ((p.value_head_stride < p.value_token_stride) != head_inner) return 0;
    const unsigned long long tokens = p.block_table ? p.block_tokens : staged ? scored_stage_tokens(p) : p.kv_tokens_max;
    const unsigned long long outer = p.block_table ? p.pool_blocks : p.sessions;
    SpMaps maps;
    if (!scored_encode_rows(&maps.query, p.query, 2, p.query_row_stride, head_stride, p.query_session_stride, p.query_rows,
                            p.query_heads, p.sessions, true, kSpM / pack, pack) ||
        !scored_encode_rows(&maps.key, p.key, 2, p.key_token_stride, p.key_head_stride, p.key_outer_stride, tokens,
                            p.kv_heads, outer, head_inner, 64u, 1u) ||
        !scored_encode_rows(&maps.value, p.value, 2, p.value_token_stride, p.value_head_stride, p.value_outer_stride,
                            tokens, p.kv_heads, outer, head_inner, 64u, 1u))
        return 0;
    // lanes whose K + V fit half of the 126 MB L2 together form a group
    const unsigned long long lanes = (unsigned long long)(p.query_heads / pack) * p.sessions, group = p.query_heads / p.kv_heads / pack;
    unsigned long long streams = (64ull << 20) / ((unsigned long long)p.kv_tokens_max * kSpD * 4ull);
    if (streams < 1ull) streams = 1ull;
    const unsigned long long lane_group = streams * group < lanes ? streams * group : lanes;
    const unsigned long long pairs = (p.query_rows + pair_rows - 1ull) / pair_rows;
    const unsigned long long ctas = (lanes + lane_group - 1ull) / lane_group * lane_group * pairs * p.max_splits;
    if (lanes > 0xffffffffull || ctas > 0x7fffffffull) return 0;
    const bool cap = p.cap > 0.0f, bias = p.slopes != nullptr;
    typedef void (*Kernel)(const yvx_scored_problem, const SpMaps, const int, const unsigned int, const int);
    const Kernel kernels[4][3] = {   // without a cap, with one, with a wide one
        {scored_prompt_kernel<false, false, false, false>, scored_prompt_kernel<true, false, false, false>, scored_prompt_kernel<true, false, false, true>},
        {scored_prompt_kernel<false, true, false, false>, scored_prompt_kernel<true, true, false, false>, scored_prompt_kernel<true, true, false, true>},
        {scored_prompt_kernel<false, false, true, false>, scored_prompt_kernel<true, false, true, false>, scored_prompt_kernel<true, false, true, true>},
        {scored_prompt_kernel<false, true, true, false>, scored_prompt_kernel<true, true, true, false>, scored_prompt_kernel<true, true, true, true>}};
    const Kernel kernel = kernels[(bias ? 1 : 0) + (p.max_splits > 1u ? 2 : 0)][cap ? p.cap > kSpWideCap ? 2 : 1 : 0];
    YVX_CUDA_TRY(cudaFuncSetAttribute((const void *)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSpSmemBytes));
    kernel<<<dim3((unsigned int)ctas, 1, 1), kSpThreads, kSpSmemBytes, stream>>>(p, maps, head_inner ? 1 : 0,
                                                                              (unsigned int)lane_group, staged ? 1 : 0);
    const int rc = yvx_cuda_check(cudaGetLastError(), "scored_prompt_kernel");
    return rc != 0 ? rc : 1;
}

}  // namespace yvx
