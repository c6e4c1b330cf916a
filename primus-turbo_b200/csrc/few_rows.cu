// Products with few rows: one to some hundred tokens through a weight matrix, dense (bias, activation and residual in the
// epilogue) or through the chosen experts of a mixture (gate and up projection with the gated activation; down projection with
// the weighted sum).
//
// Bound: the bytes of the weights, each read once.  The weight is therefore the 128-row operand of tcgen05.mma and the tokens are
// its narrow one (N = 16 .. 256), so that a CTA streams 16 KiB weight blocks [128 features][64 of K] through a TMA ring and the
// tensor core takes each of them in four instructions, far faster than it arrives.  Blocks of up to 128 tokens: two CTAs to an SM with
// about 100 KiB each on their way, which covers the memory latency (148 SMs x 200 KiB = 29 MiB in flight) and lets one CTA's start and
// write-out hide behind the other's stream.  Up to 192: one CTA with 200 KiB and more warps for the write-out.  Up to 256: pairs of CTAs
// whose tensor cores multiply 256 features together (cta_group::2), each holding half of the tokens, because there what an SM takes in
// from L2 (about 108 GB/s) bounds it: 512 x 4096 x 4096 24.8 us by blocks of 192, 20.8 by pairs.
//   The contraction is split over the CTAs of a cluster when the features alone would leave SMs idle: every CTA puts its partial
// [tokens][128] block of fp32 sums into its own shared memory and the CTAs add each other's blocks for their share of the tokens
// through distributed shared memory, beginning with their own and going on by rank.  So there is no workspace, no counter and no
// atomic: results do not depend on timing, and calls on different streams or in different graphs share nothing.
//
//   warp 0      producer (TMA; for experts also which tokens chose them)
//   warp 1      one thread issues the MMAs; owns the tensor memory
//   the others  for experts: copy the tokens' rows into the stages; then tensor memory -> shared memory
//   all         sum over the cluster, epilogue, write-out
//
// Measured (B200, bf16, replayed graphs, inputs beyond L2): 1 x 14336 x 4096 (rows, features, K) 21.6 us, 5.4 TB/s of weights; 1 x
// 64128 x 4096 81 us, 6.5 TB/s; 64 x 4096 x 4096 11.3 us; 129 x 4096 x 4096 13.4 us; 333 x 4096 x 4096 18.2 us, 0.61 PFLOP/s.  One
// token through eight experts of 7168 x 2048 112.5 us, 6.3 TB/s; 64 tokens on 28 of 32 such experts 375 to 393 us, 6.3 to 6.5 TB/s.
//
// Mixture, two kernels:
//   GATE_UP  grid (blocks of 64 features x split, chosen experts): the block is 64 gate rows and the 64 up rows that belong to them.
//            The expert's tokens are the narrow operand, copied row by row from the list of them.  Writes p * act(g) * u, with p
//            the slot's probability (the sum of them where a token names an expert twice), rounded once to the tensors' type: the
//            next product's operand type.
//   DOWN     a CTA keeps one [128 features][tokens] accumulator over ALL chosen experts, one column per token, so the weighted
//            sum over a token's experts happens in tensor memory.  For every expert only the 16-token blocks that hold one of
//            its tokens are multiplied; the other tokens of such a block are rows of zeros.  Its first weight blocks are
//            fetched before the first kernel has finished (programmatic dependent launch): weights and routing do not depend
//            on it.
#include <algorithm>
#include <cmath>

#include "act_math.cuh"
#include "common.cuh"
#include "gemm_common.cuh"
#include "sm100_ptx.cuh"

namespace ptb {
using namespace sm100;

constexpr int kFrFeat = 128;              // features (weight rows) of a CTA
constexpr int kFrABytes = kFrFeat * 128;  // a weight block: 128 rows of 64 16-bit elements
constexpr int kFrMaxSlots = 2048;         // tokens x experts per token
constexpr int kFrMaxTopK = 32;
constexpr int kFrMaxSplit = 8;            // CTAs of a cluster
constexpr int kFrMaxStages = 12;          // of a ring
constexpr int kFrPairTok = 256;           // the block that pairs of CTAs take

enum FewRowsKind { FR_LINEAR = 0, FR_GATE_UP = 1, FR_DOWN = 2 };

struct FewRowsArgs {
    int rows;                // LINEAR: M; else tokens
    int n, k;                // features of the output (GATE_UP: of one half), contraction length
    int ring_bytes;          // of shared memory for stages
    int x_rows, stages;      // token rows of a stage, a multiple of 8; how many stages fit.  GATE_UP: by the expert's tokens, in the kernel
    int split;               // CTAs (wide blocks: pairs of CTAs) of a cluster
    int fmt;                 // 0 = fp16, 1 = bf16 operands
    void *out;               // LINEAR / DOWN [rows, n]; GATE_UP [slots, n]
    int out_dtype;
    int act;
    // LINEAR
    int block;               // tokens from one block to the next, at most TOK: a multiple of 16
    int w_mn;                // the weight is stored [k, n]: two boxes of 64 features x 64 contraction rows, read in place
    const void *bias, *residual;
    int bias_dtype;
    void *z;                 // pre-activation in the operands' type, or null
    int vec_ok;              // rows of out / residual / z / bias take four elements at a time
    // mixture
    const void *x;           // rows of x_pitch bytes: GATE_UP [tokens, k], DOWN [slots, k]
    int64_t x_pitch;
    const void *ids;         // [tokens, top_k] int32 / int64
    int id_bytes, top_k, experts;
    const float *probs;
    int *status;
};

template <int TOK, bool PAIR> struct FrCfg {
    // per quarter of the accumulator's rows: one, two or four that share the tokens
    static constexpr int kEpiWarps = TOK <= 32 ? 4 : TOK <= 128 ? 8 : 16;
    static constexpr int kThreads = 64 + 32 * kEpiWarps;
    static constexpr int kCtas = TOK > 128 ? 1 : 2;           // per SM
    // Six, five, four and three full stages of two CTAs per SM; five of single CTAs, six of pairs.  Smaller stages fit more often.
    static constexpr int kRing = (TOK <= 16 ? 6 : TOK <= 32 ? 5 : TOK <= 64 ? 4 : TOK <= 128 ? 3 : PAIR ? 6 : 5) * (kFrABytes + (PAIR ? TOK / 2 : TOK) * 128);
    static constexpr int kMaxRing = kCtas * kRing;            // of a launch that leaves an SM to each CTA
    static constexpr int kIdSlots = TOK * kFrMaxTopK < kFrMaxSlots ? TOK * kFrMaxTopK : kFrMaxSlots;
    static constexpr int smem_bytes(int ring) { return ring + 1024 /* alignment */ + 2 * kIdSlots; }
    static constexpr int kTmemCols = TOK < 32 ? 32 : TOK > 128 ? 256 : TOK;
    static_assert(TOK * kFrFeat * 4 <= kRing, "the partial block must fit the ring");
    static_assert(kCtas * (smem_bytes(kRing) + 3584 /* static and reserved */) <= 228 * 1024, "CTAs per SM");
    static_assert(smem_bytes(kMaxRing) + 3584 <= 228 * 1024, "one CTA per SM");
};

// Four elements of each of ROWS rows, under predicates
template <int ROWS> __device__ __forceinline__ void store4_rows(void *p, int dtype, int64_t at, int64_t pitch, const bool (&st)[ROWS], const float (&v)[ROWS][4]) {
    if (dtype == PT_F32) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (st[u]) *reinterpret_cast<float4 *>(reinterpret_cast<float *>(p) + at + u * pitch) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
    } else {
#pragma unroll
        for (int u = 0; u < ROWS; ++u) {
            const uint2 h = dtype == PT_BF16 ? make_uint2(pack2<__nv_bfloat16>(v[u][0], v[u][1]), pack2<__nv_bfloat16>(v[u][2], v[u][3]))
                                             : make_uint2(pack2<__half>(v[u][0], v[u][1]), pack2<__half>(v[u][2], v[u][3]));
            if (st[u]) *reinterpret_cast<uint2 *>(reinterpret_cast<uint16_t *>(p) + at + u * pitch) = h;
        }
    }
}
template <int ROWS> __device__ __forceinline__ void load4_rows(const void *p, int dtype, int64_t at, int64_t pitch, const bool (&st)[ROWS], uint4 (&raw)[ROWS]) {
#pragma unroll
    for (int u = 0; u < ROWS; ++u) raw[u] = make_uint4(0u, 0u, 0u, 0u);
    if (dtype == PT_F32) {
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (st[u]) raw[u] = *reinterpret_cast<const uint4 *>(reinterpret_cast<const float *>(p) + at + u * pitch);
    } else {
#pragma unroll
        for (int u = 0; u < ROWS; ++u)
            if (st[u]) {
                const uint2 h = *reinterpret_cast<const uint2 *>(reinterpret_cast<const uint16_t *>(p) + at + u * pitch);
                raw[u].x = h.x;
                raw[u].y = h.y;
            }
    }
}

template <int TOK, int KIND, bool PAIR>
__global__ void __launch_bounds__(FrCfg<TOK, PAIR>::kThreads, FrCfg<TOK, PAIR>::kCtas)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, FewRowsArgs a) {
    using Cfg = FrCfg<TOK, PAIR>;
    constexpr bool kMoe = KIND != FR_LINEAR, kPair = PAIR;
    static_assert(!kMoe || (TOK <= 128 && !PAIR), "wide blocks are for dense products");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int16_t *s_ids = reinterpret_cast<int16_t *>(ring + a.ring_bytes);   // [tokens * top_k], -1: no expert of this call
    __shared__ uint64_t full_bar[kFrMaxStages], empty_bar[kFrMaxStages], done_bar;
    __shared__ uint32_t s_tmem, s_mask[kFrMaxStages], s_touched;   // s_mask: DOWN, which 16-token blocks a stage holds
    __shared__ int s_abort, s_count;
    __shared__ uint32_t s_bits[kMoe ? 32 : 1];
    __shared__ int16_t s_active[KIND == FR_DOWN ? kMaxGroups : 1];
    __shared__ int s_row[KIND == FR_GATE_UP ? TOK : 1], s_slot[KIND == FR_GATE_UP ? TOK : 1];
    __shared__ float s_prob[KIND == FR_GATE_UP ? TOK : 1];

    const int warp = __shfl_sync(0xffffffffu, (int) threadIdx.x >> 5, 0), lane = threadIdx.x & 31;   // the shuffle tells the compiler: uniform
    // `rank`: which share of the contraction.  Wide blocks: CTAs 2 rank and 2 rank + 1 of the cluster are a pair.
    const bool cluster = kPair || a.split > 1;
    const int cta_rank = cluster ? (int) cluster_ctarank() : 0, half = kPair ? cta_rank & 1 : 0;
    const int rank = kPair ? cta_rank >> 1 : cta_rank;
    const int tile = kPair ? (int) blockIdx.x / (2 * a.split) * 2 + half : (int) blockIdx.x / a.split;
    const int T = a.rows;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < (KIND == FR_GATE_UP ? kFrMaxStages : a.stages); ++s) {
            mbar_init(&full_bar[s], kMoe ? 1 + 32 * Cfg::kEpiWarps : 1);   // the weights' bytes, and the copying threads
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 2);   // the MMA thread's commit, and an arrival of this CTA's warp 1 (publishes s_tmem and s_touched)
        fence_barrier_init();
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_x);
    }
    if (TOK <= 128 && warp == 1) {   // while the kernel before this one finishes
        tmem_alloc(&s_tmem, Cfg::kTmemCols);
        tmem_relinquish();
    }
    if (KIND == FR_LINEAR && threadIdx.x == 64 && blockIdx.y == 0 && tile * kFrFeat < a.n) {
        // The first weight blocks on their way into L2 while the kernel before this one finishes.  A prefetch is not a read: were the
        // weight being written, L2 would hold the new values all the same.
        constexpr int kPrefetch = 6;
        const int chunks = (a.k + 63) / 64, l0 = chunks * rank / a.split, l1 = chunks * (rank + 1) / a.split;
        for (int l = l0; l < min(l1, l0 + kPrefetch); ++l) {
            if (a.w_mn) {
                prefetch_l2_2d(&tmap_w, tile * kFrFeat * 2, l * 64);
                prefetch_l2_2d(&tmap_w, tile * kFrFeat * 2 + 128, l * 64);
            } else {
                prefetch_l2_2d(&tmap_w, l * 128, tile * kFrFeat);
            }
        }
    }
    if (KIND != FR_DOWN) {   // DOWN waits later: what it reads up to there is not written by the kernel before it
        grid_dep_wait();
        // after this warp's allocation: what is launched then cannot wait for us holding its columns
        if (TOK <= 128 && warp == 1) grid_dep_launch();
    }

    // ---- routing: which experts are chosen, and by whom
    int cnt = KIND == FR_LINEAR ? min(a.block, T - (int) blockIdx.y * a.block) : 0;   // rows of this CTA
    int expert = 0, n_active = 0;
    if constexpr (kMoe) {
        if (threadIdx.x < 32) s_bits[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < T * a.top_k; i += Cfg::kThreads) {
            int64_t id;
            if constexpr (KIND == FR_DOWN) {   // before its wait for the kernel ahead: from L2, where what was written earlier stands, not from L1
                id = a.id_bytes == 8 ? (int64_t) __ldcg(reinterpret_cast<const long long *>(a.ids) + i)
                                     : (int64_t) __ldcg(reinterpret_cast<const int *>(a.ids) + i);
            } else {
                id = a.id_bytes == 8 ? reinterpret_cast<const int64_t *>(a.ids)[i] : (int64_t) reinterpret_cast<const int *>(a.ids)[i];
            }
            const bool valid = id >= 0 && id < a.experts;
            s_ids[i] = valid ? (int16_t) id : (int16_t) -1;
            if (valid) atomicOr(&s_bits[id >> 5], 1u << (id & 31));
        }
        __syncthreads();
        const uint32_t bits = s_bits[lane];
        int incl = __popc(bits);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        n_active = __shfl_sync(0xffffffffu, incl, 31);
        const int excl = incl - __popc(bits);
        if constexpr (KIND == FR_GATE_UP) {
            const int want = (int) blockIdx.y;
            if (want >= n_active) {   // the same for every CTA of the cluster
                if (warp == 1) tmem_dealloc(s_tmem, Cfg::kTmemCols);
                return;
            }
            const bool here = want >= excl && want < incl;
            uint32_t b = bits;
            for (int i = here ? want - excl : 0; i > 0; --i) b &= b - 1;
            const uint32_t who = __ballot_sync(0xffffffffu, here);
            expert = __shfl_sync(0xffffffffu, lane * 32 + __ffs(b) - 1, __ffs(who) - 1);
            if (warp == 0) {   // its tokens, in order; the probability of a slot named twice is the sum
                int base = 0;
                for (int t0 = 0; t0 < T; t0 += 32) {
                    const int t = t0 + lane;
                    int slot = -1;
                    float p = 0.f;
                    if (t < T)
                        for (int j = 0; j < a.top_k; ++j)
                            if (s_ids[t * a.top_k + j] == expert) {
                                if (slot < 0) slot = t * a.top_k + j;
                                p += a.probs[t * a.top_k + j];
                            }
                    const uint32_t has = __ballot_sync(0xffffffffu, slot >= 0);
                    if (slot >= 0) {
                        const int at = base + __popc(has & ((1u << lane) - 1));
                        s_row[at] = t; s_slot[at] = slot; s_prob[at] = p;
                    }
                    base += __popc(has);
                }
                if (lane == 0) s_count = base;
            }
        } else {
            if (warp == 0) {
                int at = excl;
                for (uint32_t b = bits; b != 0; b &= b - 1) s_active[at++] = (int16_t) (lane * 32 + __ffs(b) - 1);
            }
        }
    }
    tc_fence_before_sync();
    __syncwarp();
    if constexpr (kPair) cluster_sync_all();   // the other CTA's barriers stand before anything arrives there
    else __syncthreads();
    tc_fence_after_sync();
    if constexpr (KIND == FR_GATE_UP) cnt = s_count;
    if constexpr (KIND == FR_DOWN) cnt = T;

    // ---- the stages and this CTA's share of the contraction
    const int stage_bytes = kFrABytes + (KIND == FR_GATE_UP ? (cnt + 15) / 16 * 16 : a.x_rows) * 128;
    const int stages = KIND == FR_GATE_UP ? min(kFrMaxStages, a.ring_bytes / stage_bytes) : a.stages;
    const int chunks = (a.k + 63) / 64;   // per expert
    const int64_t total = KIND == FR_DOWN ? (int64_t) n_active * chunks : chunks;
    const int l0 = (int) (total * rank / a.split), l1 = (int) (total * (rank + 1) / a.split);
    if (TOK > 128 && warp == 1) {   // one CTA per SM starts when the kernel before it is done: the first loads do not wait for this (0.5 us)
        if constexpr (kPair) {
            tmem_alloc_pair(&s_tmem, Cfg::kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(&s_tmem, Cfg::kTmemCols);
            tmem_relinquish();
        }
        grid_dep_launch();
        __syncwarp();
    }
    volatile int *abort_flag = &s_abort;
    bool ok = true;

    if (warp == 0) {
        // ================================================================ producer
        const uint64_t stream_pol = l2_policy_evict_first(), keep_pol = l2_policy_evict_last();
        if constexpr (KIND != FR_DOWN) {
            if (elect_one()) {
                const int expert_row = expert * 2 * a.n + tile * 64;
                const int x_row = (int) blockIdx.y * a.block + half * 8 * ((cnt + 15) / 16);
                const uint32_t x_bytes = kMoe ? 0 : a.x_rows * 128;
                uint32_t stage = 0, phase = 0;
                for (int l = l0; l < l1; ++l) {
                    if (!(ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag))) break;
                    uint8_t *A = ring + stage * stage_bytes;
                    if constexpr (kPair) {   // the bytes of both CTAs on the barrier of the first
                        const uint32_t full = map_to_rank(&full_bar[stage], cta_rank & ~1);
                        if (half == 0) mbar_arrive_expect_tx(&full_bar[stage], 2 * (kFrABytes + x_bytes));
                        if (a.w_mn) {
                            tma_load_2d_pair_hint(A, &tmap_w, full, tile * kFrFeat * 2, l * 64, stream_pol);
                            tma_load_2d_pair_hint(A + kFrABytes / 2, &tmap_w, full, tile * kFrFeat * 2 + 128, l * 64, stream_pol);
                        } else {
                            tma_load_2d_pair_hint(A, &tmap_w, full, l * 128, tile * kFrFeat, stream_pol);
                        }
                        tma_load_2d_pair_hint(A + kFrABytes, &tmap_x, full, l * 128, x_row, keep_pol);
                        if (++stage == stages) { stage = 0; phase ^= 1; }
                        continue;
                    }
                    mbar_arrive_expect_tx(&full_bar[stage], kFrABytes + x_bytes);
                    if (KIND == FR_GATE_UP) {
                        tma_load_2d_hint(A, &tmap_w, &full_bar[stage], l * 128, expert_row, stream_pol);
                        tma_load_2d_hint(A + kFrABytes / 2, &tmap_w, &full_bar[stage], l * 128, expert_row + a.n, stream_pol);
                    } else {
                        if (a.w_mn) {
                            tma_load_2d_hint(A, &tmap_w, &full_bar[stage], tile * kFrFeat * 2, l * 64, stream_pol);
                            tma_load_2d_hint(A + kFrABytes / 2, &tmap_w, &full_bar[stage], tile * kFrFeat * 2 + 128, l * 64, stream_pol);
                        } else {
                            tma_load_2d_hint(A, &tmap_w, &full_bar[stage], l * 128, tile * kFrFeat, stream_pol);
                        }
                        tma_load_2d_hint(A + kFrABytes, &tmap_x, &full_bar[stage], l * 128, x_row, keep_pol);
                    }
                    if (++stage == stages) { stage = 0; phase ^= 1; }
                }
            }
        } else {
            // the weights of the chosen experts one after the other, and for every stage which 16-token blocks hold one of its tokens;
            // nothing here depends on the kernel before this one
            int ai = l0 / max(chunks, 1), c = l0 - ai * chunks, cur = -1;
            uint32_t blocks = 0, stage = 0, phase = 0;
            for (int l = l0; l < l1; ++l) {
                if (ai != cur) {
                    cur = ai;
                    blocks = 0;
                    for (int t0 = 0; t0 < TOK; t0 += 32) {
                        bool has = false;
                        if (t0 + lane < T)
                            for (int j = 0; j < a.top_k; ++j) has |= s_ids[(t0 + lane) * a.top_k + j] == s_active[ai];
                        const uint32_t who = __ballot_sync(0xffffffffu, has);
                        blocks |= (uint32_t) ((who & 0xFFFFu) != 0) << (t0 / 16) | (uint32_t) ((who >> 16) != 0) << (t0 / 16 + 1);
                    }
                }
                if (lane == 0 && (ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag))) {
                    s_mask[stage] = blocks;
                    mbar_arrive_expect_tx(&full_bar[stage], kFrABytes);
                    tma_load_2d_hint(ring + stage * stage_bytes, &tmap_w, &full_bar[stage], c * 128, s_active[ai] * a.n + tile * kFrFeat, stream_pol);
                }
                if (!(ok = __shfl_sync(0xffffffffu, (int) ok, 0) != 0)) break;
                if (++c == chunks) { c = 0; ++ai; }
                if (++stage == stages) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ================================================================ MMA issuer
        const uint32_t tmem = s_tmem;
        if (half == 1) {
            if (elect_one()) mbar_arrive(&done_bar);
        } else if (elect_one()) {
            const bool w_mn = KIND == FR_LINEAR && a.w_mn;
            const uint16_t both = (uint16_t) (3u << cta_rank);   // the CTAs of the pair
            const uint32_t idesc0 = idesc_f8(a.fmt, a.fmt, kPair ? 2 * kFrFeat : kFrFeat, 0) | ((uint32_t) w_mn << 15);
            const uint64_t w_step = w_mn ? (16 * 128) >> 4 : 32 >> 4;   // 16 contraction rows, or 32 bytes along a row
            uint32_t touched = 0;   // 16-token blocks that hold sums
            const uint32_t all = (1u << ((cnt + 15) / 16)) - 1;
            uint32_t stage = 0, phase = 0;
            for (int l = l0; l < l1; ++l) {
                if (!(ok = mbar_wait(&full_bar[stage], phase, abort_flag))) break;
                if constexpr (kMoe) fence_proxy_async_smem();   // the copied rows were written through the generic proxy
                tc_fence_after_sync();
                const uint32_t A = smem_u32(ring + stage * stage_bytes);
                const uint64_t a_desc = w_mn ? smem_desc_sw128_mn(A, kFrABytes / 2) : smem_desc_sw128(A);
                uint32_t m = KIND == FR_DOWN ? s_mask[stage] : all;
                const uint32_t used = m;
                while (m != 0) {   // runs of blocks that all hold sums, or none of which does
                    const int b0 = __ffs(m) - 1;
                    const uint32_t same = (touched >> b0 & 1) ? touched : ~touched;
                    const uint32_t run = ~((m & same) >> b0);
                    const int len = run == 0 ? 32 : __ffs(run) - 1;
                    const uint64_t b_desc = smem_desc_sw128(A + kFrABytes + b0 * 2048);
                    const uint32_t idesc = idesc0 | ((uint32_t) (2 * len) << 17);   // N = 16 len, in units of 8
                    const uint32_t acc0 = touched >> b0 & 1;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if constexpr (kPair) mma_f16_pair(tmem, a_desc + k * w_step, b_desc + 2 * k, idesc, acc0 | (uint32_t) (k > 0));
                        else mma_f16(tmem + 16 * b0, a_desc + k * w_step, b_desc + 2 * k, idesc, acc0 | (uint32_t) (k > 0));
                    }
                    m &= ~(((1u << len) - 1) << b0);
                }
                touched |= used;
                if constexpr (kPair) tc_commit_pair(&empty_bar[stage], both);
                else tc_commit(&empty_bar[stage]);
                if (++stage == stages) { stage = 0; phase ^= 1; }
            }
            if (ok) {
                s_touched = touched;
                mbar_arrive(&done_bar);
                if constexpr (kPair) tc_commit_pair(&done_bar, both);
                else tc_commit(&done_bar);
            }
        }
    }
    if constexpr (kMoe) {
        if (warp >= 2) {
            // ================================================================ rows of activations (the epilogue's warps, idle until then)
            // Every warp owns kMine consecutive rows of the token tile.  Eight lanes copy the 128 bytes of a row, 16 each, to where the swizzle
            // of the weights' TMA would put them; rows of other tokens and what lies past the contraction's end become zeros.  (TMA loads of
            // single rows, or of four with tile::gather4, cost their issuing thread 100 to 250 cycles each, and one warp copying all rows is
            // as slow: 816 and 617 us for 64 tokens on eight experts of 4096 x 14336.)
            constexpr int kMine = TOK / Cfg::kEpiWarps, kCopies = kMine / 4;
            static_assert(kMine % 4 == 0 && (16 % kMine == 0 || kMine % 16 == 0), "rows of a warp");
            const int first = (warp - 2) * kMine, c16 = (lane & 7) * 16;
            const uint8_t *base = reinterpret_cast<const uint8_t *>(a.x) + c16;
            const uint8_t *src[kCopies];   // null: a row of zeros
            uint32_t dst[kCopies];
#pragma unroll
            for (int i = 0; i < kCopies; ++i) {
                const int t = first + 4 * i + (lane >> 3);
                dst[i] = (uint32_t) (kFrABytes + t * 128 + (c16 ^ ((t & 7) << 4)));
                src[i] = KIND == FR_GATE_UP && t < cnt ? base + s_row[t] * a.x_pitch : nullptr;
            }
            bool needed = KIND == FR_GATE_UP && first / 16 * 16 < cnt;   // the multiplication reads the block these rows lie in
            if constexpr (KIND == FR_DOWN) grid_dep_wait();
            int ai = KIND == FR_DOWN ? l0 / max(chunks, 1) : 0, c = l0 - ai * chunks, cur = -1;
            uint32_t stage = 0, phase = 0;
            for (int l = l0; l < l1; ++l) {
                if (KIND == FR_DOWN && ai != cur) {   // the slots in which this warp's block of 16 tokens names the next expert
                    cur = ai;
                    const int t = first / 16 * 16 + (lane & 15);
                    int slot = -1;
                    if (t < T)
                        for (int j = a.top_k - 1; j >= 0; --j)
                            if (s_ids[t * a.top_k + j] == s_active[ai]) slot = t * a.top_k + j;   // the first of them
                    needed = __any_sync(0xffffffffu, slot >= 0);
#pragma unroll
                    for (int i = 0; i < kCopies; ++i) {
                        const int mine = __shfl_sync(0xffffffffu, slot, first % 16 + 4 * i + (lane >> 3));
                        src[i] = mine >= 0 ? base + mine * a.x_pitch : nullptr;
                    }
                }
                int good = 1;
                if (lane == 0) good = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag);
                if (!(ok = __shfl_sync(0xffffffffu, good, 0) != 0)) break;
                if (needed) {
                    const int64_t k0 = (int64_t) c * 128;
                    const bool inside = k0 + c16 < a.x_pitch;
#pragma unroll
                    for (int i = 0; i < kCopies; ++i)
                        cp_async_16_or_zero(ring + stage * stage_bytes + dst[i], src[i] != nullptr && inside ? src[i] + k0 : reinterpret_cast<const uint8_t *>(a.x),
                                            src[i] != nullptr && inside);
                }
                cp_async_arrive_noinc(&full_bar[stage]);
                if (++c == chunks) { c = 0; ++ai; }
                if (++stage == stages) { stage = 0; phase ^= 1; }
            }
        }
    }
    // ================================================================ partial sums -> shared memory (the ring is free by now)
    float *part = reinterpret_cast<float *>(ring);   // [tokens][128]
    const int blocks = (cnt + 15) / 16;
    if (warp >= 2) {
        const int q = warp & 3;   // tensor memory lanes this warp may read
        ok = mbar_wait_warp(&done_bar, 0, abort_flag);
        tc_fence_after_sync();
        const uint32_t touched = !ok ? 0 : kPair ? (l1 > l0 ? (1u << blocks) - 1 : 0) : s_touched;
        // Two blocks of 16 tokens at a time, both loads in flight.  They are made whether or not the columns hold sums (a pair never
        // reaches past the allocation): between a load and its wait nothing may touch the registers, a branch's merge neither.
        for (int b = 2 * ((warp - 2) >> 2); b < blocks; b += Cfg::kEpiWarps / 2) {
            uint32_t r[2][16];
            const uint32_t at = s_tmem + ((uint32_t) (q * 32) << 16) + 16 * b;
            tmem_ld16(at, r[0]);
            tmem_ld16(at + 16, r[1]);
            tmem_ld_wait();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (b + h >= blocks) continue;
                const bool have = touched >> (b + h) & 1;
#pragma unroll
                for (int i = 0; i < 16; ++i) part[(16 * (b + h) + i) * kFrFeat + q * 32 + lane] = have ? __uint_as_float(r[h][i]) : 0.f;
            }
        }
    }
    if (!ok || s_abort) {
        if (lane == 0) report_status(a.status, PT_ERR_TIMEOUT);
        __nanosleep(200000);   // let copies in flight land before the shared memory is released
    }
    tc_fence_before_sync();
    __syncwarp();
    if (cluster) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        if constexpr (kPair) tmem_dealloc_pair(s_tmem, Cfg::kTmemCols);
        else tmem_dealloc(s_tmem, Cfg::kTmemCols);
    }
    if constexpr (KIND == FR_DOWN) grid_dep_wait();

    // ================================================================ sum over the cluster, epilogue, write-out
    const uint32_t part_addr = smem_u32(part);
    // The features of a lane: four neighbours, accessed together; where a row of the output does not take that (ragged N), four that
    // lie 32 apart, so that the warp's scalar accesses stay coalesced.  GATE_UP: two of the gate half and the same two of the up half.
    const bool vec = KIND != FR_LINEAR || a.vec_ok;
    const uint32_t lane_at = KIND == FR_GATE_UP ? lane * 8 : vec ? lane * 16 : lane * 4;
    float bias[4] = {0.f, 0.f, 0.f, 0.f};
    const int f0 = KIND == FR_GATE_UP ? tile * 64 + 2 * lane : tile * kFrFeat + (vec ? 4 * lane : lane);
    if (KIND == FR_LINEAR && a.bias != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int f = vec ? f0 + i : f0 + 32 * i;
            if (f < a.n) bias[i] = load_as_f32(a.bias, a.bias_dtype, f);
        }
    }
    // A warp takes up to kAtOnce tokens at once.  There are few warps, so this part is bound by the latency of its instructions, not
    // their number: every step runs over all of the tokens before the next, under predicates instead of branches (128 x 4096 x 128: 7.6 us
    // with two tokens at once and a branch around each step, now 5.6).  The sums begin with this CTA's own block and go on with the other ranks'
    // after it, the loads of kOthers of them on their way before the first addition: a remote round trip takes about 0.6 us, and the
    // instantiations below make one do.
    const int step = a.split * (Cfg::kThreads / 32);   // tokens between two of this warp's
    auto write_out = [&](auto at_once, auto others) {
        constexpr int kAtOnce = decltype(at_once)::value, kOthers = decltype(others)::value;
        for (int t0 = rank + a.split * warp; t0 < cnt; t0 += kAtOnce * step) {
            float v[kAtOnce][4];
            bool in[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) in[u] = t0 + u * step < cnt;
            auto load = [&](int u, uint32_t src, bool remote, float (&w)[4]) {
                if (KIND == FR_GATE_UP) {
                    ld_cluster_f32x2(src, remote, in[u], w[0], w[1]);
                    ld_cluster_f32x2(src + 256, remote, in[u], w[2], w[3]);
                } else if (vec) {
                    ld_cluster_f32x4(src, remote, in[u], w);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) ld_cluster_f32(src + 128 * i, remote, in[u], w[i]);
                }
            };
            auto row_at = [&](int u) { return part_addr + (uint32_t) (t0 + u * step) * (kFrFeat * 4) + lane_at; };
            float w[kOthers > 0 ? kOthers : 1][kAtOnce][4];
#pragma unroll
            for (int s = 0; s < kOthers; ++s) {
                const int other = (rank + 1 + s) & (a.split - 1);
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) load(u, map_addr_to_rank(row_at(u), kPair ? 2 * other + half : other), true, w[s][u]);
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) load(u, row_at(u), false, v[u]);
#pragma unroll
            for (int s = 0; s < kOthers; ++s)
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[u][i] += w[s][u][i];
            if constexpr (KIND == FR_GATE_UP) {
                float p[kAtOnce];
                int slot[kAtOnce];
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const int t = in[u] ? t0 + u * step : 0;
                    p[u] = s_prob[t];
                    slot[u] = s_slot[t];
                }
                auto gated = [&](auto f) {
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                        for (int i = 0; i < 2; ++i) v[u][i] = f(v[u][i]) * v[u][2 + i] * p[u];
                };
                if (a.act == PT_ACT_SILU) gated([](float x) { return act_value<PT_ACT_SILU>(x); });
                else gated([](float x) { return gelu_epilogue(x); });
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const uint32_t h = a.fmt ? pack2<__nv_bfloat16>(v[u][0], v[u][1]) : pack2<__half>(v[u][0], v[u][1]);
                    if (in[u] && f0 < a.n) *reinterpret_cast<uint32_t *>(reinterpret_cast<uint16_t *>(a.out) + (int64_t) slot[u] * a.n + f0) = h;
                }
            } else if constexpr (KIND == FR_DOWN) {
                bool st[kAtOnce];
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) st[u] = in[u] && f0 < a.n;
                store4_rows<kAtOnce>(a.out, a.out_dtype, (int64_t) t0 * a.n + f0, (int64_t) step * a.n, st, v);
            } else {
                const int64_t o0 = ((int64_t) blockIdx.y * a.block + t0) * a.n + f0, o_step = (int64_t) step * a.n;
                const int zt = a.fmt ? PT_BF16 : PT_F16;
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[u][i] += bias[i];
                if (vec) {
                    bool st[kAtOnce];
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u) st[u] = in[u] && f0 < a.n;
                    uint4 res[kAtOnce];
                    if (a.residual != nullptr) load4_rows<kAtOnce>(a.residual, a.out_dtype, o0, o_step, st, res);
                    if (a.z != nullptr) store4_rows<kAtOnce>(a.z, zt, o0, o_step, st, v);
                    act_any_all<kAtOnce>(a.act, v);
                    if (a.residual != nullptr) {
#pragma unroll
                        for (int u = 0; u < kAtOnce; ++u) {
                            float x[4];
                            raw4_as_f32(res[u], a.out_dtype, x);
#pragma unroll
                            for (int i = 0; i < 4; ++i) v[u][i] += x[i];
                        }
                    }
                    store4_rows<kAtOnce>(a.out, a.out_dtype, o0, o_step, st, v);
                } else {
                    bool st[kAtOnce][4];
#pragma unroll
                    for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i) st[u][i] = in[u] && f0 + 32 * i < a.n;
                    uint32_t res[kAtOnce][4];   // raw, all on their way before the first is used
                    if (a.residual != nullptr) {
                        auto fetch = [&](auto *p) {
#pragma unroll
                            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    res[u][i] = 0;
                                    if (st[u][i]) res[u][i] = p[o0 + u * o_step + 32 * i];
                                }
                        };
                        if (a.out_dtype == PT_F32) fetch(reinterpret_cast<const uint32_t *>(a.residual));
                        else fetch(reinterpret_cast<const uint16_t *>(a.residual));
                    }
                    auto put = [&](void *out, int dtype) {
                        if (dtype == PT_F32) {
#pragma unroll
                            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if (st[u][i]) reinterpret_cast<float *>(out)[o0 + u * o_step + 32 * i] = v[u][i];
                        } else {
#pragma unroll
                            for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const uint32_t h = dtype == PT_BF16 ? pack2<__nv_bfloat16>(v[u][i], 0.f) : pack2<__half>(v[u][i], 0.f);
                                    if (st[u][i]) reinterpret_cast<uint16_t *>(out)[o0 + u * o_step + 32 * i] = (uint16_t) h;
                                }
                        }
                    };
                    if (a.z != nullptr) put(a.z, zt);
                    act_any_all<kAtOnce>(a.act, v);
                    if (a.residual != nullptr) {
#pragma unroll
                        for (int u = 0; u < kAtOnce; ++u)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                v[u][i] += a.out_dtype == PT_F32 ? __uint_as_float(res[u][i]) : a.out_dtype == PT_BF16 ? lo_f32<__nv_bfloat16>(res[u][i]) : lo_f32<__half>(res[u][i]);
                    }
                    put(a.out, a.out_dtype);
                }
            }
        }
    };
    using std::integral_constant;
    if (a.split == 1) write_out(integral_constant<int, TOK <= 16 ? 1 : TOK <= 32 ? 2 : 4>(), integral_constant<int, 0>());
    else if (a.split == 2) write_out(integral_constant<int, TOK <= 16 ? 2 : 4>(), integral_constant<int, 1>());
    else if (a.split == 4) write_out(integral_constant<int, TOK <= 16 ? 1 : TOK <= 64 ? 2 : 3>(), integral_constant<int, 3>());
    else if constexpr (!kPair) write_out(integral_constant<int, 1>(), integral_constant<int, kFrMaxSplit - 1>());
    if (a.split > 1) {
        __syncwarp();
        cluster_sync_all();   // no CTA leaves while another still reads its block
    }
}

// ------------------------------------------------------------------------------------------------ host side
// CTAs that are resident at once in clusters of `ctas`, two or one (wide) per SM.  GPCs do not divide evenly: on 148 SMs with one CTA per SM, 33
// clusters of four and 14 of eight ran together, 34 and 16 in two waves.  With two CTAs per SM no such loss was seen.
static double fr_resident(bool wide, int ctas) {
    const double sms = sm_count();
    return !wide ? 2.0 * sms : ctas <= 2 ? sms : ctas == 4 ? sms * 33 / 37 : sms * 28 / 37;
}
// Whether a launch of `ctas` CTAs on a kernel for two per SM takes the ring of both: if each of them gets an SM for itself.  Measured (us): 64 x
// 4096 x 4096 12.9 -> 12.0, 4000 x 512 x 512 11.9 -> 11.3; experts, 37 tokens in two of 60 of 1744 x 568 66.9 -> 63.9, but with 16 clusters of
// eight, of which two would start late, 64 tokens in six of 64 of 2048 x 1408 215 -> 271.  Up to 16 tokens it gains nothing (1 x 1024 x 4096 6.5
// -> 6.7).
static bool fr_deep(int tok, int64_t ctas, int cluster) { return tok > 16 && tok <= 128 && (double) ctas <= fr_resident(true, cluster); }

template <int TOK, int KIND, bool PAIR = false>
static int fr_launch(const CUtensorMap &tw, const CUtensorMap &tx, FewRowsArgs a, int64_t tiles, int64_t grid_y, cudaStream_t st) {
    using Cfg = FrCfg<TOK, PAIR>;
    auto kern = few_rows_kernel<TOK, KIND, PAIR>;
    static bool attr_set[64] = {};   // per instantiation and device
    const int dev = current_device_slot();
    if (!attr_set[dev]) {
        PT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem_bytes(Cfg::kMaxRing)));
        attr_set[dev] = true;
    }
    const int cluster_ctas = PAIR ? 2 * a.split : a.split;
    if (PAIR) tiles = ceil_div(tiles, 2);
    PT_REQUIRE(tiles * cluster_ctas < (1ll << 31) && grid_y < 65536, "few-row product: grid too large");
    a.ring_bytes = fr_deep(TOK, tiles * cluster_ctas * grid_y, cluster_ctas) ? Cfg::kMaxRing : Cfg::kRing;
    a.x_rows = KIND != FR_LINEAR ? TOK : PAIR ? a.block / 2 : a.block;
    a.stages = std::min(kFrMaxStages, a.ring_bytes / (kFrABytes + a.x_rows * 128));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (tiles * cluster_ctas), (unsigned) grid_y);
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = (size_t) Cfg::smem_bytes(a.ring_bytes);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned) cluster_ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    const bool overlap = getenv("PT_NO_PDL") == nullptr, cluster = cluster_ctas > 1;   // as in launch_overlapped
    cfg.attrs = overlap ? attr : attr + 1;
    cfg.numAttrs = (overlap ? 1 : 0) + (cluster ? 1 : 0);
    PT_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, tw, tx, a));
    return PT_OK;
}

// Estimated time of a launch in us: `tiles` weight blocks wide, `blocks` blocks of `block` tokens on the kernel for up to `tok`, `chunks`
// 64-wide steps of the contraction, s CTAs or pairs per cluster.  A fixed part, and the longest of: a CTA's own steps (an SM takes in about 108
// GB/s), the bytes from and to memory (one CTA per SM does not quite saturate it), all stages out of L2 (15 TB/s).  CTAs beyond those resident
// at once are further waves.  Measured (us, SiLU epilogue; rows x features x K, kernel : block / s): 64 x 4096 x 4096 64 / 1, 2, 4, 8 24.8,
// 16.1, 12.8, 13.0; 129 x 4096 x 4096 128 : 80 / 4 15.6, 192 : 144 / 2, 4 17.1, 13.6, 256 : 144 / 2, 4 16.7, 26.5 (two waves); 333 x 4096 x 4096
// 128 : 112 / 2 23.3, 192 : 176 / 2 19.0, 256 : 176 / 2 19.0; 512 x 4096 x 4096 128 : 128 / 2 24.6, 192 : 128 / 1 24.8, 256 : 256 / 2 21.1.
// What the estimates pick, the tiles of gemm_bias_act included, is within 5 % of the best plan in 41 of 54 sizes of 65 to 1030 rows and 22 %
// from it at worst (1030 x 4096 x 14336, 141 us); the misses are mostly products of 6 to 12 us.
static double fr_cost(int tok, int block, int64_t tiles, int64_t blocks, int64_t chunks, int s) {
    const bool wide = tok > 128, pair = tok == kFrPairTok;
    if (pair) tiles = (tiles + 1) / 2 * 2;
    const double ctas = (double) (tiles * blocks * s), share = ctas / fr_resident(wide, pair ? 2 * s : s);
    const double waves = std::max(1.0, wide ? std::ceil(share) : share);   // two CTAs per SM: a later one starts when either ends
    const double x_bytes = (pair ? 64.0 : 128.0) * block;   // of tokens per step
    // (Counting the deeper ring for 128 tokens too chose it over the wide kernel, whose write-out is faster: 512 x 1536 x 1024 9.7 -> 11.9 us.)
    const bool own_sm = wide || (tok <= 64 && fr_deep(tok, tiles * blocks * s, s));
    double step = pair ? 0.18 + 0.0007 * block : own_sm ? 0.2 + 0.0005 * block : 0.25 + 0.00125 * block;
    if (!wide && ctas > sm_count()) step = std::max(step, 2.0 * (kFrABytes + x_bytes) / 108e3);   // two CTAs share what an SM takes in
    const double rows = (double) (blocks * block), k_bytes = 128.0 * (double) chunks;
    const double memory = ((double) tiles * kFrFeat * (k_bytes + 2.0 * rows) + rows * k_bytes) / (!wide && ctas <= sm_count() ? 5.6e6 : 6.5e6);
    const double l2 = (double) (tiles * blocks * chunks) * (kFrABytes + x_bytes) / 15e6;
    double fixed;   // launch, first bytes, exchange of partial sums, write-out
    if (pair) fixed = s == 1 ? 5.7 + 0.0025 * block : 7.2 + 0.0075 * block;
    else if (wide) fixed = s == 1 ? 6.8 : 6.4 + 0.012 * block;
    else if (tok > 32) fixed = (s == 1 ? 4.2 : 5.1 + (0.0065 + 0.006 * s) * block) + (tok > 64 && ctas > sm_count() ? 3.0 : 0.0);
    else fixed = 4.5 + 0.008 * block * s;
    return fixed + std::max(waves * step * (double) ceil_div(chunks, s), std::max(memory, l2)) + (waves - 1.0) * (tok > 64 ? fixed + 5.0 : 6.0);
}
// Kernel, tokens per block and CTAs (pairs) per cluster with the smallest estimate.
struct FrPlan { int tok, block, split; double us; };
static FrPlan fr_plan(int64_t rows, int64_t n, int64_t k) {
    const int64_t tiles = ceil_div(n, kFrFeat), chunks = ceil_div(k, 64);
    FrPlan best{0, 0, 1, 0.0};
    for (int tok : {16, 32, 64, 128, 192, kFrPairTok}) {
        // no room, or more than half of it empty
        if ((tok < 128 && tok < rows) || (tok > 16 && tok <= 128 && tok / 2 >= rows) || (tok > 128 && rows <= 64)) continue;
        for (int more = 0; more <= (tok >= 128 && rows > 64 ? 1 : 0); ++more) {   // as few blocks as possible, or one more
            const int block = (int) ceil_div(ceil_div(rows, ceil_div(rows, tok) + more), 16) * 16;
            const int64_t blocks = ceil_div(rows, block);
            if (blocks > 65535) continue;   // the grid's second extent
            const int max_split = tok == kFrPairTok ? kFrMaxSplit / 2 : kFrMaxSplit;
            for (int s = 1; s <= max_split && (s == 1 || (tiles * blocks * s <= (tok > 128 ? 1 : 2) * (int64_t) sm_count() && chunks >= 2 * s)); s *= 2) {
                const double us = fr_cost(tok, block, tiles, blocks, chunks, s);
                if (best.tok == 0 || us < best.us) best = {tok, block, s, us};
            }
        }
    }
    return best;
}

// CTAs per cluster of the experts' kernels, by the same estimate with the number of experts that can be chosen.
static int fr_split_experts(int tok, int64_t tiles, int64_t chunks) {
    int best = 1;
    for (int s = 2; s <= kFrMaxSplit && tiles * s <= 2 * (int64_t) sm_count() && chunks >= 2 * s; s *= 2)
        if (fr_cost(tok, tok, tiles, 1, chunks, s) < fr_cost(tok, tok, tiles, 1, chunks, best)) best = s;
    return best;
}

template <int KIND>
static int fr_dispatch(const CUtensorMap &tw, const CUtensorMap &tx, const FewRowsArgs &a, int tok, int64_t tiles, int64_t grid_y, cudaStream_t st) {
    switch (tok) {
    case 16: return fr_launch<16, KIND>(tw, tx, a, tiles, grid_y, st);
    case 32: return fr_launch<32, KIND>(tw, tx, a, tiles, grid_y, st);
    case 64: return fr_launch<64, KIND>(tw, tx, a, tiles, grid_y, st);
    case 128: return fr_launch<128, KIND>(tw, tx, a, tiles, grid_y, st);
    }
    if constexpr (KIND == FR_LINEAR) {
        if (tok == 192) return fr_launch<192, KIND>(tw, tx, a, tiles, grid_y, st);
        if (tok == 256) return fr_launch<256, KIND, true>(tw, tx, a, tiles, grid_y, st);
    }
    return set_error(PT_ERR_INVALID, "few-row product: no kernel for %d tokens per block", tok);
}

double few_rows_us(int64_t M, int64_t N, int64_t K) { return fr_plan(M, N, K).us; }

// y = act(a . b^T + bias) + residual for few rows of a
int few_rows_linear(const void *a, const void *b, int b_mn, int ab_dtype, const void *bias, int bias_dtype, const void *residual, void *c, int c_dtype,
                    void *z, int act, int64_t M, int64_t N, int64_t K, int *status, cudaStream_t st) {
    const FrPlan plan = fr_plan(M, N, K);
    const int tok = plan.tok;
    CUtensorMap tw, tx;
    int rc;
    if ((rc = b_mn ? make_tmap_bytes(&tw, b, K, 2 * N, 2 * N, 64) : make_tmap_bytes(&tw, b, N, 2 * K, 2 * K, kFrFeat)) != PT_OK) return rc;
    if ((rc = make_tmap_bytes(&tx, a, M, 2 * K, 2 * K, tok == kFrPairTok ? plan.block / 2 : plan.block)) != PT_OK) return rc;
    FewRowsArgs r{};
    r.block = plan.block;
    r.w_mn = b_mn; r.rows = (int) M; r.n = (int) N; r.k = (int) K; r.fmt = ab_dtype == PT_BF16 ? 1 : 0;
    r.out = c; r.out_dtype = c_dtype; r.act = act; r.bias = bias; r.bias_dtype = bias_dtype; r.residual = residual; r.z = z; r.status = status;
    const int esize = c_dtype == PT_F32 ? 4 : 2;
    r.vec_ok = N % 4 == 0 && aligned(c, 4 * esize) && aligned(residual, 4 * esize) && aligned(z, 8) && aligned(bias, bias_dtype == PT_F32 ? 16 : 8);
    const int64_t tiles = ceil_div(N, kFrFeat), grid_y = ceil_div(M, plan.block);
    r.split = plan.split;
    return fr_dispatch<FR_LINEAR>(tw, tx, r, tok, tiles, grid_y, st);
}

}  // namespace ptb

using namespace ptb;

extern "C" {

size_t pt_moe_few_tokens_scratch_bytes(int64_t T, int top_k, int64_t I) {
    if (T <= 0 || top_k <= 0 || I <= 0) return 0;
    return (size_t) (T * top_k * I * 2);
}

int pt_moe_few_tokens(const void *x, const void *gate_up, const void *down, int dtype, const void *ids, int id_bytes, const float *probs, int64_t T,
                      int E, int top_k, int64_t H, int64_t I, int act, void *scratch, size_t scratch_bytes, void *out, int *status, void *stream) {
    PT_REQUIRE(dtype == PT_BF16 || dtype == PT_F16, "moe_few_tokens: bf16 or fp16 tensors");
    PT_REQUIRE(act == PT_ACT_SILU || act == PT_ACT_GELU, "moe_few_tokens: bad activation");
    PT_REQUIRE(id_bytes == 4 || id_bytes == 8, "moe_few_tokens: expert indices must be int32 or int64");
    PT_REQUIRE(T >= 0 && T <= PT_MOE_FEW_TOKENS_MAX && E >= 1 && E <= kMaxGroups, "moe_few_tokens: takes at most %d tokens and %d experts (got %lld, %d)",
               PT_MOE_FEW_TOKENS_MAX, kMaxGroups, (long long) T, E);
    PT_REQUIRE(top_k >= 1 && top_k <= kFrMaxTopK && T * top_k <= kFrMaxSlots, "moe_few_tokens: takes at most %d experts per token and %d slots",
               kFrMaxTopK, kFrMaxSlots);
    PT_REQUIRE(H >= 8 && I >= 8 && H % 8 == 0 && I % 8 == 0, "moe_few_tokens: hidden and expert width must be multiples of 8 (got %lld, %lld)",
               (long long) H, (long long) I);
    PT_REQUIRE(H < (1 << 24) && I < (1 << 24) && 2 * I * E < (1ll << 31) && H * E < (1ll << 31) && (int64_t) E * ceil_div(I, 64) < (1ll << 31),
               "moe_few_tokens: extent exceeds 32-bit tile coordinates");
    if (T == 0) return PT_OK;
    PT_REQUIRE(x && gate_up && down && ids && probs && scratch && out, "moe_few_tokens: null pointer");
    PT_REQUIRE(scratch_bytes >= pt_moe_few_tokens_scratch_bytes(T, top_k, I) && aligned(scratch, 16), "moe_few_tokens: scratch too small or unaligned");
    PT_REQUIRE(aligned(x, 16) && aligned(gate_up, 16) && aligned(down, 16) && aligned(out, 8),
               "moe_few_tokens: x and the weights must start on 16-byte boundaries, out on an 8-byte one");
    cudaStream_t st = (cudaStream_t) stream;
    const int tok = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
    const int64_t slots = T * top_k, most = std::min<int64_t>(E, slots);   // experts that can be chosen
    CUtensorMap t_gate_up, t_down;
    int rc;
    if ((rc = make_tmap_bytes(&t_gate_up, gate_up, (int64_t) E * 2 * I, 2 * H, 2 * H, 64)) != PT_OK) return rc;
    if ((rc = make_tmap_bytes(&t_down, down, (int64_t) E * H, 2 * I, 2 * I, kFrFeat)) != PT_OK) return rc;
    FewRowsArgs a{};
    a.rows = (int) T; a.fmt = dtype == PT_BF16 ? 1 : 0; a.act = act; a.ids = ids; a.id_bytes = id_bytes; a.top_k = top_k; a.experts = E;
    a.probs = probs; a.status = status; a.out_dtype = dtype;
    a.n = (int) I; a.k = (int) H; a.out = scratch; a.x = x; a.x_pitch = 2 * H;
    int64_t tiles = ceil_div(I, 64);
    a.split = fr_split_experts(tok, tiles * most, ceil_div(H, 64));
    if ((rc = fr_dispatch<FR_GATE_UP>(t_gate_up, t_gate_up, a, tok, tiles, most, st)) != PT_OK) return rc;
    a.n = (int) H; a.k = (int) I; a.out = out; a.x = scratch; a.x_pitch = 2 * I;
    tiles = ceil_div(H, kFrFeat);
    a.split = fr_split_experts(tok, tiles, most * ceil_div(I, 64));
    return fr_dispatch<FR_DOWN>(t_down, t_down, a, tok, tiles, 1, st);
}

}  // extern "C"
