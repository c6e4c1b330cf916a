// Products with few rows: one to some hundred tokens through a weight matrix, dense (bias, activation and residual in the
// epilogue) or through the chosen experts of a mixture (gate and up projection with the gated activation; down projection with
// the weighted sum).
//
// Bound: the bytes of the weights, each read once.  The weight is therefore the 128-row operand of tcgen05.mma and the tokens are
// its narrow one (N = 16 .. 128), so that a CTA streams 16 KiB weight blocks [128 features][64 of K] through a TMA ring and the
// tensor core takes each of them in four instructions, far faster than it arrives.  About 100 KiB of weights are on their way per
// CTA, two CTAs to an SM, which covers the memory latency (148 SMs x 200 KiB = 29 MiB in flight) and lets one CTA's start and
// write-out hide behind the other's stream.
//   The contraction is split over the CTAs of a cluster when the features alone would leave SMs idle: every CTA puts its partial
// [tokens][128] block of fp32 sums into its own shared memory and the CTAs add each other's blocks for their share of the tokens
// through distributed shared memory, in the order of their ranks.  So there is no workspace, no counter and no atomic: results do
// not depend on timing, and calls on different streams or in different graphs share nothing.
//
//   warp 0      producer (TMA; for experts also the lists of the tokens that chose them)
//   warp 1      one thread issues the MMAs; owns the tensor memory
//   warps 2-5   tensor memory -> shared memory; then all warps reduce and write out
//
// Mixture, two kernels:
//   GATE_UP  grid (blocks of 64 features x split, chosen experts): the block is 64 gate rows and the 64 up rows that belong to them.
//            Rows of x are gathered by TMA (tile::gather4) from the list of the expert's tokens.  Writes p * act(g) * u, with p
//            the slot's probability (the sum of them where a token names an expert twice), rounded once to the tensors' type: the
//            next product's operand type.
//   DOWN     a CTA keeps one [128 features][tokens] accumulator over ALL chosen experts, one column per token, so the weighted
//            sum over a token's experts happens in tensor memory.  For every expert only the 16-token blocks that hold one of
//            its tokens are multiplied; the other tokens of such a block read a row of zeros.  Its first weight blocks are
//            fetched before the first kernel has finished (programmatic dependent launch): weights and routing do not depend
//            on it.
#include <algorithm>

#include "act_math.cuh"
#include "common.cuh"
#include "gemm_common.cuh"
#include "sm100_ptx.cuh"

namespace ptb {
using namespace sm100;

constexpr int kFrThreads = 192;
constexpr int kFrFeat = 128;              // features (weight rows) of a CTA
constexpr int kFrABytes = kFrFeat * 128;  // a weight block: 128 rows of 64 16-bit elements
constexpr int kFrMaxSlots = 2048;         // tokens x experts per token
constexpr int kFrMaxTopK = 32;
constexpr int kFrMaxSplit = 8;            // CTAs of a cluster

enum FewRowsKind { FR_LINEAR = 0, FR_GATE_UP = 1, FR_DOWN = 2 };

struct FewRowsArgs {
    int rows;                // LINEAR: M; else tokens
    int n, k;                // features of the output (GATE_UP: of one half), contraction length
    int split;               // CTAs of a cluster
    int fmt;                 // 0 = fp16, 1 = bf16 operands
    void *out;               // LINEAR / DOWN [rows, n]; GATE_UP [slots + 1, n], the last row zeros
    int out_dtype;
    int act;
    // LINEAR
    int w_mn;                // the weight is stored [k, n]: two boxes of 64 features x 64 contraction rows, read in place
    const void *bias, *residual;
    int bias_dtype;
    void *z;                 // pre-activation in the operands' type, or null
    int vec_ok;              // rows of out / residual / z / bias take four elements at a time
    // mixture
    const void *ids;         // [tokens, top_k] int32 / int64
    int id_bytes, top_k, experts;
    const float *probs;
    int *status;
};

template <int TOK> struct FrCfg {
    static constexpr int kBBytes = TOK * 128;
    static constexpr int kStageBytes = kFrABytes + kBBytes;
    static constexpr int kStages = TOK <= 16 ? 6 : TOK <= 32 ? 5 : TOK <= 64 ? 4 : 3;   // two CTAs per SM
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kIdSlots = TOK * kFrMaxTopK < kFrMaxSlots ? TOK * kFrMaxTopK : kFrMaxSlots;
    static constexpr int kSmem = kRing + 1024 /* alignment */ + 2 * kIdSlots;
    static constexpr int kTmemCols = TOK < 32 ? 32 : TOK;
    static_assert(TOK * kFrFeat * 4 <= kRing, "the partial block must fit the ring");
    static_assert(2 * (kSmem + 3584 /* static and reserved */) <= 228 * 1024, "two CTAs per SM");
};

template <int TOK, int KIND>
__global__ void __launch_bounds__(kFrThreads, 2)
    few_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, FewRowsArgs a) {
    using Cfg = FrCfg<TOK>;
    constexpr int kStages = Cfg::kStages;
    constexpr bool kMoe = KIND != FR_LINEAR;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    int16_t *s_ids = reinterpret_cast<int16_t *>(ring + Cfg::kRing);   // [tokens * top_k], -1: no expert of this call
    __shared__ uint64_t full_bar[kStages], empty_bar[kStages], done_bar;
    __shared__ uint32_t s_tmem, s_mask[kStages], s_touched;   // s_mask: DOWN, which 16-token blocks a stage holds
    __shared__ int s_abort, s_count;
    __shared__ uint32_t s_bits[kMoe ? 32 : 1];
    __shared__ int16_t s_active[KIND == FR_DOWN ? kMaxGroups : 1];
    __shared__ int s_row[kMoe ? TOK : 1], s_slot[KIND == FR_GATE_UP ? TOK : 1];
    __shared__ float s_prob[KIND == FR_GATE_UP ? TOK : 1];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = a.split > 1 ? (int) cluster_ctarank() : 0;
    const int tile = (int) blockIdx.x / a.split;
    const int T = a.rows;

    if (threadIdx.x == 0) {
        s_abort = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        mbar_init(&done_bar, 2);   // the MMA thread's own arrival (publishes s_touched) and its commit
        fence_barrier_init();
        prefetch_tmap(&tmap_w);
        prefetch_tmap(&tmap_x);
    }
    if (warp == 1) {
        tmem_alloc(&s_tmem, Cfg::kTmemCols);
        tmem_relinquish();
    }
    if (KIND != FR_DOWN) {   // DOWN waits later: what it reads up to there is not written by the kernel before it
        grid_dep_wait();
        grid_dep_launch();
    }

    // ---- routing: which experts are chosen, and by whom
    int cnt = KIND == FR_LINEAR ? min(TOK, T - (int) blockIdx.y * TOK) : 0;   // rows of this CTA
    int expert = 0, n_active = 0;
    if constexpr (kMoe) {
        if (threadIdx.x < 32) s_bits[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < T * a.top_k; i += kFrThreads) {
            const int64_t id = a.id_bytes == 8 ? reinterpret_cast<const int64_t *>(a.ids)[i] : (int64_t) reinterpret_cast<const int *>(a.ids)[i];
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
                __syncwarp();
                if (lane < 3 && base + lane < TOK && (base + lane) / 4 == (base - 1) / 4) s_row[base + lane] = s_row[0];   // fill the last group of four
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
    __syncthreads();
    tc_fence_after_sync();
    if constexpr (KIND == FR_GATE_UP) cnt = s_count;
    if constexpr (KIND == FR_DOWN) cnt = T;

    // ---- this CTA's share of the contraction
    const int chunks = (a.k + 63) / 64;   // per expert
    const int64_t total = KIND == FR_DOWN ? (int64_t) n_active * chunks : chunks;
    const int l0 = (int) (total * rank / a.split), l1 = (int) (total * (rank + 1) / a.split);
    const uint32_t tmem = s_tmem;
    volatile int *abort_flag = &s_abort;
    bool ok = true;

    if (warp == 0) {
        // ================================================================ producer
        const uint64_t stream_pol = l2_policy_evict_first(), keep_pol = l2_policy_evict_last();
        if constexpr (KIND != FR_DOWN) {
            if (elect_one()) {
                const int groups = (cnt + 3) / 4;
                const uint32_t bytes = kFrABytes + (KIND == FR_LINEAR ? Cfg::kBBytes : groups * 512);
                uint32_t stage = 0, phase = 0;
                for (int l = l0; l < l1; ++l) {
                    if (!(ok = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag))) break;
                    uint8_t *A = ring + stage * Cfg::kStageBytes, *B = A + kFrABytes;
                    mbar_arrive_expect_tx(&full_bar[stage], bytes);
                    if constexpr (KIND == FR_LINEAR) {
                        if (a.w_mn) {
                            tma_load_2d_hint(A, &tmap_w, &full_bar[stage], tile * kFrFeat * 2, l * 64, stream_pol);
                            tma_load_2d_hint(A + kFrABytes / 2, &tmap_w, &full_bar[stage], tile * kFrFeat * 2 + 128, l * 64, stream_pol);
                        } else {
                            tma_load_2d_hint(A, &tmap_w, &full_bar[stage], l * 128, tile * kFrFeat, stream_pol);
                        }
                        tma_load_2d_hint(B, &tmap_x, &full_bar[stage], l * 128, (int) blockIdx.y * TOK, keep_pol);
                    } else {
                        const int row = expert * 2 * a.n + tile * 64;
                        tma_load_2d_hint(A, &tmap_w, &full_bar[stage], l * 128, row, stream_pol);
                        tma_load_2d_hint(A + kFrABytes / 2, &tmap_w, &full_bar[stage], l * 128, row + a.n, stream_pol);
                        for (int g = 0; g < groups; ++g)
                            tma_gather4(B + g * 512, &tmap_x, &full_bar[stage], l * 128, s_row[4 * g], s_row[4 * g + 1], s_row[4 * g + 2], s_row[4 * g + 3], keep_pol);
                    }
                    if (++stage == kStages) { stage = 0; phase ^= 1; }
                }
            }
        } else {
            // rows of the activations of every token for the expert at hand (the row of zeros for the others), in s_row
            int cur = -1;
            uint32_t mask = 0;
            auto set_expert = [&](int ai) {
                if (ai == cur) return;
                cur = ai;
                const int e = s_active[ai];
                mask = 0;
                __syncwarp();
                for (int t0 = 0; t0 < TOK; t0 += 32) {
                    const int t = t0 + lane;
                    int row = T * a.top_k;
                    if (t < T)
                        for (int j = a.top_k - 1; j >= 0; --j)
                            if (s_ids[t * a.top_k + j] == e) row = t * a.top_k + j;   // the first of them
                    const uint32_t has = __ballot_sync(0xffffffffu, row != T * a.top_k);
                    if (t < TOK) s_row[t] = row;
                    mask |= (uint32_t) ((has & 0xFFFFu) != 0) << (t0 / 16) | (uint32_t) ((has >> 16) != 0) << (t0 / 16 + 1);
                }
                __syncwarp();
            };
            auto load_w = [&](int l, uint32_t stage) {
                s_mask[stage] = mask;
                mbar_arrive_expect_tx(&full_bar[stage], kFrABytes + __popc(mask) * 2048);
                tma_load_2d_hint(ring + stage * Cfg::kStageBytes, &tmap_w, &full_bar[stage], (l % chunks) * 128, s_active[cur] * a.n + tile * kFrFeat, stream_pol);
            };
            auto load_x = [&](int l, uint32_t stage) {
                uint8_t *B = ring + stage * Cfg::kStageBytes + kFrABytes;
                for (uint32_t m = mask; m != 0; m &= m - 1) {
                    const int blk = __ffs(m) - 1;
#pragma unroll
                    for (int g = 4 * blk; g < 4 * blk + 4; ++g)
                        tma_gather4(B + g * 512, &tmap_x, &full_bar[stage], (l % chunks) * 128, s_row[4 * g], s_row[4 * g + 1], s_row[4 * g + 2], s_row[4 * g + 3], keep_pol);
                }
            };
            const int pre = min(kStages, l1 - l0);   // the ring is empty: these stages need no wait
            for (int i = 0; i < pre; ++i) {
                set_expert((l0 + i) / chunks);
                if (lane == 0) load_w(l0 + i, i);
            }
            grid_dep_wait();
            for (int i = 0; i < pre; ++i) {
                set_expert((l0 + i) / chunks);
                if (lane == 0) load_x(l0 + i, i);
            }
            uint32_t stage = pre == kStages ? 0 : pre, phase = pre == kStages ? 1 : 0;
            for (int l = l0 + pre; l < l1; ++l) {
                set_expert(l / chunks);
                int good = 1;
                if (lane == 0) {
                    good = mbar_wait(&empty_bar[stage], phase ^ 1, abort_flag);
                    if (good) {
                        load_w(l, stage);
                        load_x(l, stage);
                    }
                }
                if (!(ok = __shfl_sync(0xffffffffu, good, 0) != 0)) break;
                if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
        }
    } else if (warp == 1) {
        // ================================================================ MMA issuer
        if (elect_one()) {
            const bool w_mn = KIND == FR_LINEAR && a.w_mn;
            const uint32_t idesc0 = idesc_f8(a.fmt, a.fmt, kFrFeat, 0) | ((uint32_t) w_mn << 15);
            const uint64_t w_step = w_mn ? (16 * 128) >> 4 : 32 >> 4;   // 16 contraction rows, or 32 bytes along a row
            uint32_t touched = 0;   // 16-token blocks that hold sums
            const uint32_t all = (1u << ((cnt + 15) / 16)) - 1;
            uint32_t stage = 0, phase = 0;
            for (int l = l0; l < l1; ++l) {
                if (!(ok = mbar_wait(&full_bar[stage], phase, abort_flag))) break;
                tc_fence_after_sync();
                const uint32_t A = smem_u32(ring + stage * Cfg::kStageBytes);
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
                    for (int k = 0; k < 4; ++k)
                        mma_f16(tmem + 16 * b0, a_desc + k * w_step, b_desc + 2 * k, idesc, acc0 | (uint32_t) (k > 0));
                    m &= ~(((1u << len) - 1) << b0);
                }
                touched |= used;
                tc_commit(&empty_bar[stage]);
                if (++stage == kStages) { stage = 0; phase ^= 1; }
            }
            if (ok) {
                s_touched = touched;
                mbar_arrive(&done_bar);
                tc_commit(&done_bar);
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
        const uint32_t touched = ok ? s_touched : 0;
        for (int b = 0; b < blocks; ++b) {
            uint32_t r[16];
            if (touched >> b & 1) {
                tmem_ld16(tmem + ((uint32_t) (q * 32) << 16) + 16 * b, r);
                tmem_ld_wait();
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) r[i] = 0u;
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) part[(16 * b + i) * kFrFeat + q * 32 + lane] = __uint_as_float(r[i]);
        }
    }
    if (!ok || s_abort) {
        if (a.status != nullptr && lane == 0) *reinterpret_cast<volatile int *>(a.status) = PT_ERR_TIMEOUT;
        __nanosleep(200000);   // let copies in flight land before the shared memory is released
    }
    tc_fence_before_sync();
    __syncwarp();
    if (a.split > 1) cluster_sync_all();
    else __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, Cfg::kTmemCols);
    }
    if constexpr (KIND == FR_DOWN) grid_dep_wait();

    // ================================================================ sum over the cluster, epilogue, write-out
    // a warp takes one token at a time, a lane four neighbouring features
    if constexpr (KIND == FR_GATE_UP) {
        if (blockIdx.y == 0 && rank == 0 && warp == 0) {   // the row of zeros that DOWN reads for tokens of other experts
            const int f = tile * 64 + 2 * lane;
            if (f < a.n) *reinterpret_cast<uint32_t *>(reinterpret_cast<uint16_t *>(a.out) + (int64_t) T * a.top_k * a.n + f) = 0u;
        }
    }
    const uint32_t part_addr = smem_u32(part);
    for (int t = rank + a.split * warp; t < cnt; t += a.split * (kFrThreads / 32)) {
        float vv[1][4] = {{0.f, 0.f, 0.f, 0.f}};
        float(&v)[4] = vv[0];
        // GATE_UP: features 2 lane, 2 lane + 1 of the gate half and of the up half
        constexpr uint32_t kSecond = KIND == FR_GATE_UP ? 256 : 8;
        const uint32_t at = part_addr + (uint32_t) t * (kFrFeat * 4) + lane * (KIND == FR_GATE_UP ? 8 : 16);
        if (a.split == 1) {
            ld_cluster_f32x2(at, false, v[0], v[1]);
            ld_cluster_f32x2(at + kSecond, false, v[2], v[3]);
        } else {
            float w[kFrMaxSplit][4];   // all loads on their way before the first addition: one remote round trip, not one per CTA
#pragma unroll
            for (int s = 0; s < kFrMaxSplit; ++s) {
                if (s >= a.split) continue;
                const uint32_t src = map_addr_to_rank(at, s);
                ld_cluster_f32x2(src, true, w[s][0], w[s][1]);
                ld_cluster_f32x2(src + kSecond, true, w[s][2], w[s][3]);
            }
#pragma unroll
            for (int s = 0; s < kFrMaxSplit; ++s)
                if (s < a.split) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[i] += w[s][i];
                }
        }
        if constexpr (KIND == FR_GATE_UP) {
            const int f = tile * 64 + 2 * lane;
            const float p = s_prob[t];
            const float h0 = act_any(a.act, v[0]) * v[2] * p, h1 = act_any(a.act, v[1]) * v[3] * p;
            if (f < a.n)
                *reinterpret_cast<uint32_t *>(reinterpret_cast<uint16_t *>(a.out) + (int64_t) s_slot[t] * a.n + f) =
                    a.fmt ? pack2<__nv_bfloat16>(h0, h1) : pack2<__half>(h0, h1);
        } else {
            const int f = tile * kFrFeat + 4 * lane;
            const int64_t row = KIND == FR_LINEAR ? (int64_t) blockIdx.y * TOK + t : t;
            const int64_t o = row * a.n + f;
            if constexpr (KIND == FR_LINEAR) {
                const int zt = a.fmt ? PT_BF16 : PT_F16;
                if (a.vec_ok && f < a.n) {
                    float x[4];
                    if (a.bias != nullptr) {
                        load4_as_f32(a.bias, a.bias_dtype, f, x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] += x[i];
                    }
                    if (a.z != nullptr) store4_from_f32(a.z, zt, o, v);
                    act_any_all<1>(a.act, vv);
                    if (a.residual != nullptr) {
                        load4_as_f32(a.residual, a.out_dtype, o, x);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] += x[i];
                    }
                    store4_from_f32(a.out, a.out_dtype, o, v);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (f + i >= a.n) continue;
                        if (a.bias != nullptr) v[i] += load_as_f32(a.bias, a.bias_dtype, f + i);
                        if (a.z != nullptr) store_from_f32(a.z, zt, o + i, v[i]);
                        v[i] = act_any(a.act, v[i]);
                        if (a.residual != nullptr) v[i] += load_as_f32(a.residual, a.out_dtype, o + i);
                        store_from_f32(a.out, a.out_dtype, o + i, v[i]);
                    }
                }
            } else {
                if (f < a.n) store4_from_f32(a.out, a.out_dtype, o, v);
            }
        }
    }
    if (a.split > 1) {
        __syncwarp();
        cluster_sync_all();   // no CTA leaves while another still reads its block
    }
}

// ------------------------------------------------------------------------------------------------ host side
template <int TOK, int KIND>
static int fr_launch(const CUtensorMap &tw, const CUtensorMap &tx, const FewRowsArgs &a, int64_t tiles, int64_t grid_y, cudaStream_t st) {
    using Cfg = FrCfg<TOK>;
    auto kern = few_rows_kernel<TOK, KIND>;
    static bool attr_set[64] = {};   // per instantiation and device
    const int dev = current_device_slot();
    if (!attr_set[dev]) {
        PT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmem));
        attr_set[dev] = true;
    }
    PT_REQUIRE(tiles * a.split < (1ll << 31) && grid_y < 65536, "few-row product: grid too large");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (tiles * a.split), (unsigned) grid_y);
    cfg.blockDim = dim3(kFrThreads);
    cfg.dynamicSmemBytes = Cfg::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned) a.split; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.split > 1 ? 2 : 1;
    PT_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, tw, tx, a));
    return PT_OK;
}

// CTAs per cluster: double while the grid would still be resident at once (two CTAs per SM) and each CTA keeps a ring's worth of
// blocks.
static int fr_split(int64_t tiles, int64_t chunks) {
    int s = 1;
    while (s < kFrMaxSplit && tiles * s * 2 <= 2 * (int64_t) sm_count() && chunks / (s * 2) >= 4) s *= 2;
    return s;
}

template <int KIND>
static int fr_dispatch(const CUtensorMap &tw, const CUtensorMap &tx, const FewRowsArgs &a, int tok, int64_t tiles, int64_t grid_y, cudaStream_t st) {
    switch (tok) {
    case 16: return fr_launch<16, KIND>(tw, tx, a, tiles, grid_y, st);
    case 32: return fr_launch<32, KIND>(tw, tx, a, tiles, grid_y, st);
    case 64: return fr_launch<64, KIND>(tw, tx, a, tiles, grid_y, st);
    default: return fr_launch<128, KIND>(tw, tx, a, tiles, grid_y, st);
    }
}
static int fr_tokens(int64_t rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128; }

// y = act(a . b^T + bias) + residual for few rows of a
int few_rows_linear(const void *a, const void *b, int b_mn, int ab_dtype, const void *bias, int bias_dtype, const void *residual, void *c, int c_dtype,
                    void *z, int act, int64_t M, int64_t N, int64_t K, int *status, cudaStream_t st) {
    const int tok = fr_tokens(M);
    CUtensorMap tw, tx;
    int rc;
    if ((rc = b_mn ? make_tmap_bytes(&tw, b, K, 2 * N, 2 * N, 64) : make_tmap_bytes(&tw, b, N, 2 * K, 2 * K, kFrFeat)) != PT_OK) return rc;
    if ((rc = make_tmap_bytes(&tx, a, M, 2 * K, 2 * K, tok)) != PT_OK) return rc;
    FewRowsArgs r{};
    r.w_mn = b_mn; r.rows = (int) M; r.n = (int) N; r.k = (int) K; r.fmt = ab_dtype == PT_BF16 ? 1 : 0;
    r.out = c; r.out_dtype = c_dtype; r.act = act; r.bias = bias; r.bias_dtype = bias_dtype; r.residual = residual; r.z = z; r.status = status;
    const int esize = c_dtype == PT_F32 ? 4 : 2;
    r.vec_ok = N % 4 == 0 && aligned(c, 4 * esize) && aligned(residual, 4 * esize) && aligned(z, 8) && aligned(bias, bias_dtype == PT_F32 ? 16 : 8);
    const int64_t tiles = ceil_div(N, kFrFeat), grid_y = ceil_div(M, tok);
    r.split = fr_split(tiles * grid_y, ceil_div(K, 64));
    return fr_dispatch<FR_LINEAR>(tw, tx, r, tok, tiles, grid_y, st);
}

}  // namespace ptb

using namespace ptb;

extern "C" {

size_t pt_moe_few_tokens_scratch_bytes(int64_t T, int top_k, int64_t I) {
    if (T <= 0 || top_k <= 0 || I <= 0) return 0;
    return (size_t) ((T * top_k + 1) * I * 2);
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
    PT_REQUIRE(aligned(out, 8), "moe_few_tokens: out must be 8-byte aligned");
    cudaStream_t st = (cudaStream_t) stream;
    const int tok = fr_tokens(T);
    const int64_t slots = T * top_k, most = std::min<int64_t>(E, slots);   // experts that can be chosen
    CUtensorMap tw, tx;
    int rc;
    FewRowsArgs a{};
    a.rows = (int) T; a.fmt = dtype == PT_BF16 ? 1 : 0; a.act = act; a.ids = ids; a.id_bytes = id_bytes; a.top_k = top_k; a.experts = E;
    a.probs = probs; a.status = status; a.out_dtype = dtype;
    if ((rc = make_tmap_bytes(&tw, gate_up, (int64_t) E * 2 * I, 2 * H, 2 * H, 64)) != PT_OK) return rc;
    if ((rc = make_tmap_bytes(&tx, x, T, 2 * H, 2 * H, 1)) != PT_OK) return rc;
    a.n = (int) I; a.k = (int) H; a.out = scratch;
    int64_t tiles = ceil_div(I, 64);
    a.split = fr_split(tiles * most, ceil_div(H, 64));
    if ((rc = fr_dispatch<FR_GATE_UP>(tw, tx, a, tok, tiles, most, st)) != PT_OK) return rc;
    if ((rc = make_tmap_bytes(&tw, down, (int64_t) E * H, 2 * I, 2 * I, kFrFeat)) != PT_OK) return rc;
    if ((rc = make_tmap_bytes(&tx, scratch, slots + 1, 2 * I, 2 * I, 1)) != PT_OK) return rc;
    a.n = (int) H; a.k = (int) I; a.out = out;
    tiles = ceil_div(H, kFrFeat);
    a.split = fr_split(tiles, std::min<int64_t>(most, T) * ceil_div(I, 64));
    return fr_dispatch<FR_DOWN>(tw, tx, a, tok, tiles, 1, st);
}

}  // extern "C"
