// Products of row groups with one int8 weight per group (the experts' linear layers), for sm_100a:
//   out[p, n] = bf16( fp32(sum_k X[src(p), k] * W[e, n, k]) * (sx[src(p)] * sw[e, n]) )    for offsets[e] <= p < offsets[e + 1]
// and, with SWIGLU, for a weight of 2 N rows (N gate rows, then N up rows) per expert:
//   out[p, n] = bf16( g / (1 + exp(-g)) * u ),  g, u = the fp32 values of channels n and N + n
// src(p) is p, or the token slots[p] / top_k.  Rows of no expert are written as zeros.  How many rows an expert has is known on the
// device alone, so every CTA works the list of tiles out of the offsets by itself.
//
// Operands are swapped: the 128 rows of a WEIGHT tile fill the M = 128 side of tcgen05.mma and the expert's rows are the N side,
// whose extent is an operand of the instruction: a tile of r rows costs roundup(r, 16) columns instead of a multiple of 128, which
// is what makes ragged groups and single tokens cheap.  An expert's rows are cut into equal tiles of at most BT.
//
// Structure (persistent CTAs, one per SM, two of 64-token tiles; 192 threads, 320 with GATHER), as in the dense kernel:
//   warp 0      TMA producer: weight tiles (128 rows x 128 bytes) and token rows, either with one instruction
//   warp 1      MMA issuer, kind::i8, two accumulators in tensor memory
//   next 4      epilogue: accumulators come as pairs of tokens of a channel, are scaled in packed arithmetic, and turned by stmatrix into runs of
//               channels of a token, which leave 16 bytes a lane.  (With a channel per lane and 2-byte stores, three times the
//               instructions, 32768 x 4096 x 2048 took 241 us for 235, SwiGLU 4096 x 4096 491 for 472.)
//   last 4      (GATHER) token rows from wherever they lie, by 16-byte asynchronous copies into the places where TMA's 128-byte swizzle
//               would put them: eight lanes a row, a whole line per row; their arrivals follow the copies by themselves, and the issuer
//               makes them visible to the tensor core behind its wait.  SwiGLU of 4096 tokens to 8 of 64 experts, 4096 x 4096, took
//               472 us for 454 with loader warps that wait for their copies, two stages behind those they issue.  TMA's own gather,
//               four rows an instruction, delivers a row in 14 cycles: 32768 rows gathered for 4096 x 4096 that way took 2010 us, put
//               in order by a pass in front 475, rows that lie in order 446.
// SWIGLU: a weight tile is 64 gate rows and their 64 up rows in alternating runs of 16, so that gate and up of a channel lie 16 lanes of tensor
// memory apart and come to the same thread.
#pragma once

#include "../k_dense.cuh"
#include "../k_quant.cuh"

namespace gi8 {

constexpr int kExpertsEpilogueThreads = 128;  // (eight warps instead of four: level with SwiGLU's exponentials, slower without)
constexpr int kExpertsLoaderWarps = 4;
constexpr int experts_threads(bool gather) { return 64 + kExpertsEpilogueThreads + (gather ? 32 * kExpertsLoaderWarps : 0); }
constexpr int kExpertsMaxExperts = 1024;
// Tokens at a time, and shared memory behind the stages: per epilogue warp 32 channels (SwiGLU: 16) of so many tokens, bf16.
__host__ __device__ constexpr int experts_chunk(bool pair) { return pair ? 32 : 16; }
__host__ __device__ constexpr int experts_turn_bytes(bool swiglu, bool pair) { return experts_chunk(pair) * (swiglu ? 32 * 4 : 64 * 4); }

struct ExpertsParams {
    const int8_t* x;         // int8 [tokens, K]
    uint16_t* out;           // bf16 [rows, N]
    const float* sx;         // [rows of x]
    const float* sw;         // [E, Nw]
    const int32_t* offsets;  // [E + 1]
    const int32_t* slots;    // [rows], or null: row p reads x[p]
    uint32_t* status;
    int64_t rows;            // S
    int tokens;              // rows of x
    int E, N, K;             // N: columns of out; Nw = N or 2 N rows of weight per expert
    int top_k;
    int band;                // token tiles of a band
    int vec;                 // rows of out are whole 16-byte pieces
    int interleave;          // SWIGLU: the weight's map is over runs of 16 rows and loads a whole tile (N a multiple of 16)
    int early;               // the kernel in front writes neither weights nor offsets: the first weights are requested while it runs
    int weight_policy_first; // weights are met once or twice: keep them from displacing the rest of L2
};

// g / (1 + exp(-g)), by the exponential that does not overflow: far below zero the result fades out through the subnormals.  The fast
// exponential is off by 2 + 1.173 |g| units in the last place, the reciprocal by one (its argument lies in [1, 2]): next to nothing to a
// result that is rounded to 8 bits.
GI8_DEVICE float silu(float g)
{
    const float t = __expf(-fabsf(g));
    return g * ((g < 0.0f ? t : 1.0f) * approx_reciprocal(1.0f + t));
}

GI8_DEVICE uint4 ld_shared_v4(uint32_t addr)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}

// Tensor maps of the token rows, with boxes of a quarter, half, three quarters and all of a token tile: a tile's rows are loaded by one
// instruction whatever their number.
struct TokenMaps {
    CUtensorMap m[4];
};

// One tile of the list.
struct ExpertTile {
    int expert, weight_tile;
    int row0, rows;  // of out
};

// What the tiles are worked out from, in shared memory: start[e] = clamped offsets, tiles_end[e] = token tiles of experts 0 .. e.
template <int BT>
struct ExpertList {
    int32_t start[kExpertsMaxExperts + 1];
    int32_t tiles_end[kExpertsMaxExperts];
    int32_t chunk_tiles[kExpertsMaxExperts / 32];
};

// Whole CTA.  Offsets that are no ascending sequence within [0, rows] give wrong rows, never an access out of bounds.
template <int BT>
GI8_DEVICE void build_expert_list(ExpertList<BT>& list, const int32_t* offsets, int E, int64_t rows)
{
    for (int e = threadIdx.x; e <= E; e += blockDim.x)
        list.start[e] = static_cast<int32_t>(min(max(static_cast<int64_t>(__ldg(offsets + e)), static_cast<int64_t>(0)), rows));
    __syncthreads();
    // sums within chunks of 32 experts, a warp each, then what lies in front of a chunk
    const int lane = threadIdx.x & 31, warps = blockDim.x / 32, chunks = (E + 31) / 32;
    for (int c = threadIdx.x >> 5; c < chunks; c += warps) {
        const int e = c * 32 + lane;
        int n = e < E ? max(0, list.start[e + 1] - list.start[e]) : 0;
        n = (n + BT - 1) / BT;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) n += v;
        }
        if (e < E) list.tiles_end[e] = n;
        if (lane == 31) list.chunk_tiles[c] = n;
    }
    __syncthreads();
    if (chunks == 1) return;
    for (int c = threadIdx.x >> 5; c < chunks; c += warps) {
        const int before = __reduce_add_sync(0xffffffffu, lane < c ? list.chunk_tiles[lane] : 0);
        if (c * 32 + lane < E) list.tiles_end[c * 32 + lane] += before;
    }
    __syncthreads();
}

// Tile `item` of the list, if there is one: experts in order, within an expert bands of `band` token tiles, whose rows stay in L2 while the
// band goes through the weights, within a band weight tile by weight tile with the token tiles inside, so that CTAs that run at the same
// time share weights.  Whole warp: the chunk of 32 experts that the tile lies in, then the expert.
template <int BT, int ALIGN>
GI8_DEVICE bool find_expert_tile(const ExpertList<BT>& list, int E, int weight_tiles, int band, int64_t item, ExpertTile& t)
{
    const int lane = threadIdx.x & 31;
    auto past = [&](int e) { return e < E && static_cast<int64_t>(list.tiles_end[e]) * weight_tiles > item; };
    int chunk = 0;
    if (E > 32) {
        const uint32_t hit = __ballot_sync(0xffffffffu, lane * 32 < E && past(min(lane * 32 + 31, E - 1)));
        if (!hit) return false;
        chunk = __ffs(hit) - 1;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, past(chunk * 32 + lane));
    if (!hit) return false;
    t.expert = chunk * 32 + __ffs(hit) - 1;
    const int before = t.expert ? list.tiles_end[t.expert - 1] : 0;
    const int tiles = list.tiles_end[t.expert] - before;
    const int r = static_cast<int>(item - static_cast<int64_t>(before) * weight_tiles);
    const int band0 = r / (band * weight_tiles) * band;  // first token tile of its band
    const int in_band = r - band0 * weight_tiles, wide = min(band, tiles - band0);
    t.weight_tile = in_band / wide;
    const int n = list.start[t.expert + 1] - list.start[t.expert];
    const int per = ((n + tiles - 1) / tiles + ALIGN - 1) & ~(ALIGN - 1);  // <= BT, and the last tile keeps at least a row
    const int first = (band0 + in_band - t.weight_tile * wide) * per;
    t.row0 = list.start[t.expert] + first;
    t.rows = min(per, n - first);
    return true;
}

// Tile loads whose bytes are counted on the barrier at cluster address `bar` (the leader's) or on one of this CTA.
template <bool PAIR>
GI8_DEVICE void load_tile_2d(void* dst, const CUtensorMap* map, uint32_t bar, int32_t c0, int32_t c1, uint64_t policy)
{
    if constexpr (PAIR) tma_load_2d_pair_hint(dst, map, bar, c0, c1, policy);
    else tma_load_2d_hint_addr(dst, map, bar, c0, c1, policy);
}
template <bool PAIR>
GI8_DEVICE void load_tile_5d(void* dst, const CUtensorMap* map, uint32_t bar, int32_t c0, int32_t c1, int32_t c2, int32_t c3, int32_t c4, uint64_t policy)
{
    if constexpr (PAIR) tma_load_5d_pair_hint(dst, map, bar, c0, c1, c2, c3, c4, policy);
    else tma_load_5d_hint(dst, map, bar, c0, c1, c2, c3, c4, policy);
}

// PAIR: two CTAs on neighbouring SMs share a tile of 2 x 128 weight rows, as in the dense kernel; each loads half of the token rows.
// GATHER: row p of the result reads token slots[p] / top_k.
template <int BT, int STAGES, bool SWIGLU, bool PAIR, bool GATHER>
__global__ void __launch_bounds__(experts_threads(GATHER), BT == 64 ? 2 : 1)
experts_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ TokenMaps map_x, const ExpertsParams p)
{
    static_assert(BT == 32 || BT == 64 || BT == 256, "at most 256 columns of an MMA, boxes of a quarter of the rows");
    constexpr uint32_t kBytesW = kBM * kBK;
    constexpr int kRowsX = PAIR ? BT / 2 : BT;  // token rows that this CTA loads
    constexpr int kAlign = PAIR ? 32 : 16;      // what the columns of an MMA are a multiple of
    constexpr uint32_t kStageBytes = kBytesW + kRowsX * kBK;
    constexpr uint32_t kTmemCols = 2 * BT;
    constexpr int kEpilogueThreads = kExpertsEpilogueThreads;
    constexpr int kChannels = SWIGLU ? kBM / 2 : kBM;  // output channels of a weight tile
    constexpr int kChunk = experts_chunk(PAIR);        // tokens that an epilogue warp turns at a time
    constexpr uint32_t kTurnBytes = experts_turn_bytes(SWIGLU, PAIR) / (kEpilogueThreads / 32);  // of a warp

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    __shared__ __align__(8) uint64_t bar_full[STAGES];
    __shared__ __align__(8) uint64_t bar_empty[STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile uint32_t abort_flag;
    __shared__ __align__(16) float token_scale[2][BT];
    __shared__ __align__(8) uint64_t bar_loaded[STAGES];  // PAIR and GATHER: the peer's copies have landed
    __shared__ __align__(8) uint64_t bar_drained;         // GATHER: all copies of this CTA have
    __shared__ ExpertList<BT> list;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int num_kb = (p.K + kBK - 1) / kBK;
    // PAIR: the two CTAs of a cluster take neighbouring weight tiles of one pair of them; the pair is the scheduling unit.
    const int weight_tiles = (p.N + kChannels * (PAIR ? 2 : 1) - 1) / (kChannels * (PAIR ? 2 : 1));
    const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
    const int64_t first_item = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const int64_t item_step = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int rows_w = SWIGLU ? 2 * p.N : p.N;  // of one expert

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            // the producer's own arrival, the loader threads', and the one that speaks for the peer's loader threads
            mbar_init(&bar_full[s], 1 + (GATHER ? 32 * kExpertsLoaderWarps : 0) + (GATHER && PAIR ? 1 : 0));
            mbar_init(&bar_empty[s], 1);
            if constexpr (GATHER && PAIR) mbar_init(&bar_loaded[s], 32 * kExpertsLoaderWarps);
        }
        if constexpr (GATHER) mbar_init(&bar_drained, 32 * kExpertsLoaderWarps);
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_acc_full[b], 1);
            mbar_init(&bar_acc_empty[b], (PAIR ? 2 : 1) * kEpilogueThreads / 32);
        }
        fence_barrier_init();
        prefetch_tensormap(&map_w);
        if constexpr (!GATHER) {
#pragma unroll
            for (int i = 0; i < 4; ++i) prefetch_tensormap(&map_x.m[i]);
        }
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            tmem_alloc_pair(&tmem_base_slot, kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(&tmem_base_slot, kTmemCols);
            tmem_relinquish_alloc_permit();
        }
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // both CTAs' barriers exist before anything signals them remotely
    tcgen05_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    if (!p.early) pdl_wait();
    build_expert_list(list, p.offsets, p.E, p.rows);

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        uint32_t s = 0, ph = 0;
        uint32_t armed = 0;
        bool ok = true;
        ExpertTile t;
        const uint64_t pol_x = l2_policy_evict_normal();
        const uint64_t pol_w = p.weight_policy_first ? l2_policy_evict_first() : pol_x;
        for (int64_t item = first_item; ok && find_expert_tile<BT, kAlign>(list, p.E, weight_tiles, p.band, item, t); item += item_step) {
            const int cols = ((t.rows + kAlign - 1) & ~(kAlign - 1)) / (PAIR ? 2 : 1);  // of this CTA
            if constexpr (PAIR) t.weight_tile = 2 * t.weight_tile + static_cast<int>(rank), t.row0 += static_cast<int>(rank) * cols;
            const int box = (cols - 1) / (kRowsX / 4);  // the smallest one that holds the tile
            const uint32_t bytes = kBytesW + (GATHER ? 0 : (box + 1) * (kRowsX / 4) * kBK);
            const int w_row = t.weight_tile * kChannels;
            // (one lane) PAIR: the leader arms its barrier for the bytes of both CTAs, the peer only sends bytes
            auto load_weights = [&](int stage, int kb) {
                const uint32_t full = PAIR ? map_to_cta(smem_u32(&bar_full[stage]), 0) : smem_u32(&bar_full[stage]);
                uint8_t* dst = smem + stage * kStageBytes;
                if (rank == 0) mbar_arrive_expect_tx(&bar_full[stage], PAIR ? 2 * bytes : bytes);
                if constexpr (!SWIGLU) {
                    load_tile_2d<PAIR>(dst, &map_w, full, kb * kBK, t.expert * rows_w + w_row, pol_w);
                } else if (p.interleave) {
                    load_tile_5d<PAIR>(dst, &map_w, full, kb * kBK, 0, 0, w_row / 16, t.expert, pol_w);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        load_tile_2d<PAIR>(dst + i * 16 * kBK, &map_w, full, kb * kBK, t.expert * rows_w + w_row + (i >> 1) * 16 + (i & 1) * p.N, pol_w);
                }
            };
            // The weights of the first tile's first K blocks need nothing but its place in the list.
            int ahead = 0;
            if (item == first_item) {
                ahead = min(num_kb, STAGES);
                if (elect_one())
                    for (int kb = 0; kb < ahead; ++kb) load_weights(kb, kb);
                __syncwarp();
                if (p.early) pdl_wait();
                if (lane == 0) pdl_launch_dependents();
            }
            auto load_tokens = [&](int stage, int kb) {  // (one lane)
                if constexpr (!GATHER) {
                    const uint32_t full = PAIR ? map_to_cta(smem_u32(&bar_full[stage]), 0) : smem_u32(&bar_full[stage]);
                    load_tile_2d<PAIR>(smem + stage * kStageBytes + kBytesW, &map_x.m[box], full, kb * kBK, t.row0, pol_x);
                }
            };
            if (ahead > 0) {
                if (elect_one())
                    for (int kb = 0; kb < ahead; ++kb) load_tokens(kb, kb);
                __syncwarp();
                armed = ahead;
                if (ahead == STAGES) s = 0, ph ^= 1;
                else s = ahead;
            }
            for (int kb = ahead; kb < num_kb; ++kb) {
                if (!warp_agrees(wait_or_abort(&bar_empty[s], ph ^ 1, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_PRODUCER)) {
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    load_weights(s, kb);
                    load_tokens(s, kb);
                }
                __syncwarp();
                if (armed < STAGES) ++armed;
                if (++s == STAGES) s = 0, ph ^= 1;
            }
        }
        // (PAIR: the leader's bar_full complete only when both CTAs' bytes have landed; the peer's own are never used)
        drain_stages<STAGES>(PAIR && rank != 0 ? nullptr : bar_full, bar_empty, s, ph, armed, p.status, &abort_flag);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer (of the leader)
        if constexpr (PAIR && GATHER) {
            // In the peer this warp passes on that the loader warps' copies have landed, with one arrival per stage in the leader's shared
            // memory.  What reads the copies is the peer's own tensor core, through its own shared memory: they have landed when this warp sees
            // their barrier complete, it makes them visible to the async proxy there, and nothing of them has to become visible in the
            // leader, whose instruction only starts that read.  So the arrival has the default semantics of the hand-backs between the
            // CTAs; a release at cluster scope takes longer than the MMAs of a K block (32768 rows, SwiGLU 4096 x 4096: 1290 us for 485).
            if (rank != 0) {
                uint32_t fs = 0, fph = 0;
                bool going = true;
                ExpertTile f;
                for (int64_t item = first_item; going && find_expert_tile<BT, kAlign>(list, p.E, weight_tiles, p.band, item, f); item += item_step)
                    for (int kb = 0; kb < num_kb; ++kb) {
                        if (!warp_agrees(wait_or_abort(&bar_loaded[fs], fph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_MMA)) {
                            going = false;
                            break;
                        }
                        fence_proxy_async_smem();
                        if (elect_one()) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_full[fs]), 0));
                        __syncwarp();
                        if (++fs == STAGES) fs = 0, fph ^= 1;
                    }
            }
        }
        uint32_t s = 0, ph = 0;
        uint32_t local_tile = 0;
        bool ok = rank == 0;
        ExpertTile t;
        const uint32_t w_0 = smem_desc_lo(smem_u32(smem));
        for (int64_t item = first_item; ok && find_expert_tile<BT, kAlign>(list, p.E, weight_tiles, p.band, item, t); item += item_step, ++local_tile) {
            const uint32_t buf = local_tile & 1;
            const uint32_t acc_ph = (local_tile >> 1) & 1;
            if (!warp_agrees(wait_or_abort(&bar_acc_empty[buf], acc_ph ^ 1, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_MMA)) break;
            tcgen05_fence_after_sync();
            const uint32_t idesc = make_idesc_i8(PAIR ? 2 * kBM : kBM, 0, false) | (static_cast<uint32_t>((t.rows + kAlign - 1) & ~(kAlign - 1)) >> 3) << 17;
            const uint32_t tmem_d = tmem_base + buf * BT;
            for (int kb = 0; kb < num_kb; ++kb) {
                if (!warp_agrees(wait_or_abort(&bar_full[s], ph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_MMA)) {
                    ok = false;
                    break;
                }
                if constexpr (GATHER) fence_proxy_async_smem();  // the loader threads' copies, made by the generic proxy
                tcgen05_fence_after_sync();
                const uint32_t dw = w_0 + s * (kStageBytes / 16), dx = dw + kBytesW / 16;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kBK / kUmmaK; ++k) {
                        if constexpr (PAIR) umma_i8_pair(tmem_d, smem_desc_k128_of(dw + 2 * k), smem_desc_k128_of(dx + 2 * k), idesc, (kb | k) != 0);
                        else umma_i8(tmem_d, smem_desc_k128_of(dw + 2 * k), smem_desc_k128_of(dx + 2 * k), idesc, (kb | k) != 0);
                    }
                    if constexpr (PAIR) {
                        umma_commit_pair(map_to_cta(smem_u32(&bar_empty[s]), 0));
                        umma_commit_pair(map_to_cta(smem_u32(&bar_empty[s]), 1));
                    } else {
                        umma_commit(&bar_empty[s]);
                    }
                }
                __syncwarp();
                if (++s == STAGES) s = 0, ph ^= 1;
            }
            if (ok && elect_one()) {
                if constexpr (PAIR) {
                    umma_commit_pair(map_to_cta(smem_u32(&bar_acc_full[buf]), 0));
                    umma_commit_pair(map_to_cta(smem_u32(&bar_acc_full[buf]), 1));
                } else {
                    umma_commit(&bar_acc_full[buf]);
                }
            }
            __syncwarp();
        }
    } else if (GATHER && warp >= 2 + kEpilogueThreads / 32) {
        // ------------------------------------------------------------------ loader warps
        if constexpr (GATHER) {
            if (p.early) pdl_wait();
            const int chunk = lane & 7;                // 16 bytes of a row's 128
            const int sub = (warp - 2 - kEpilogueThreads / 32) * 4 + (lane >> 3);  // of 16 rows
            const uint32_t place = smem_u32(smem) + kBytesW + sub * kBK + ((chunk ^ (sub & 7)) << 4);
            uint32_t s = 0, ph = 0;
            bool ok = true;
            ExpertTile t;
            for (int64_t item = first_item; ok && find_expert_tile<BT, kAlign>(list, p.E, weight_tiles, p.band, item, t); item += item_step) {
                const int cols = ((t.rows + kAlign - 1) & ~(kAlign - 1)) / (PAIR ? 2 : 1);  // of this CTA
                const int before = static_cast<int>(rank) * cols;
                const int8_t* src[kRowsX / 16];
#pragma unroll
                for (int j = 0; j < kRowsX / 16; ++j) {
                    const int r = before + j * 16 + sub;  // rows that pad the tile read token 0, and are not stored
                    const int slot = j * 16 < cols && r < t.rows ? __ldg(p.slots + t.row0 + r) : 0;
                    src[j] = p.x + static_cast<int64_t>(min(max(slot, 0) / p.top_k, p.tokens - 1)) * p.K;
                }
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!warp_agrees(wait_or_abort(&bar_empty[s], ph ^ 1, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_PRODUCER)) {
                        ok = false;
                        break;
                    }
                    const int k = kb * kBK + chunk * 16;
                    const uint32_t bytes = k < p.K ? 16u : 0u;  // zeros behind K
                    const uint32_t dst = place + s * kStageBytes;
#pragma unroll
                    for (int j = 0; j < kRowsX / 16; ++j)
                        if (j * 16 < cols) cp_async_16(dst + j * 16 * kBK, src[j] + (bytes ? k : 0), bytes);
                    // every thread's arrival follows its copies when they have landed; whoever waits for it makes them visible to the async proxy
                    cp_async_arrive(PAIR && rank != 0 ? &bar_loaded[s] : &bar_full[s]);
                    if (++s == STAGES) s = 0, ph ^= 1;
                }
            }
            // No copy and no arrival is on its way any more when the CTA exits (those on the stages have been waited for by the roles behind
            // them, unless a wait has failed).
            cp_async_arrive(&bar_drained);
            cp_async_wait_all();
            mbar_wait(&bar_drained, 0);
        }
    } else {
        // ------------------------------------------------------------------ epilogue warps
        const int quarter = warp & 3;  // TMEM lanes [32 * quarter, 32 * quarter + 32)
        const int et = static_cast<int>(threadIdx.x) - 64;
        const uint32_t turn = smem_u32(smem) + STAGES * kStageBytes + (et >> 5) * kTurnBytes;
        if (p.early) pdl_wait();
        // rows that belong to no expert: in front of the first and behind the last
        auto clear = [&](int64_t first, int64_t end) {
            const int64_t step = static_cast<int64_t>(gridDim.x) * kEpilogueThreads, at = static_cast<int64_t>(blockIdx.x) * kEpilogueThreads + et;
            if (p.vec) {
                for (int64_t i = first / 8 + at; i < end / 8; i += step) reinterpret_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
            } else {
                for (int64_t i = first + at; i < end; i += step) p.out[i] = 0;
            }
        };
        clear(0, static_cast<int64_t>(list.start[0]) * p.N);
        clear(static_cast<int64_t>(max(list.start[p.E], list.start[0])) * p.N, p.rows * p.N);
        uint32_t local_tile = 0;
        bool ok = true;
        ExpertTile t;
        for (int64_t item = first_item; find_expert_tile<BT, kAlign>(list, p.E, weight_tiles, p.band, item, t); item += item_step, ++local_tile) {
            const uint32_t buf = local_tile & 1;
            const uint32_t acc_ph = (local_tile >> 1) & 1;
            if constexpr (PAIR) t.weight_tile = 2 * t.weight_tile + static_cast<int>(rank);
            // The scales are fetched while the tile is computed.  (A warp that fills this buffer again has passed the barrier of the tile
            // in between, behind which nobody reads it any more.)
            for (int r = et; r < BT; r += kEpilogueThreads) {
                float v = 0.0f;
                if (r < t.rows) {
                    int src = t.row0 + r;
                    if constexpr (GATHER) src = min(max(__ldg(p.slots + src), 0) / p.top_k, p.tokens - 1);
                    v = __ldg(p.sx + src);
                }
                token_scale[buf][r] = v;
            }
            // This thread's channels: lane / 4 + 0, 8 (SWIGLU: gate and up of them), 16, 24 of the warp's run.
            const int channel0 = t.weight_tile * kChannels + quarter * (kChannels / 4);
            uint64_t channel_scale[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int ch = channel0 + (lane >> 2) + (SWIGLU ? (m & 1) * 8 : m * 8);
                const float v = ch < p.N ? __ldg(p.sw + static_cast<int64_t>(t.expert) * rows_w + ch + (SWIGLU && m >= 2 ? p.N : 0)) : 0.0f;
                channel_scale[m] = f32x2(v, v);
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory");  // the epilogue warps
            // After a failed wait the warp goes on through the list without touching anything: the named barrier above has no time limit and
            // needs every warp once per tile.
            if (!ok || !warp_agrees(wait_or_abort(&bar_acc_full[buf], acc_ph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_EPILOGUE)) {
                ok = false;
                continue;
            }
            tcgen05_fence_after_sync();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * BT;
#pragma unroll 1
            for (int c = 0; c < t.rows; c += kChunk) {
                uint32_t v[2][kChunk / 2];  // lanes 0 .. 15 and 16 .. 31 of the warp's quarter
                __syncwarp();  // (the last chunk has left the turning buffer)
                tmem_ld_16x256b(taddr + c, v[0]);
                tmem_ld_16x256b(taddr + (16u << 16) + c, v[1]);
                tmem_ld_wait();
                uint32_t w[kChunk / 8][SWIGLU ? 2 : 4];  // pairs of tokens, per run of eight channels
#pragma unroll
                for (int i = 0; i < kChunk / 8; ++i) {
                    const uint64_t token_pair = *reinterpret_cast<const uint64_t*>(&token_scale[buf][c + 8 * i + 2 * (lane & 3)]);
                    uint64_t f[4];
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const uint32_t a = v[m >> 1][4 * i + 2 * (m & 1)], b = v[m >> 1][4 * i + 2 * (m & 1) + 1];
                        f[m] = mul2(f32x2(__int2float_rn(static_cast<int32_t>(a)), __int2float_rn(static_cast<int32_t>(b))), mul2(token_pair, channel_scale[m]));
                    }
#pragma unroll
                    for (int m = 0; m < (SWIGLU ? 2 : 4); ++m) {
                        float x, y;
                        f32x2_split(f[m], x, y);
                        if constexpr (SWIGLU) {
                            float ux, uy;
                            f32x2_split(f[m + 2], ux, uy);
                            x = silu(x) * ux, y = silu(y) * uy;
                        }
                        w[i][m] = pack_bf16x2(x, y);
                    }
                }
                // Rows of the turning buffer are tokens, of 64 (32) bytes, whose 16-byte pieces are permuted so that neither side meets bank conflicts.
                if constexpr (SWIGLU) {
                    const uint32_t at = turn + (lane & 7) * 32 + (lane >> 4) * 256 + ((((lane >> 3) & 1) ^ ((lane >> 2) & 1)) << 4);
#pragma unroll
                    for (int i = 0; i < kChunk / 8; i += 2) stmatrix_x4_trans(at + i * 256, w[i][0], w[i][1], w[i + 1][0], w[i + 1][1]);
                } else {
                    const uint32_t at = turn + (lane & 7) * 64 + (((lane >> 3) ^ ((lane >> 1) & 3)) << 4);
#pragma unroll
                    for (int i = 0; i < kChunk / 8; ++i) stmatrix_x4_trans(at + i * 512, w[i][0], w[i][1], w[i][2], w[i][3]);
                }
                __syncwarp();
                constexpr int kPieces = SWIGLU ? 2 : 4;  // of 16 bytes in a token's run
                auto piece_at = [&](int token, int piece) {
                    return turn + token * (16 * kPieces) + ((piece ^ (SWIGLU ? (token >> 2) & 1 : (token >> 1) & 3)) << 4);
                };
                if (p.vec) {
                    const int piece = lane & (kPieces - 1), ch = channel0 + piece * 8;
                    uint16_t* dst = p.out + static_cast<int64_t>(t.row0 + c + lane / kPieces) * p.N + ch;
#pragma unroll
                    for (int i = 0; i < kChunk * kPieces / 32; ++i) {
                        const int token = i * (32 / kPieces) + lane / kPieces;
                        const uint4 u = ld_shared_v4(piece_at(token, piece));
                        if (c + token < t.rows && ch < p.N) *reinterpret_cast<uint4*>(dst) = u;
                        dst += static_cast<int64_t>(32 / kPieces) * p.N;
                    }
                } else {
                    // 2 bytes a lane: a token's run (SWIGLU: those of two) at a time, eight of them read before the first is written
                    const int ch = lane & (8 * kPieces - 1);
                    constexpr int kStep = 4 / kPieces;
                    const bool ch_ok = channel0 + ch < p.N;
#pragma unroll
                    for (int first = 0; first < kChunk; first += 8 * kStep) {
                        const int token0 = first + lane / (8 * kPieces);
                        uint16_t u[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) u[i] = ld_shared_u16(piece_at(token0 + i * kStep, ch >> 3) + (ch & 7) * 2);
                        uint16_t* dst = p.out + static_cast<int64_t>(t.row0 + c + token0) * p.N + channel0 + ch;
#pragma unroll
                        for (int i = 0; i < 8; ++i, dst += static_cast<int64_t>(kStep) * p.N)
                            if (ch_ok && c + token0 + i * kStep < t.rows) *dst = u[i];
                    }
                }
            }
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if constexpr (PAIR) mbar_arrive_cluster(map_to_cta(smem_u32(&bar_acc_empty[buf]), 0));
                else mbar_arrive(&bar_acc_empty[buf]);
            }
        }
    }

    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // neither CTA leaves while the other may still read or signal it
    if (warp == 1) {
        __syncwarp();
        tcgen05_fence_after_sync();
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, kTmemCols);
        else tmem_dealloc(tmem_base, kTmemCols);
    }
}

}  // namespace gi8
