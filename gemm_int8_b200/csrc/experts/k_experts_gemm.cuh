// Products of row groups with one int8 weight per group (the experts' linear layers), for sm_100a:
//   out[p, n] = bf16( fp32(sum_k X[src(p), k] * W[e, n, k]) * (sx[src(p)] * sw[e, n]) )    for offsets[e] <= p < offsets[e + 1]
// and, with SWIGLU, for a weight of 2 N rows (N gate rows, then N up rows) per expert:
//   out[p, n] = bf16( g / (1 + exp(-g)) * u ),  g, u = the fp32 values of channels n and N + n
// src(p) is p, or the token slots[p] / top_k.  Rows behind offsets[E] are written as zeros.  How many rows an expert has is known on the
// device alone, so every CTA works the list of tiles out of the offsets by itself.
//
// Operands are swapped: the 128 rows of a WEIGHT tile fill the M = 128 side of tcgen05.mma and the expert's rows are the N side,
// whose extent is an operand of the instruction: a tile of r rows costs roundup(r, 16) columns instead of a multiple of 128, which
// is what makes ragged groups and single tokens cheap.  An expert's rows are cut into equal tiles of at most BT.
//
// Structure (one persistent CTA per SM, 192 threads), as in the dense kernel:
//   warp 0      TMA producer: weight tiles (128 rows x 128 bytes) and token rows, the latter in boxes of 32 rows or, gathered, four
//               rows per instruction wherever they lie; all lanes issue
//   warp 1      MMA issuer, kind::i8, two accumulators in tensor memory
//   warps 2..5  epilogue: a lane holds one output channel and walks over the tile's tokens
// SWIGLU: a weight tile is 64 gate rows and their 64 up rows in alternating runs of 16, so that gate and up of a channel lie 16 lanes
// apart in one warp, which exchanges half of the tokens by shuffles and computes 16 results per lane.
#pragma once

#include "../k_dense.cuh"

namespace gi8 {

constexpr int kExpertsThreads = 192;
constexpr int kExpertsMaxExperts = 1024;

struct ExpertsParams {
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
    int vec_zero;            // rows behind the last group can be cleared in 16-byte pieces
    int weight_policy_first; // weights are met once or twice: keep them from displacing the rest of L2
};

// g / (1 + exp(-g)), by the exponential that does not overflow: far below zero the result fades out through the subnormals.
GI8_DEVICE float silu(float g)
{
    const float t = expf(-fabsf(g));
    return g * ((g < 0.0f ? t : 1.0f) / (1.0f + t));
}

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
};

// Whole CTA.  Offsets that are no ascending sequence within [0, rows] give wrong rows, never an access out of bounds.
template <int BT>
GI8_DEVICE void build_expert_list(ExpertList<BT>& list, const int32_t* offsets, int E, int64_t rows)
{
    for (int e = threadIdx.x; e <= E; e += blockDim.x)
        list.start[e] = static_cast<int32_t>(min(max(static_cast<int64_t>(__ldg(offsets + e)), static_cast<int64_t>(0)), rows));
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int carry = 0;
        for (int base = 0; base < E; base += 32) {
            const int e = base + lane;
            int n = e < E ? max(0, list.start[e + 1] - list.start[e]) : 0;
            n = (n + BT - 1) / BT;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, n, o);
                if (lane >= o) n += v;
            }
            if (e < E) list.tiles_end[e] = carry + n;
            carry += __shfl_sync(0xffffffffu, n, 31);
        }
    }
    __syncthreads();
}

// Tile `item` of the list, if there is one: experts in order, within an expert weight tile by weight tile with the token tiles inside,
// so that CTAs that run at the same time share weights.  Whole warp; `chunk` is the 32 experts where the last search ended.
template <int BT>
GI8_DEVICE bool find_expert_tile(const ExpertList<BT>& list, int E, int weight_tiles, int64_t item, int& chunk, ExpertTile& t)
{
    const int lane = threadIdx.x & 31;
    for (; chunk < E; chunk += 32) {
        const int e = chunk + lane;
        const bool past = e < E && static_cast<int64_t>(list.tiles_end[e]) * weight_tiles > item;
        const uint32_t hit = __ballot_sync(0xffffffffu, past);
        if (hit) {
            t.expert = chunk + __ffs(hit) - 1;
            const int before = t.expert ? list.tiles_end[t.expert - 1] : 0;
            const int tiles = list.tiles_end[t.expert] - before;
            const int r = static_cast<int>(item - static_cast<int64_t>(before) * weight_tiles);
            t.weight_tile = r / tiles;
            const int n = list.start[t.expert + 1] - list.start[t.expert];
            const int per = ((n + tiles - 1) / tiles + 15) & ~15;  // <= BT, and the last tile keeps at least a row
            const int first = (r - t.weight_tile * tiles) * per;
            t.row0 = list.start[t.expert] + first;
            t.rows = min(per, n - first);
            return true;
        }
    }
    return false;
}

template <int BT, int STAGES, bool SWIGLU>
__global__ void __launch_bounds__(kExpertsThreads, 1)
experts_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const ExpertsParams p)
{
    static_assert(BT == 32 || BT == 64 || BT == 128 || BT == 256, "token rows come in boxes of 32, at most 256 columns of an MMA");
    constexpr uint32_t kBytesW = kBM * kBK;
    constexpr uint32_t kStageBytes = kBytesW + BT * kBK;
    constexpr uint32_t kTmemCols = 2 * BT;
    constexpr int kChannels = SWIGLU ? kBM / 2 : kBM;  // output channels of a weight tile

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    __shared__ __align__(8) uint64_t bar_full[STAGES];
    __shared__ __align__(8) uint64_t bar_empty[STAGES];
    __shared__ __align__(8) uint64_t bar_acc_full[2];
    __shared__ __align__(8) uint64_t bar_acc_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile uint32_t abort_flag;
    __shared__ __align__(16) float token_scale[2][BT];
    __shared__ ExpertList<BT> list;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int num_kb = (p.K + kBK - 1) / kBK;
    const int weight_tiles = (p.N + kChannels - 1) / kChannels;
    const int rows_w = SWIGLU ? 2 * p.N : p.N;  // of one expert

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&bar_full[s], 1);
            mbar_init(&bar_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&bar_acc_full[b], 1);
            mbar_init(&bar_acc_empty[b], 4);
        }
        fence_barrier_init();
        prefetch_tensormap(&map_w);
        prefetch_tensormap(&map_x);
    }
    if (warp == 1) {
        tmem_alloc(&tmem_base_slot, kTmemCols);
        tmem_relinquish_alloc_permit();
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    tcgen05_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    pdl_wait();
    if (threadIdx.x == 0) pdl_launch_dependents();
    build_expert_list(list, p.offsets, p.E, p.rows);

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        uint32_t s = 0, ph = 0;
        uint32_t armed = 0;
        bool ok = true;
        int chunk = 0;
        ExpertTile t;
        const uint64_t pol_w = p.weight_policy_first ? l2_policy_evict_first() : l2_policy_evict_normal();
        for (int64_t item = blockIdx.x; ok && find_expert_tile(list, p.E, weight_tiles, item, chunk, t); item += gridDim.x) {
            const int cols = (t.rows + 15) & ~15;
            // This lane's part of the token rows: four consecutive places of the tile per gather, 32 per box.
            constexpr int kGathers = (BT + 127) / 128;
            int32_t src[kGathers][4];
            if (p.slots) {
#pragma unroll
                for (int g = 0; g < kGathers; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = (g * 32 + lane) * 4 + i;  // rows that pad the tile read token 0, and are not stored
                        const int slot = r < t.rows ? __ldg(p.slots + t.row0 + r) : 0;
                        src[g][i] = min(max(slot, 0) / p.top_k, p.tokens - 1);
                    }
            }
            const uint32_t bytes = kBytesW + (p.slots ? cols : (cols + 31) & ~31) * kBK;
            const int w_row = t.expert * rows_w + t.weight_tile * kChannels;
            for (int kb = 0; kb < num_kb; ++kb) {
                if (!warp_agrees(wait_or_abort(&bar_empty[s], ph ^ 1, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_PRODUCER)) {
                    ok = false;
                    break;
                }
                uint8_t* sw_tile = smem + s * kStageBytes;
                uint8_t* sx_tile = sw_tile + kBytesW;
                if (elect_one()) {
                    mbar_arrive_expect_tx(&bar_full[s], bytes);
                    if constexpr (!SWIGLU) tma_load_2d_hint(sw_tile, &map_w, &bar_full[s], kb * kBK, w_row, pol_w);
                }
                __syncwarp();
                if constexpr (SWIGLU) {
                    // runs of 16 rows: gate, up, gate, up, ...
                    if (lane < 8) tma_load_2d_hint(sw_tile + lane * 16 * kBK, &map_w, &bar_full[s], kb * kBK, w_row + (lane >> 1) * 16 + (lane & 1) * p.N, pol_w);
                }
                if (p.slots) {
#pragma unroll
                    for (int g = 0; g < kGathers; ++g)
                        if ((g * 32 + lane) * 4 < cols)
                            tma_gather4(sx_tile + (g * 32 + lane) * 4 * kBK, &map_x, &bar_full[s], kb * kBK, src[g][0], src[g][1], src[g][2], src[g][3]);
                } else {
                    if (lane * 32 < cols) tma_load_2d(sx_tile + lane * 32 * kBK, &map_x, &bar_full[s], kb * kBK, t.row0 + lane * 32);
                }
                __syncwarp();
                if (armed < STAGES) ++armed;
                if (++s == STAGES) s = 0, ph ^= 1;
            }
        }
        drain_stages<STAGES>(bar_full, bar_empty, s, ph, armed, p.status, &abort_flag);
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        uint32_t s = 0, ph = 0;
        uint32_t local_tile = 0;
        bool ok = true;
        int chunk = 0;
        ExpertTile t;
        const uint32_t w_0 = smem_desc_lo(smem_u32(smem));
        for (int64_t item = blockIdx.x; ok && find_expert_tile(list, p.E, weight_tiles, item, chunk, t); item += gridDim.x, ++local_tile) {
            const uint32_t buf = local_tile & 1;
            const uint32_t acc_ph = (local_tile >> 1) & 1;
            if (!warp_agrees(wait_or_abort(&bar_acc_empty[buf], acc_ph ^ 1, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_MMA)) break;
            tcgen05_fence_after_sync();
            const uint32_t idesc = make_idesc_i8(kBM, 0, false) | (static_cast<uint32_t>((t.rows + 15) & ~15) >> 3) << 17;
            const uint32_t tmem_d = tmem_base + buf * BT;
            for (int kb = 0; kb < num_kb; ++kb) {
                if (!warp_agrees(wait_or_abort(&bar_full[s], ph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_MMA)) {
                    ok = false;
                    break;
                }
                tcgen05_fence_after_sync();
                const uint32_t dw = w_0 + s * (kStageBytes / 16), dx = dw + kBytesW / 16;
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kBK / kUmmaK; ++k) umma_i8(tmem_d, smem_desc_k128_of(dw + 2 * k), smem_desc_k128_of(dx + 2 * k), idesc, (kb | k) != 0);
                    umma_commit(&bar_empty[s]);
                }
                __syncwarp();
                if (++s == STAGES) s = 0, ph ^= 1;
            }
            if (ok && elect_one()) umma_commit(&bar_acc_full[buf]);
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------------ epilogue warps
        const int quarter = warp & 3;  // TMEM lanes [32 * quarter, 32 * quarter + 32)
        const int et = static_cast<int>(threadIdx.x) - 64;
        {
            // rows that belong to no expert
            const int64_t first = static_cast<int64_t>(list.start[p.E]) * p.N, end = p.rows * p.N;
            const int64_t step = static_cast<int64_t>(gridDim.x) * 128, at = static_cast<int64_t>(blockIdx.x) * 128 + et;
            if (p.vec_zero) {
                for (int64_t i = first / 8 + at; i < end / 8; i += step) reinterpret_cast<uint4*>(p.out)[i] = make_uint4(0, 0, 0, 0);
            } else {
                for (int64_t i = first + at; i < end; i += step) p.out[i] = 0;
            }
        }
        uint32_t local_tile = 0;
        bool ok = true;
        int chunk = 0;
        ExpertTile t;
        for (int64_t item = blockIdx.x; find_expert_tile(list, p.E, weight_tiles, item, chunk, t); item += gridDim.x, ++local_tile) {
            const uint32_t buf = local_tile & 1;
            const uint32_t acc_ph = (local_tile >> 1) & 1;
            // The scales are fetched while the tile is computed.  (A warp that fills this buffer again has passed the barrier of the tile
            // in between, behind which nobody reads it any more.)
            for (int r = et; r < BT; r += 128) {
                float v = 0.0f;
                if (r < t.rows) {
                    int src = t.row0 + r;
                    if (p.slots) src = min(max(__ldg(p.slots + src), 0) / p.top_k, p.tokens - 1);
                    v = __ldg(p.sx + src);
                }
                token_scale[buf][r] = v;
            }
            const int channel = t.weight_tile * kChannels + (SWIGLU ? quarter * 16 + (lane & 15) : quarter * 32 + lane);
            const bool channel_ok = channel < p.N;
            float channel_scale = 0.0f;
            if (channel_ok) channel_scale = __ldg(p.sw + static_cast<int64_t>(t.expert) * rows_w + channel + (SWIGLU && lane >= 16 ? p.N : 0));
            asm volatile("bar.sync 1, 128;" ::: "memory");  // the four epilogue warps
            // After a failed wait the warp goes on through the list without touching anything: the named barrier above has no time limit and
            // needs all four warps once per tile.
            if (!ok || !warp_agrees(wait_or_abort(&bar_acc_full[buf], acc_ph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_EPILOGUE)) {
                ok = false;
                continue;
            }
            tcgen05_fence_after_sync();
            const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + buf * BT;
#pragma unroll 1
            for (int c = 0; c < t.rows; c += 32) {
                uint32_t v[32];
                __syncwarp();
                tmem_ld_32x32b_x32(taddr + c, v);
                tmem_ld_wait();
                float f[32];
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    const float4 s4 = *reinterpret_cast<const float4*>(&token_scale[buf][c + j]);
                    f[j] = __int2float_rn(static_cast<int32_t>(v[j])) * (s4.x * channel_scale);
                    f[j + 1] = __int2float_rn(static_cast<int32_t>(v[j + 1])) * (s4.y * channel_scale);
                    f[j + 2] = __int2float_rn(static_cast<int32_t>(v[j + 2])) * (s4.z * channel_scale);
                    f[j + 3] = __int2float_rn(static_cast<int32_t>(v[j + 3])) * (s4.w * channel_scale);
                }
                if constexpr (SWIGLU) {
                    const bool up_lane = lane >= 16;
                    const int first = c + (up_lane ? 16 : 0);  // this lane's sixteen tokens
                    uint16_t* dst = p.out + static_cast<int64_t>(t.row0 + first) * p.N + channel;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float other = __shfl_xor_sync(0xffffffffu, up_lane ? f[j] : f[16 + j], 16);
                        const float gate = up_lane ? other : f[j], up = up_lane ? f[16 + j] : other;
                        if (channel_ok && first + j < t.rows) *dst = to_bf16_bits(silu(gate) * up);
                        dst += p.N;
                    }
                } else {
                    uint16_t* dst = p.out + static_cast<int64_t>(t.row0 + c) * p.N + channel;
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (channel_ok && c + j < t.rows) *dst = to_bf16_bits(f[j]);
                        dst += p.N;
                    }
                }
            }
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_acc_empty[buf]);
        }
    }

    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tcgen05_fence_after_sync();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

}  // namespace gi8
