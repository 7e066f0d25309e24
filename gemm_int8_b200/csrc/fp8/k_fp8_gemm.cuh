// Block-scaled product of e4m3 operands for sm_100a:
//   out[m,n] = bf16( sum_kb P[m,n,kb] * (sa[m,kb] * sw[n/128,kb]) (+ bias[n]) ),  kb ascending, one fused multiply-add in fp32 per K block
//   (128 wide), P the block's fp32 dot product on the tensor cores, one rounding at the end.
//
// Structure, as in k_blockwise.cuh (one persistent CTA per SM, or two CTAs on one 256 x 256 tile): warp 0 loads operand tiles by TMA, warps 1 and 3 issue the MMAs,
// whose partials of a K block lie in tensor memory, warps 4..11 promote them: tensor-memory loads and one fma.rn.f32x2 per pair of columns into fp32 accumulators in
// registers, then the epilogue.  Partials are fp32 as they come, so there is no bias MMA and no conversion.  What is done otherwise than there:
//   - A half of the wide tile (128 columns) belongs to ONE of the two column groups of promotion warps, with an issuer, buffers and barriers of its own.  A warp has one
//     hand-over a K block, not two, and while the warps of one half wait for theirs those of the other work: 8192^3 495 -> 453 us, 2048 x 11008 x 4096 90 -> 82.
//     In the two-CTA form each CTA loads 64 weight rows of either half, so that a half is 128 neighbouring columns, one weight block.
//   - The barrier that frees a stage also says that its partial is there: one commit a half and K block.
//   - Row scales come through shared memory, 64 bytes of a row at a time, by asynchronous copies of warp 2; as 16-byte loads of the promotion warps, each touching
//     32 rows, they cost 80 - 100 of 800 cycles.  The weight block's scales are held by the lanes of a warp and broadcast by shuffles.
//   - Packed multiply-adds: scalar ones, with the register banks they get, took 760 cycles a K block for 705.
//   - No branch leaves the loop over the K blocks: with early exits it spilled accumulators (205 us for 136).  The split forms of 256 and 128 columns still spill 12 and 16
//     bytes, reloaded at 11 and 32 places: 265 ns a K block of 128 columns in four splits of sixteen tiles, next to 230 - 300 of the form without splits.
//
// Bound (two-CTA form, 2048 x 9472 x 8192, cycles a K block, copies of the kernel with parts left out): all 705; without scale loads 612; without multiply-adds 567; with
// neither multiply-adds nor tensor-memory loads 570: the MMAs with their operands, 512 at the nominal rate; without MMAs 620.  So the promotion loop, a chain of
// four loads and their arithmetic and one hand-over for each warp, binds, not far in front of the MMAs; tensor pipe 70 % of the active cycles.  For a second on end the chip
// holds 1.1 GHz at 1000 W (8192^3 561 us with random codes) and takes as long as it needs energy: N = 256 MMAs, which fetch the rows of x once, took 806 cycles at
// 1.24 GHz, 581 us.  The one-CTA 256-wide form is bound by its operand bytes (48 KB a K block at 67 bytes a cycle, the most an SM drew from L2: 719 cycles without any
// MMA).  An epilogue takes 3000 cycles a tile, half of them its TMA stores (with three staging blocks a warp 2800, with one fence a tile 2500, as plain 16-byte stores 4100;
// nothing of it showed in the times).  Stages of the two-CTA form: six, five and four level, level and 5 % slower.
//
// Barrier protocol: see k_blockwise.cuh.  bar_full[s]: TMA bytes; waiters: the issuers.  bar_done[h][s]: the commit of half h; waiters: the producer, whose refill the
// next completion needs, and half h's promotion warps, whose hand-back the next completion needs (STAGES >= NBUF).  bar_part_empty[h][b]: the arrivals of half h's promotion
// warps, of both CTAs of a pair; waiter: the half's issuer.  bar_scale_full[g]: arrivals of warp 2's lanes behind their copies; waiters: the promotion warps, whose
// arrivals on bar_scale_empty[g] the next completion needs.  Narrow tiles have one part, whose K blocks the issuers take in turn.
#pragma once

#include "../k_blockwise.cuh"
#include "../k_quant.cuh"  // packed arithmetic

namespace gi8 {

struct Fp8GemmParams {
    void* out;             // bf16 [M, N], leading dimension ldo
    const float* sa;       // [M, KB], row stride ld_sa
    const float* sw;       // [ceil(N/128), KB], row stride ld_sw
    const void* bias;      // [N], bf16 or fp32 (BIAS)
    uint32_t* status;
    int64_t ldo, ld_sa, ld_sw;
    int M, N, K;
    int tiles_m, tiles_n;
    int group_m;       // row blocks per rasterisation band
    int tma_store;     // rows of the output can be written by TMA
    int pair_ok;       // out is 4-byte aligned and ldo even
    int bias_vec;      // bias is 16-byte aligned
    int after_quant;   // launched as the programmatic dependent of the quantiser that writes x and sa (and of nothing else)
    int scale_vec;     // ceil(K/128) % 4 == 0 and the rows of sa are 16-byte aligned: scales are copied four at a time
    int splits, kb_per_split;  // SPLITK: CTAs of a cluster (BN / splits a multiple of 32), K blocks of each (a multiple of 4; the last has the rest)
    int box_rows;      // rows of x that a load brings: all 128, or as many as there are (the tile's other rows are whatever lies there, and stored by nobody)
    int release_late;  // do not let the next launch start before the CTAs have ended (see the host's release_late)
};

// (224 and 48, 240 and 24: the same)
constexpr int kFp8PromoRegs = 232, kFp8ControlRegs = 40;
static_assert(kPromoWarps * (kFp8PromoRegs - kLaunchRegs) <= 4 * (kLaunchRegs - kFp8ControlRegs), "setmaxnreg pool unbalanced");

constexpr int kFp8ScaleGroup = 16;                                   // K blocks whose row scales are brought into shared memory together ...
constexpr uint32_t kFp8ScaleBytes = kBM * kFp8ScaleGroup * 4;         // ... 64 bytes of each row, two groups in turn
constexpr int kFp8StoreCols = 32;                                     // columns of a store box: 32 rows x 64 bytes, 64-byte swizzle
constexpr uint32_t kFp8StoreBytes = 32 * kFp8StoreCols * 2;

__host__ __device__ constexpr size_t fp8_smem_bytes(int bn, int stages, bool pair)
{
    return static_cast<size_t>(stages) * (kBM + (pair ? bn / 2 : bn)) * kBK + kPromoWarps * kFp8StoreBytes + 2 * kFp8ScaleBytes + 1024;
}

// global -> shared copy of 4 bytes, see cp_async_16.
GI8_DEVICE void cp_async_4(uint32_t smem_dst, const void* src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_dst), "l"(src) : "memory");
}

// Where the four scales c (of four) of row r lie in a group: eight neighbouring rows' 16 bytes take different banks.
GI8_DEVICE uint32_t fp8_scale_at(int r, int c) { return static_cast<uint32_t>(r * 64 + ((c ^ ((r >> 1) & 3)) * 16)); }

// (A type of the kernel, not an argument: with both in one epilogue the layer of 2048 x 11008 x 4096 with a bf16 bias took 103 us for 96.)
enum class Fp8Bias { kNone, kBf16, kF32 };

// The bias of column col, and of eight columns from col on as fp32 pairs (0 behind the last; vec: 16-byte loads where all eight exist).
template <Fp8Bias BIAS>
GI8_DEVICE float fp8_bias(const void* bias, int col)
{
    if constexpr (BIAS == Fp8Bias::kF32) return __ldg(static_cast<const float*>(bias) + col);
    else return __uint_as_float(static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(bias) + col)) << 16);
}

template <Fp8Bias BIAS>
GI8_DEVICE void fp8_bias8(const void* bias, int col, int N, bool vec, uint64_t (&b)[4])
{
    if constexpr (BIAS == Fp8Bias::kBf16) {
        const uint4 u = load_bias8(static_cast<const uint16_t*>(bias), col, N, vec);
        unpack16<__nv_bfloat16>(u, b);
    } else if (vec && col + 8 <= N) {
        const uint4* at = reinterpret_cast<const uint4*>(static_cast<const float*>(bias) + col);
        unpack16<float>(__ldg(at), reinterpret_cast<uint64_t(&)[2]>(b[0])), unpack16<float>(__ldg(at + 1), reinterpret_cast<uint64_t(&)[2]>(b[2]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            b[i] = f32x2(col + 2 * i < N ? fp8_bias<BIAS>(bias, col + 2 * i) : 0.0f, col + 2 * i + 1 < N ? fp8_bias<BIAS>(bias, col + 2 * i + 1) : 0.0f);
    }
}

// SPLITK: the CTAs of a cluster share one tile, each over K blocks of its own (ranges of kb_per_split in rank order); at the end every CTA is
// sent the other ones' sums of its share of the columns, adds them up in rank order and stores them.
template <int BN, int STAGES, bool PAIR, Fp8Bias BIAS, bool SPLITK = false>
__global__ void __launch_bounds__(kBlockwiseThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_y, const __grid_constant__ CUtensorMap map_out,
                const Fp8GemmParams p)
{
    static_assert(!(PAIR && SPLITK), "a cluster is a pair or a split");
    static_assert(BN == 256 || (!PAIR && (BN == 128 || BN == 64)), "tile widths");
    constexpr int NBUF = 512 / BN;            // partial buffers in tensor memory ...
    constexpr int SPLIT = BN == 256 ? 2 : 1;  // ... each in as many parts with an issuer and barriers of their own
    constexpr int DONE_RINGS = SPLIT;
    constexpr int NSUB = BN / SPLIT;          // N of one MMA
    constexpr int CW = BN / 2;                // columns per promotion warp: one half of the wide tile's buffer each, or half of the narrow one's
    constexpr int PART_WARPS = kPromoWarps / SPLIT;
    constexpr int CHW = CW < 64 ? 16 : 32;    // columns per tensor-memory load
    constexpr int NC = CW / CHW;
    static_assert(NC % 2 == 0, "a K block's first chunk goes to the same registers every time");
    constexpr int STORE_W = kFp8StoreCols;
    constexpr int kTileM = PAIR ? 2 * kBM : kBM;
    constexpr int kRowsB = PAIR ? BN / 2 : BN;
    constexpr uint32_t kBytesA = kBM * kBK, kBytesB = kRowsB * kBK, kStageBytes = kBytesA + kBytesB;
    constexpr uint32_t kTmemCols = 512;
    constexpr uint32_t kIdesc = make_idesc_e4m3(kTileM, NSUB);
    static_assert(STAGES >= NBUF, "a partial's barrier completes again only after its buffer has been handed back");
    static_assert(STAGES % 2 == 0 && NBUF % 2 == 0, "two issuers on alternate K blocks own their stages and buffers");

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    __shared__ __align__(8) uint64_t bar_full[STAGES];
    __shared__ __align__(8) uint64_t bar_done[DONE_RINGS][STAGES];
    __shared__ __align__(8) uint64_t bar_part_empty[SPLIT][NBUF];
    __shared__ __align__(8) uint64_t bar_scale_full[2];
    __shared__ __align__(8) uint64_t bar_scale_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ volatile uint32_t abort_flag;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int num_tiles = p.tiles_m * p.tiles_n;
    const int kb_all = (p.K + kBK - 1) / kBK;
    const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
    // K blocks kb_0 .. kb_0 + num_kb - 1 are this CTA's
    const uint32_t share = SPLITK ? cluster_cta_rank() : 0u;
    const int kb_0 = SPLITK ? static_cast<int>(share) * p.kb_per_split : 0;
    const int num_kb = SPLITK ? min(p.kb_per_split, kb_all - kb_0) : kb_all;
    const int first_tile = PAIR ? static_cast<int>(blockIdx.x >> 1) : static_cast<int>(blockIdx.x);
    const int tile_step = PAIR ? static_cast<int>(gridDim.x >> 1) : static_cast<int>(gridDim.x);

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) mbar_init(&bar_full[s], 1);
        for (int s = 0; s < 2; ++s) mbar_init(&bar_scale_full[s], 32), mbar_init(&bar_scale_empty[s], kPromoWarps);
        for (int h = 0; h < SPLIT; ++h) {
            for (int s = 0; s < STAGES; ++s) mbar_init(&bar_done[h][s], 1);
            for (int b = 0; b < NBUF; ++b) mbar_init(&bar_part_empty[h][b], PAIR ? 2 * PART_WARPS : PART_WARPS);
        }
        fence_barrier_init();
        prefetch_tensormap(&map_x);
        prefetch_tensormap(&map_y);
    }
    if (warp == 2) {
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
    const uint32_t stage_end = smem_u32(smem) + STAGES * kStageBytes;  // store staging, then the scales
    const uint32_t scales_0 = stage_end + kPromoWarps * kFp8StoreBytes;
    // A programmatic dependent waits here for the kernel in front.  Behind a quantiser, which writes only x and sa and has waited for what was in
    // front of it, the producer of the narrow tiles requests its first weights before it waits.
    const bool early_weights = BN < 256 && p.after_quant;
    if (!(early_weights && warp == 0)) pdl_wait();
    if (!p.release_late && threadIdx.x == 32) pdl_launch_dependents();  // (a thread of warp 1, which has waited)

    if (warp < 4) {
        setmaxnreg_dec<kFp8ControlRegs>();
        // Whole warps with uniform control flow; one lane is elected around the TMA, MMA and commit instructions only.
        if (warp == 0) {
            // -------------------------------------------------------------- TMA producer
            uint32_t s = 0, ph = 0, armed = 0;
            bool ok = true;
            int kb_early = 0;
            if constexpr (BN < 256) {
                if (early_weights) {
                    int mb, nb;
                    tile_coords(first_tile, p.tiles_m, p.tiles_n, mb, nb, p.group_m);
                    kb_early = min(num_kb, STAGES);
                    if (elect_one()) {
                        for (int kb = 0; kb < kb_early; ++kb) {
                            mbar_arrive_expect_tx(&bar_full[kb], kBytesB + p.box_rows * kBK);
                            tma_load_2d(smem + kb * kStageBytes + kBytesA, &map_y, &bar_full[kb], (kb_0 + kb) * kBK, nb * BN);
                        }
                    }
                    __syncwarp();
                    pdl_wait();
                    if (elect_one()) {
                        for (int kb = 0; kb < kb_early; ++kb) tma_load_2d(smem + kb * kStageBytes, &map_x, &bar_full[kb], (kb_0 + kb) * kBK, mb * kBM);
                    }
                    __syncwarp();
                    armed = static_cast<uint32_t>(kb_early);
                    s = armed;
                    if (s == STAGES) s = 0, ph ^= 1;
                }
            }
            for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
                int mb, nb;
                tile_coords(tile, p.tiles_m, p.tiles_n, mb, nb, p.group_m);
                for (int kb = tile == first_tile ? kb_early : 0; kb < num_kb; ++kb) {
                    const bool ready = wait_or_abort(&bar_done[0][s], ph ^ 1, &abort_flag) &&
                                       (DONE_RINGS == 1 || wait_or_abort(&bar_done[DONE_RINGS - 1][s], ph ^ 1, &abort_flag));
                    if (!warp_agrees(ready, p.status, &abort_flag, ERR_TIMEOUT_PRODUCER)) {
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        uint8_t* a_tile = smem + s * kStageBytes;
                        if constexpr (PAIR) {
                            // The leader arms its barrier for the bytes of both CTAs; the peer only sends bytes.
                            const uint32_t leader_full = map_to_cta(smem_u32(&bar_full[s]), 0);
                            if (rank == 0) mbar_arrive_expect_tx(&bar_full[s], 2 * kStageBytes);
                            tma_load_2d_pair(a_tile, &map_x, leader_full, kb * kBK, mb * kTileM + static_cast<int>(rank) * kBM);
                            // (64 rows of either half, so that a half of the partial is 128 neighbouring columns)
                            for (int h = 0; h < SPLIT; ++h)
                                tma_load_2d_pair(a_tile + kBytesA + h * (kBytesB / SPLIT), &map_y, leader_full, kb * kBK,
                                                 nb * BN + h * NSUB + static_cast<int>(rank) * (NSUB / 2));
                        } else {
                            mbar_arrive_expect_tx(&bar_full[s], kBytesB + p.box_rows * kBK);
                            tma_load_2d(a_tile, &map_x, &bar_full[s], (kb_0 + kb) * kBK, mb * kBM);
                            tma_load_2d(a_tile + kBytesA, &map_y, &bar_full[s], (kb_0 + kb) * kBK, nb * BN);
                        }
                    }
                    __syncwarp();
                    if (armed < STAGES) ++armed;
                    if (++s == STAGES) s = 0, ph ^= 1;
                }
            }
            drain_stages<STAGES, DONE_RINGS>(PAIR && rank != 0 ? nullptr : bar_full, bar_done[0], s, ph, armed, p.status, &abort_flag);
        } else if ((warp == 1 || warp == 3) && rank == 0) {
            // -------------------------------------------------------------- MMA issuers (PAIR: the leader's)
            // Wide tiles: each issues its half of every K block.  Narrow ones: alternate K blocks.
            const uint32_t me = warp == 1 ? 0u : 1u;
            constexpr uint32_t kStep = SPLIT == 2 ? 1u : 2u;
            const uint32_t h = SPLIT == 2 ? me : 0u;
            const uint32_t begin = SPLIT == 2 ? 0u : me;
            int my_tiles = 0;
            for (int tile = first_tile; tile < num_tiles; tile += tile_step) ++my_tiles;
            const uint32_t total = static_cast<uint32_t>(my_tiles) * static_cast<uint32_t>(num_kb);
            uint32_t s = begin, ph = 0, buf = begin, bph = 0;
            const uint32_t da_0 = smem_desc_lo(smem_u32(smem)), db_0 = smem_desc_lo(smem_u32(smem) + kBytesA + h * (kBytesB / SPLIT));
            const uint32_t full_0 = smem_u32(&bar_full[0]), done_0 = smem_u32(&bar_done[h][0]);
            const uint32_t empty_0 = smem_u32(&bar_part_empty[h][0]);
            for (uint32_t it = begin; it < total; it += kStep) {
                const bool ready = wait_or_abort_addr(full_0 + 8 * s, ph, &abort_flag) && wait_or_abort_addr(empty_0 + 8 * buf, bph ^ 1, &abort_flag);
                if (!warp_agrees(ready, p.status, &abort_flag, ERR_TIMEOUT_MMA)) break;
                const uint32_t tmem_d = tmem_base + buf * BN + h * NSUB;
                const uint32_t da = da_0 + s * (kStageBytes / 16), db = db_0 + s * (kStageBytes / 16);
                tcgen05_fence_after_sync();
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kBK / kUmmaK; ++k) {
                        if constexpr (PAIR) umma_f8_pair(tmem_d, smem_desc_k128_of(da + 2 * k), smem_desc_k128_of(db + 2 * k), kIdesc, k != 0 ? 1u : 0u);
                        else umma_f8(tmem_d, smem_desc_k128_of(da + 2 * k), smem_desc_k128_of(db + 2 * k), kIdesc, k != 0 ? 1u : 0u);
                    }
                    if constexpr (PAIR) {
                        umma_commit_pair(map_to_cta(done_0 + 8 * s, 0));
                        umma_commit_pair(map_to_cta(done_0 + 8 * s, 1));
                    } else {
                        umma_commit(&bar_done[h][s]);
                    }
                }
                __syncwarp();
                s += kStep;
                if (s >= STAGES) s -= STAGES, ph ^= 1;
                buf += kStep;
                if (buf >= NBUF) buf -= NBUF, bph ^= 1;
            }
        } else if (warp == 2) {
            // -------------------------------------------------------------- row scales
            // 64 bytes of every row of the tile at a time, by copies of 16 bytes where the rows of sa allow it.
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
                int mb, nb;
                tile_coords(tile, p.tiles_m, p.tiles_n, mb, nb, p.group_m);
                const int row0 = mb * kTileM + static_cast<int>(rank) * kBM;
                for (int kb = 0; kb < num_kb; kb += kFp8ScaleGroup) {
                    if (!warp_agrees(wait_or_abort(&bar_scale_empty[s], ph ^ 1, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_PRODUCER)) {
                        ok = false;
                        break;
                    }
                    const uint32_t dst = scales_0 + s * kFp8ScaleBytes;
                    if (p.scale_vec) {
                        const int c = lane & 3;
#pragma unroll 4
                        for (int r = lane >> 2; r < kBM; r += 8) {
                            const bool in = row0 + r < p.M && kb + 4 * c < num_kb;
                            cp_async_16(dst + fp8_scale_at(r, c), in ? p.sa + static_cast<int64_t>(row0 + r) * p.ld_sa + kb_0 + kb + 4 * c : p.sa, in ? 16u : 0u);
                        }
                    } else {
                        // Four times as many copies; scales that nobody uses (rows behind the last, columns behind num_kb) are read from the last row or column
                        // instead of being tested for at every copy (a K block of the 128-wide tile 369 -> 275 ns, of the 64-wide one 350 -> 230, next to 265 and 225
                        // with copies of 16 bytes; 1024 x 4736 x 6912 46.1 -> 34.2 us).
                        const int k = lane & 15, last = p.M - 1 - row0;
                        const float* src = p.sa + static_cast<int64_t>(row0) * p.ld_sa + kb_0 + min(kb + k, num_kb - 1);
#pragma unroll 4
                        for (int r = lane >> 4; r < kBM; r += 2)
                            cp_async_4(dst + fp8_scale_at(r, k >> 2) + (k & 3) * 4, src + static_cast<int64_t>(min(r, last)) * p.ld_sa);
                    }
                    cp_async_arrive(&bar_scale_full[s]);
                    s ^= 1;
                    if (s == 0) ph ^= 1;
                }
            }
            cp_async_wait_all();  // (no copy is under way when the CTA ends, whatever has failed)
        }
        if constexpr (SPLITK) {  // the two barriers of the split's exchange (a warp's lanes come together for them)
            __syncwarp();
            cluster_sync_all();
            cluster_sync_all();
        }
    } else {
        // ------------------------------------------------------------------ promotion + epilogue warps
        setmaxnreg_inc<kFp8PromoRegs>();
        const int quarter = warp & 3;
        const int cg = (warp - 4) >> 2;
        uint32_t tm_warp = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(cg * CW);
        GI8_PIN(tm_warp);
        const int part = SPLIT == 2 ? cg : 0;
        uint32_t part_0 = smem_u32(&bar_done[part][0]);
        uint32_t empty_0 = PAIR ? map_to_cta(smem_u32(&bar_part_empty[part][0]), 0) : smem_u32(&bar_part_empty[part][0]);
        GI8_PIN(part_0);
        GI8_PIN(empty_0);
        uint32_t buf = 0;           // partial buffer of the running K block
        uint32_t slot = 0, sph = 0;  // group of row scales and its phase
        uint32_t scale_row = fp8_scale_at(quarter * 32 + lane, 0);
        GI8_PIN(scale_row);
        uint32_t st = 0, ph = 0;    // its stage, whose barrier says that the partial is there, and the phase
        bool ok = true;
        // A wait that has failed does not end the tile (its results are invalid, and the waits that follow fail at once): with branches out of the loop
        // over the K blocks the compiler spilled accumulators in it.
        auto wait_partial = [&](bool ready) {
            if (!ready)
                ok &= warp_agrees(wait_or_abort_addr(part_0 + 8 * st, ph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_EPILOGUE);
            tcgen05_fence_after_sync();
        };
        auto release = [&] {
            tcgen05_fence_before_sync();
            __syncwarp();
            if constexpr (PAIR) {
                if (elect_one()) mbar_arrive_cluster(empty_0 + 8 * buf);
            } else {
                mbar_arrive_elected_addr(empty_0 + 8 * buf);
            }
            if (++buf == NBUF) buf = 0;
            if (++st == STAGES) st = 0, ph ^= 1;
        };
        for (int tile = first_tile; tile < num_tiles && ok; tile += tile_step) {
            uint64_t acc[CW / 2];
#pragma unroll
            for (int j = 0; j < CW / 2; ++j) acc[j] = 0ull;
            int mb, nb;
            tile_coords(tile, p.tiles_m, p.tiles_n, mb, nb, p.group_m);
            const int col_base = nb * BN + cg * CW;  // (inside one 128-wide weight-scale block)
            // 32-bit element offset (the host checks the array's size)
            uint32_t sw = static_cast<uint32_t>(col_base < p.N ? col_base / 128 : 0) * static_cast<uint32_t>(p.ld_sw) + static_cast<uint32_t>(kb_0);
            GI8_PIN(sw);
            // The row's scales of this K block and those behind it in its four; the weight block's: a lane each, for 32 K blocks.
            float a[4];
            auto load_rows = [&](int kb) {
                const int c = (kb >> 2) & 3;
                if (c == 0) ok &= warp_agrees(wait_or_abort(&bar_scale_full[slot], sph, &abort_flag), p.status, &abort_flag, ERR_TIMEOUT_EPILOGUE);
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(a[0]), "=f"(a[1]), "=f"(a[2]), "=f"(a[3])
                             : "r"(scales_0 + slot * kFp8ScaleBytes + (scale_row ^ (c * 16)))
                             : "memory");
                if (c == 3 || kb + 4 >= num_kb) {
                    __syncwarp();
                    mbar_arrive_elected_addr(smem_u32(&bar_scale_empty[slot]));
                    slot ^= 1;
                    if (slot == 0) sph ^= 1;
                }
            };
            load_rows(0);
            float b32 = ldg_in_place(p.sw + (sw + min(lane, num_kb - 1)));
            float b = __shfl_sync(0xffffffffu, b32, 0);
            uint32_t v[2][CHW];
            wait_partial(false);
            tmem_ld(tm_warp + buf * BN, v[0]);
            // A K block's first chunk is on its way into v[0].  The next chunk's load runs under this one's arithmetic, the buffer goes back as soon as its
            // last chunk has landed, and the next K block's first chunk is requested before the last one's arithmetic.
#pragma unroll 1
            for (int kb = 0; kb < num_kb; ++kb) {
                const float t = mul_in_place(a[0], b);
                a[0] = a[1], a[1] = a[2], a[2] = a[3];
                if ((kb & 3) == 3) {
                    if (kb + 1 < num_kb) load_rows(kb + 1);
                    if ((kb & 31) == 31) b32 = ldg_in_place(p.sw + (sw + min(kb + 1 + lane, num_kb - 1)));
                }
                b = __shfl_sync(0xffffffffu, b32, (kb + 1) & 31);
                bool ready = false;
                const uint64_t t2 = f32x2(t, t);
                auto accumulate = [&](const uint32_t (&r)[CHW], int c) {
#pragma unroll
                    for (int q = 0; q < CHW / 2; ++q) promote_pair_f32(acc[c * (CHW / 2) + q], r[2 * q], r[2 * q + 1], t2);
                };
                tmem_ld_wait();
#pragma unroll
                for (int c = 0; c + 1 < NC; ++c) {
                    const int cur = c & 1;
                    tmem_ld(tm_warp + buf * BN + (c + 1) * CHW, v[cur ^ 1]);
                    // (the next K block's partial, tested here so that the answer is there when it is needed)
                    if (c + 2 == NC) {
                        const uint32_t next = st + 1 == STAGES ? 0 : st + 1;
                        ready = __all_sync(0xffffffffu, mbar_test_wait_addr(part_0 + 8 * next, next == 0 ? ph ^ 1 : ph));
                    }
                    accumulate(v[cur], c);
                    tmem_ld_wait();
                }
                release();
                if (kb + 1 < num_kb) {
                    wait_partial(ready);
                    tmem_ld(tm_warp + buf * BN, v[0]);
                }
                accumulate(v[1], NC - 1);
            }
            if (!SPLITK && !ok) break;  // (a split tile's CTAs meet below whatever has failed)

            // Blocks of 32 rows x STORE_W columns through swizzled shared memory and TMA stores, or row by row where TMA cannot address the rows.
            // (The tile's coordinates again, from an opaque copy, so that they occupy no registers across the loop.)
            int tile_again = tile, mb2, nb2;
            asm volatile("" : "+r"(tile_again));
            tile_coords(tile_again, p.tiles_m, p.tiles_n, mb2, nb2, p.group_m);
            const int row0 = mb2 * kTileM + static_cast<int>(rank) * kBM + quarter * 32;
            const uint32_t stg = stage_end + (warp - 4) * kFp8StoreBytes;
            // A staged block (32 rows x 32 columns, written by this warp) to the output.
            auto store_block = [&](int col0) {
                if (!p.tma_store) {
                    __syncwarp();
                    store_staged_rows<STORE_W>(stg, static_cast<uint16_t*>(p.out), p.ldo, row0, p.M, col0, p.N, p.pair_ok);
                    return;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&map_out, reinterpret_cast<const void*>(__cvta_shared_to_generic(stg)), col0, row0);
                    tma_store_commit();
                }
            };
            if constexpr (SPLITK) {
                // The sums meet in the stages, which no CTA of the cluster uses any more behind the first barrier: for each sender and 32 columns of the
                // receiver's share, four columns of all rows after each other, so that a warp's store is one run of 512 bytes.  They are added up in a loop
                // that is not unrolled: this code runs once, and what it costs is fetching it (unrolled, with the own sums from registers, 64 columns took
                // 8000 cycles).
                const int share_cols = BN / p.splits;
                const uint32_t recv = smem_u32(smem), r = static_cast<uint32_t>(quarter * 32 + lane);
                cluster_sync_all();
#pragma unroll
                for (int b = 0; b < CW / 32; ++b) {
                    if (row0 >= p.M) break;  // (rows that nobody stores)
                    const int c = cg * CW + b * 32, owner = c / share_cols;
                    const uint32_t at = map_to_cta(recv + ((share * share_cols + (c - owner * share_cols)) / 4 * kBM + r) * 16, owner);
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        asm volatile("st.shared::cluster.v2.b64 [%0], {%1, %2};" ::"r"(at + q * (kBM * 16)), "l"(acc[b * 16 + 2 * q]), "l"(acc[b * 16 + 2 * q + 1]) : "memory");
                }
                cluster_sync_all();
                if (row0 < p.M) {
#pragma unroll 1
                    for (int c = cg * 32; c < share_cols; c += 64) {
                        const int col0 = nb2 * BN + static_cast<int>(share) * share_cols + c;
                        if (col0 >= p.N) break;
                        if (p.tma_store && lane == 0) tma_store_wait_read<0>();
                        __syncwarp();
#pragma unroll 1
                        for (int q = 0; q < 8; ++q) {
                            uint64_t sum[2] = {0ull, 0ull};
                            uint32_t at = recv + ((c / 4 + q) * kBM + r) * 16;
#pragma unroll 1
                            for (int src = 0; src < p.splits; ++src, at += share_cols / 4 * kBM * 16) {  // in the order of the K blocks
                                uint64_t v0, v1;
                                asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(v0), "=l"(v1) : "r"(at) : "memory");
                                sum[0] = add2(sum[0], v0), sum[1] = add2(sum[1], v1);
                            }
                            if constexpr (BIAS != Fp8Bias::kNone) {
                                float w[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) w[j] = col0 + 4 * q + j < p.N ? fp8_bias<BIAS>(p.bias, col0 + 4 * q + j) : 0.0f;
                                sum[0] = add2(sum[0], f32x2(w[0], w[1])), sum[1] = add2(sum[1], f32x2(w[2], w[3]));
                            }
                            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(stg + lane * (STORE_W * 2) + (((q >> 1) ^ ((lane >> 1) & 3)) * 16) + (q & 1) * 8),
                                         "r"(pack_bf16x2_of(sum[0])), "r"(pack_bf16x2_of(sum[1]))
                                         : "memory");
                        }
                        store_block(col0);
                    }
                }
            }
            if (!SPLITK && row0 < p.M) {
#pragma unroll
                for (int b = 0; b < CW / STORE_W; ++b) {
                    const int col0 = nb2 * BN + cg * CW + b * STORE_W;
                    if (col0 >= p.N) continue;  // warp-uniform
                    if (p.tma_store && lane == 0) tma_store_wait_read<0>();  // the previous block has been read out of the staging
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < STORE_W / 8; ++q) {
                        const int cq = q ^ ((lane >> 1) & 3);
                        const int a0 = b * (STORE_W / 2) + 4 * q;
                        if constexpr (BIAS != Fp8Bias::kNone) {
                            uint64_t w[4];
                            fp8_bias8<BIAS>(p.bias, col0 + 8 * q, p.N, p.bias_vec, w);
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[a0 + j] = add2(acc[a0 + j], w[j]);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stg + lane * (STORE_W * 2) + cq * 16), "r"(pack_bf16x2_of(acc[a0])),
                                     "r"(pack_bf16x2_of(acc[a0 + 1])), "r"(pack_bf16x2_of(acc[a0 + 2])), "r"(pack_bf16x2_of(acc[a0 + 3]))
                                     : "memory");
                    }
                    store_block(col0);
                }
            }
            __syncwarp();
        }
        if (lane == 0) tma_store_wait_all<0>();  // stores read this CTA's shared memory: finish before exit
    }

    tcgen05_fence_before_sync();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();  // neither CTA leaves while the other may still read or signal it
    if (warp == 2) {
        __syncwarp();
        tcgen05_fence_after_sync();
        if constexpr (PAIR) tmem_dealloc_pair(tmem_base, kTmemCols);
        else tmem_dealloc(tmem_base, kTmemCols);
    }
}

}  // namespace gi8
