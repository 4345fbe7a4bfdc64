// Block-scale FP8 GEMM for skinny M (decode shapes, M <= 32): C[m,n] = sum_kb (A @ B^T)[kb] * sa[m,kb] * sb[kb,n/128],
// optionally c_a * that + c_b.
//
// The weight stream B[N,K] should bound it.  The block-scale kernel of gemm_fp8.cu does not get there: 128-column tiles
// leave SMs idle (N = 14336: 112 tiles on 148 SMs), its TMA fetches 128 rows of A of which M exist, and all accumulators
// of up to 32 tokens sit in the registers of one warp.  So the operands trade places:
//
//  * The weights are the MMA's 128 rows, the tokens (16 or 32) its N columns.  Eight epilogue warps promote a partial
//    product with one weight row and half of the tokens per thread.
//  * N is cut into 16-row units that are dealt out as (rounds) x (number of SMs) tiles of up to 128 rows; a tile's rows
//    come with ONE TMA box of exactly that height (two tensor maps: base and base + 1 units).  A tile may straddle two
//    128-row scale groups: each thread picks its row's group.
//  * Staging warps transpose the activation scales, eight K blocks at a time, into shared memory ([K block][token]), where
//    the epilogue reads them as broadcasts.
//  * What bounds it is the MMA thread and the hand-off, at about 0.3 us per K block and tile with one K block per
//    stage and two commits for each.  So a stage holds two K blocks, one commit publishes both partial products, and the
//    epilogue returns the operands: 24 x 14336 x 4096 takes 16.2 us, 18.0 with one K block per stage (and 20.3 with four
//    instead of eight epilogue warps; the MMAs of two K blocks interleaved: no difference).
//
// Every K block is promoted in order with the same fused multiply-adds as in the large kernel, so the two give the same
// bits.  Cold L2, us, large kernel / this one: 24 x 14336 x 4096 24.8 / 16.2, 32 x 28672 x 8192 53.8 / 44.7 (5.3 TB/s),
// 16 x 57344 x 4096 75.2 / 39.5 (6.0 TB/s), 32 x 1024 x 8192 26.8 / 20.3, 8 x 4096 x 4096 16.0 / 11.3, 1 x 1024 x 1024
// 7.9 / 6.0.  With multiply-add, quantizer included: 17 x 1024 x 1024 19.5 / 13.3, 17 x 4096 x 4096 27.6 / 19.5,
// 17 x 28672 x 8192 78.9 / 62.5 (c_a and c_b loaded token by token behind the stores instead: 21.5, 27.7, 76.8).  With 64
// tokens the epilogue's scale reads take over (64 x 28672 x 8192 57.4 / 64.6): those stay there.
//
// Gated (kOut == 2): a tile is up to 64 output columns, its MMA rows the gate rows of those columns and behind them the up rows (two
// boxes).  Behind the last K block the threads of the up rows hand their sums to those of the gate rows through shared memory.
//
// Split K (kSplitK, kOut 1 and 2): one tile of a narrow layer is a long chain of K steps on a few SMs.  There a cluster of 2, 4 or 8 CTAs
// shares a tile, each with a part of K; at the end all write their sums into the first one's (by then idle) operand ring through
// distributed shared memory and it adds them in rank order, so the result is the same every time.  The two cluster barriers around
// that are reached by every thread on every path, an abandoned wait included.  plan_split() below has the rule.
//
// Roles: warp 0 TMA producer, warp 1 TMEM allocator + MMA issuer, warps 2-9 epilogue, warps 10-11 scale staging.  Bounded
// waits and teardown as in gemm_fp8.cu.
#include "activation.cuh"
#include "tc_common.cuh"

namespace hkb {
namespace {

constexpr int kMaxStages = 16;
constexpr int kStep = 2;                  // K blocks per pipeline stage, hand-off and commit
constexpr int kAccs = 8;                  // accumulator sets in TMEM, kStep partial products of 32 columns each
constexpr int kSlots = 4;                 // ring of staged scales
constexpr int kChunk = 8;                 // K blocks per slot
constexpr int kPitch = 36;                // floats per K block: 32 token scales, then the weight scales of two groups (gated: two of gate, two of up)
constexpr int kSlotBytes = kChunk * kPitch * 4;
constexpr int kHeadBytes = 1024 * ((1024 + kSlots * kSlotBytes + 1023) / 1024);      // barriers (first KB), then the scale ring
constexpr int kXchgPitch = 65;            // gated: up sums [token][64 rows], one float of padding
constexpr int kXchgBytes = 9 * 1024;
static_assert(32 * kXchgPitch * 4 <= kXchgBytes, "exchange area");
constexpr int kTailPad = 16 * 1024;       // the MMA reads 128 weight rows from every stage base
constexpr int kSmemLimit = 232448;        // 227 KB
constexpr int kMaxUnits = 8;              // 128 weight rows
constexpr int kEpiWarps = 8;             // two per TMEM lane quarter, half of the token columns each
constexpr int kThreads = 32 * (4 + kEpiWarps);

struct BsSkinnyParams {
    int M, N, K;
    int64_t ldc;
    int a_box_rows;                       // rows of A fetched per stage (multiple of 8, <= 32)
    int split;                            // CTAs per tile (cluster size); above 1 every cluster has exactly one tile
    int tiles, base, rem;                 // tile t is base + (t < rem) units high and starts at unit t*base + min(t, rem)
    int stages, sub_bytes, a_off;         // one K block inside a stage; its activation rows
    const float* sa;
    const float* sb;
    __nv_bfloat16* C;
    const __nv_bfloat16* c_a;             // fused multiply-add (both [M, N]), or null
    const __nv_bfloat16* c_b;
    const __nv_bfloat16* bias;            // kOut == 1: act(gemm + bias[n]) + residual[m, n], either null
    const __nv_bfloat16* residual;
    int act;                              // kOut == 1, 2
    float* f32;                           // kOut == 2: the result [M, N] in fp32 instead of C, or null
    uint32_t* status;
};

// 8 consecutive fp32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
#define TILE_UNITS(t) (p.base + ((t) < p.rem ? 1 : 0))
#define TILE_ROW0(t) (((t) * p.base + min((t), p.rem)) * 16)

// NT: token columns (16 or 32).  kOut: 0 plain / multiply-add, 1 bias + activation + residual, 2 gated (p.N output columns, B has 2N rows).
template <int NT, int kOut, bool kSplitK = false>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_blockscale_skinny_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB0,
                                  const __grid_constant__ CUtensorMap tmB1, const BsSkinnyParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t bar_base = smem_u32(smem);
    const uint32_t ring_base = bar_base + kHeadBytes + (kOut == 2 ? kXchgBytes : 0);
    float* const xchg = reinterpret_cast<float*>(smem + kHeadBytes);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kMaxStages + s); };
    auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * kMaxStages + a); };
    auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * kMaxStages + kAccs + a); };
    auto sfull_bar = [&](int i) { return bar_base + 8u * (2 * kMaxStages + 2 * kAccs + i); };
    auto sempty_bar = [&](int i) { return bar_base + 8u * (2 * kMaxStages + 2 * kAccs + kSlots + i); };
    auto xfull_bar = [&](int i) { return bar_base + 8u * (2 * kMaxStages + 2 * kAccs + 2 * kSlots + i); };       // gated: 0 written, 1 read
    constexpr bool kGated = kOut == 2;
    constexpr int kNumBars = 2 * kMaxStages + 2 * kAccs + 2 * kSlots + 2;
    static_assert(kNumBars * 8 + 8 <= 1024, "barrier area");
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + kNumBars * 8);
    volatile uint32_t* abort_flag = tmem_slot + 1;
    float* const scales = reinterpret_cast<float*>(smem + 1024);          // [kSlots][kChunk][kPitch]
    constexpr uint32_t TMEM_COLS = 512;

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int all_kblocks = p.K / 128;
    const int all_ksteps = (all_kblocks + kStep - 1) / kStep;       // an odd last block is followed by zero-filled data and zero scales
    const int split = kSplitK ? p.split : 1;
    const int rank = kSplitK ? (int)cluster_ctarank() : 0;
    const int ks0 = all_ksteps * rank / split;                      // this CTA's part of K: whole steps, the odd block stays last
    const int ksteps = all_ksteps * (rank + 1) / split - ks0;
    const int kblock0 = ks0 * kStep;
    const int kblocks = min(ksteps * kStep, all_kblocks - kblock0);
    const int tile0 = kSplitK ? (int)blockIdx.x / split : (int)blockIdx.x;
    const int tile_step = kSplitK ? (int)gridDim.x / split : (int)gridDim.x;
    const uint32_t stage_bytes = kStep * p.sub_bytes;
    const int nchunks = (kblocks + kChunk - 1) / kChunk;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < kAccs; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), kEpiWarps);
        }
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(sfull_bar(i), 1);
            mbar_init(sempty_bar(i), kEpiWarps);
        }
        for (int i = 0; i < 2; ++i) mbar_init(xfull_bar(i), kEpiWarps);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), TMEM_COLS);
    if constexpr (kOut != 0) {
        // The first ring of weights goes towards L2 while the kernel ahead still runs.  16 layers in turn, so that the weights are cold, us:
        // gated 1 x 4096 x 2048 8.7 -> 8.3, 1 x 1024 x 8192 9.5 -> 9.1, linear 16 x 4096 x 4096 8.6 -> 8.2, 16 x 4096 x 14336 15.2 -> 14.6 (with
        // weights that are in L2 already the prefetch itself shows: gated 1 x 4096 x 2048 7.1 -> 7.4).
        if (warp == 0 && tile0 < p.tiles && elect_one()) {
            const CUtensorMap* const tmB = tile0 < p.rem ? &tmB1 : &tmB0;
            for (int kb = 0; kb < min(p.stages * kStep, kblocks); ++kb) {
                tma_prefetch_3d(tmB, (kblock0 + kb) * 128, TILE_ROW0(tile0), 0);
                if constexpr (kOut == 2) tma_prefetch_3d(tmB, (kblock0 + kb) * 128, p.N + TILE_ROW0(tile0), 0);
            }
        }
        __syncwarp();
    }
    pdl_wait();      // nothing in global memory is read or written before this; the prefetch above is a hint to L2 only
    tc_fence_before();
    __syncthreads();
    if constexpr (kOut != 0) pdl_trigger();  // the launch behind this one sets up while this one computes: 1 x 1024 x 1024 4.5 -> 4.0 us
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0) {
        if (elect_one()) {
            prefetch_tmap(&tmA);
            prefetch_tmap(&tmB0);
            prefetch_tmap(&tmB1);
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = tile0; t < p.tiles && ok; t += tile_step) {
                const CUtensorMap* const tmB = t < p.rem ? &tmB1 : &tmB0;
                const int n0 = TILE_ROW0(t);
                const uint32_t b_bytes = (uint32_t)TILE_UNITS(t) * 2048;
                const uint32_t stage_tx = kStep * ((uint32_t)p.a_box_rows * 128 + (kGated ? 2 : 1) * b_bytes);
                for (int ks = 0; ks < ksteps; ++ks) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1, abort_flag, p.status, kErrWaitProducer)) { ok = false; break; }
                    mbar_arrive_expect_tx(full_bar(s), stage_tx);
                    const uint32_t st = ring_base + s * stage_bytes;
#pragma unroll
                    for (int i = 0; i < kStep; ++i) {
                        tma_load_3d(st + i * p.sub_bytes, tmB, full_bar(s), (kblock0 + ks * kStep + i) * 128, n0, 0);
                        if constexpr (kGated) tma_load_3d(st + i * p.sub_bytes + b_bytes, tmB, full_bar(s), (kblock0 + ks * kStep + i) * 128, p.N + n0, 0);
                        tma_load_3d(st + i * p.sub_bytes + p.a_off, &tmA, full_bar(s), (kblock0 + ks * kStep + i) * 128, 0, 0);
                    }
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            constexpr uint32_t IDESC = idesc_f8(128, NT);
            int s = 0;
            uint32_t ph = 0;
            int acc = 0;
            uint32_t acc_ph = 0;
            bool ok = true;
            for (int t = tile0; t < p.tiles && ok; t += tile_step) {
                for (int ks = 0; ks < ksteps; ++ks) {
                    if (!mbar_wait(full_bar(s), ph, abort_flag, p.status, kErrWaitMma)) { ok = false; break; }
                    if (!mbar_wait(tempty_bar(acc), acc_ph ^ 1, abort_flag, p.status, kErrWaitMma)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t st = ring_base + s * stage_bytes;
                    const uint64_t dw = smem_desc_sw128(st);
                    const uint64_t dx = smem_desc_sw128(st + p.a_off);
                    const uint64_t sub = (uint64_t)(p.sub_bytes >> 4);
                    const uint32_t d = tmem_base + acc * (kStep * 32);
#pragma unroll
                    for (int i = 0; i < kStep; ++i)
#pragma unroll
                        for (int k = 0; k < 4; ++k) mma_f8(d + i * 32, dw + i * sub + (uint64_t)(k * 2), dx + i * sub + (uint64_t)(k * 2), IDESC, k != 0);
                    tc_commit(tfull_bar(acc));              // the only commit: the epilogue hands the stage back
                    if (++acc == kAccs) { acc = 0; acc_ph ^= 1; }
                    if (++s == p.stages) { s = 0; ph ^= 1; }
                }
            }
        }
    } else if (warp < 2 + kEpiWarps) {
        // ================= epilogue: one weight row per thread =================
        constexpr int NC = NT / 2;                           // token columns of this warp: col0 .. col0 + NC - 1
        const int col0 = ((warp - 2) >> 2) * NC;
        const int quarter = warp & 3;
        const int row_in_tile = quarter * 32 + lane;
        const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
        int acc = 0, slot = 0, s = 0;
        uint32_t acc_ph = 0, slot_ph = 0, x_ph = 0;
        bool ok = true;
        for (int t = tile0; t < p.tiles && ok; t += tile_step) {
            const int cols = TILE_UNITS(t) * 16;                         // output columns of the tile
            const int rows = kGated ? 2 * cols : cols;
            const int n0 = TILE_ROW0(t);
            const bool row_ok = row_in_tile < rows;
            const bool warp_has_rows = quarter * 32 < rows;              // warp-uniform
            const bool is_up = kGated && row_in_tile >= cols;
            const int n = n0 + (row_ok ? row_in_tile - (is_up ? cols : 0) : 0);
            const int group = (n >> 7) - (n0 >> 7) + (is_up ? 2 : 0);    // 0 or 1; gated: 2 or 3 for the up rows
            if constexpr (kOut == 1) {
                if (p.residual && warp_has_rows && lane < NC && col0 + lane < p.M)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(p.residual + (int64_t)(col0 + lane) * p.N + n0 + quarter * 32));
            }
            if (kOut == 0 && p.c_a && warp_has_rows && col0 + (lane & (NC - 1)) < p.M) {      // this warp's part of c_a and c_b, into L2
                const int64_t off = (int64_t)(col0 + (lane & (NC - 1))) * p.N + n0 + quarter * 32;
                asm volatile("prefetch.global.L2 [%0];" ::"l"((lane < 16 ? p.c_a : p.c_b) + off));
            }
            float2 acc2[NC / 2];
#pragma unroll
            for (int j = 0; j < NC / 2; ++j) acc2[j] = make_float2(0.0f, 0.0f);
            for (int ch = 0; ch < nchunks && ok; ++ch) {
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(sfull_bar(slot), slot_ph, abort_flag, p.status, kErrWaitEpilogue))) { ok = false; break; }
                const int ks_end = min(ksteps - ch * (kChunk / kStep), kChunk / kStep);
                for (int kk = 0; kk < ks_end; ++kk) {
                    const float* const sc = scales + (slot * kChunk + kk * kStep) * kPitch;
                    // the scales come before the wait, so that their latency passes with it
                    float2 f[kStep][NC / 2];
#pragma unroll
                    for (int i = 0; i < kStep; ++i) {
                        const float sb = sc[i * kPitch + 32 + group];
                        const float2 sb2 = make_float2(sb, sb);
#pragma unroll
                        for (int j = 0; j < NC; j += 4) {
                            const float4 s4 = *reinterpret_cast<const float4*>(sc + i * kPitch + col0 + j);
                            f[i][j / 2] = __fmul2_rn(make_float2(s4.x, s4.y), sb2);
                            f[i][j / 2 + 1] = __fmul2_rn(make_float2(s4.z, s4.w), sb2);
                        }
                    }
                    if (!__all_sync(0xFFFFFFFFu, mbar_wait(tfull_bar(acc), acc_ph, abort_flag, p.status, kErrWaitEpilogue))) { ok = false; break; }
                    if (warp == 2 && lane == 0) mbar_arrive(empty_bar(s));       // these MMAs are done with their operands
                    if (++s == p.stages) s = 0;
                    tc_fence_after();
                    uint32_t r[kStep][NC];
                    if (warp_has_rows) {
                        const uint32_t t_addr = tmem_base + lane_addr + acc * (kStep * 32) + col0;
#pragma unroll
                        for (int i = 0; i < kStep; ++i)
#pragma unroll
                            for (int c = 0; c < NC; c += 16) {
                                if constexpr (NC % 16) tmem_ld8(t_addr + i * 32 + c, r[i] + c);
                                else tmem_ld16(t_addr + i * 32 + c, *reinterpret_cast<uint32_t(*)[16]>(r[i] + c));
                            }
                        tmem_ld_wait();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(tempty_bar(acc));
                    if (++acc == kAccs) { acc = 0; acc_ph ^= 1; }
                    if (warp_has_rows) {
#pragma unroll
                        for (int i = 0; i < kStep; ++i)
#pragma unroll
                            for (int j = 0; j < NC; j += 2)
                                acc2[j / 2] = __ffma2_rn(make_float2(__uint_as_float(r[i][j]), __uint_as_float(r[i][j + 1])), f[i][j / 2], acc2[j / 2]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sempty_bar(slot));
                if (++slot == kSlots) { slot = 0; slot_ph ^= 1; }
            }
            if constexpr (kSplitK) {
                {
                    __syncwarp();
                    cluster_sync_all();                    // every CTA of the cluster is done with its operand ring
                    const uint32_t slot0 = ring_base + (uint32_t)(col0 * 128 + row_in_tile) * 4;        // [rank - 1][token][row]
                    if (ok && rank != 0 && warp_has_rows) {
                        const uint32_t dst = cluster_addr(slot0 + (uint32_t)(rank - 1) * (NT * 512), 0);
#pragma unroll
                        for (int j = 0; j < NC; ++j) st_cluster(dst + j * 512, (j & 1) ? acc2[j / 2].y : acc2[j / 2].x);
                    }
                    __syncwarp();
                    cluster_sync_all();
                    if (rank != 0) break;                  // the only tile of this cluster
                    if (warp_has_rows) {
                        const float* const part = reinterpret_cast<const float*>(smem + (slot0 - bar_base));
                        for (int r = 0; r < split - 1; ++r) {
#pragma unroll
                            for (int j = 0; j < NC; ++j) {
                                const float v = part[(r * NT + j) * 128];
                                if (j & 1) acc2[j / 2].y += v; else acc2[j / 2].x += v;
                            }
                        }
                    }
                }
            }
            if constexpr (kGated) {
                // the up sums change hands: written, all eight warps arrive, read by the gate rows, all arrive before the next tile writes
                float* const xr = xchg + col0 * kXchgPitch + (n - n0);
                if (ok && !__all_sync(0xFFFFFFFFu, mbar_wait(xfull_bar(1), x_ph ^ 1, abort_flag, p.status, kErrWaitEpilogue))) ok = false;
                if (!ok) break;
                if (row_ok && is_up) {
#pragma unroll
                    for (int j = 0; j < NC; ++j) xr[j * kXchgPitch] = (j & 1) ? acc2[j / 2].y : acc2[j / 2].x;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(xfull_bar(0));
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(xfull_bar(0), x_ph, abort_flag, p.status, kErrWaitEpilogue))) { ok = false; break; }
                float v[NC], up[NC];
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    v[j] = (j & 1) ? acc2[j / 2].y : acc2[j / 2].x;
                    up[j] = row_ok && !is_up ? xr[j * kXchgPitch] : 0.0f;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(xfull_bar(1));
                x_ph ^= 1;
                if (row_ok && !is_up) {
                    apply_act<NC>(v, p.act);
#pragma unroll
                    for (int j = 0; j < NC; ++j) {
                        if (col0 + j >= p.M) break;
                        if (p.f32) p.f32[(int64_t)(col0 + j) * p.N + n] = v[j] * up[j];
                        else p.C[(int64_t)(col0 + j) * p.ldc + n] = __float2bfloat16_rn(v[j] * up[j]);
                    }
                }
            } else if (ok && row_ok) {
                float v[NC];
#pragma unroll
                for (int j = 0; j < NC; ++j) v[j] = (j & 1) ? acc2[j / 2].y : acc2[j / 2].x;
                if constexpr (kOut == 1) {
                    float res[NC];                  // loaded together and ahead of the stores, for the same reason
#pragma unroll
                    for (int j = 0; j < NC; ++j) res[j] = p.residual ? __bfloat162float(p.residual[(int64_t)min(col0 + j, p.M - 1) * p.N + n]) : 0.0f;
                    const float bn = p.bias ? __bfloat162float(p.bias[n]) : 0.0f;
#pragma unroll
                    for (int j = 0; j < NC; ++j) v[j] += bn;
                    apply_act<NC>(v, p.act);
#pragma unroll
                    for (int j = 0; j < NC; ++j) v[j] += res[j];
                }
                if (kOut == 0 && p.c_a) {
                    // All loads go out before the first store: C may be c_a or c_b, so the compiler cannot move them up, and one
                    // round trip per token is longer than the whole K loop of a small layer.
                    __nv_bfloat16 ca[NC], cb[NC];
#pragma unroll
                    for (int j = 0; j < NC; ++j) {
                        const int64_t off = (int64_t)min(col0 + j, p.M - 1) * p.N + n;
                        ca[j] = p.c_a[off];
                        cb[j] = p.c_b[off];
                    }
#pragma unroll
                    for (int j = 0; j < NC; ++j) v[j] = __fmaf_rn(__bfloat162float(ca[j]), v[j], __bfloat162float(cb[j]));
                }
#pragma unroll
                for (int j = 0; j < NC; ++j)
                    if (col0 + j < p.M) p.C[(int64_t)(col0 + j) * p.ldc + n] = __float2bfloat16_rn(v[j]);
            }
        }
    } else {
        // ================= scale staging: warp g fills every second slot =================
        const int g = warp - 2 - kEpiWarps;
        const int nsb = p.N / 128;                           // gated: of gate and of up
        const bool vec = (all_kblocks & 3) == 0 && (kblock0 & 3) == 0 && (reinterpret_cast<uintptr_t>(p.sa) & 15) == 0;
        int slot = g, ch = g;                                // ch: chunk of the tile, in the epilogue's order
        uint32_t ph = 0;
        bool ok = true;
        for (int t = tile0; t < p.tiles && ok; t += tile_step) {
            const int g0 = TILE_ROW0(t) >> 7;
            for (; ch < nchunks; ch += 2) {
                const int kb0 = ch * kChunk;
                const int kn = min(kblocks - kb0, kChunk);
                float v[kChunk];
                const float* const src = p.sa + (int64_t)lane * all_kblocks + kblock0 + kb0;
#pragma unroll
                for (int k = 0; k < kChunk; k += 4) {
                    if (lane < p.M && vec && k + 4 <= kn) {
                        const float4 f = __ldg(reinterpret_cast<const float4*>(src + k));
                        v[k] = f.x; v[k + 1] = f.y; v[k + 2] = f.z; v[k + 3] = f.w;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[k + i] = (lane < p.M && k + i < kn) ? __ldg(src + k + i) : 0.0f;
                    }
                }
                // two weight scales per K block (gated: two of gate, two of up)
                constexpr int W = kGated ? 4 : 2;
                const int wk = lane / W, wi = lane % W, wg = min(g0 + (wi & 1), nsb - 1) + (wi >> 1) * nsb;
                const float wsc = wk < kn ? __ldg(p.sb + (int64_t)(kblock0 + kb0 + wk) * (W / 2 * nsb) + wg) : 0.0f;
                if (!__all_sync(0xFFFFFFFFu, mbar_wait(sempty_bar(slot), ph ^ 1, abort_flag, p.status, kErrWaitProducer))) { ok = false; break; }
                float* const dst = scales + slot * kChunk * kPitch;
#pragma unroll
                for (int k = 0; k < kChunk; ++k) dst[k * kPitch + lane] = v[k];
                if (wk < kChunk) dst[wk * kPitch + 32 + wi] = wsc;
                __syncwarp();
                if (lane == 0) mbar_arrive(sfull_bar(slot));
                slot += 2;
                if (slot >= kSlots) { slot -= kSlots; ph ^= 1; }
            }
            ch -= nchunks;
        }
    }

    if constexpr (kSplitK) {
        if ((warp < 2 || warp >= 2 + kEpiWarps)) {            // the epilogue warps' two cluster barriers, reached by everyone
            __syncwarp();
            cluster_sync_all();
            cluster_sync_all();
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (*abort_flag) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

#undef TILE_UNITS
#undef TILE_ROW0

template <int NT, int kOut, bool kSplitK = false>
int launch(const CUtensorMap& tmA, const CUtensorMap& tmB0, const CUtensorMap& tmB1, const BsSkinnyParams& p, int smem, int grid, cudaStream_t st) {
    // the limit is the kernel's, not the call's: every call sets the same one, whatever its own size (calls may overlap)
    auto kern = gemm_fp8_blockscale_skinny_kernel<NT, kOut, kSplitK>;
    HKB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit));
    note_kernel(kOut == 0 ? "gemm_fp8_blockscale_skinny_kernel" :
                kOut == 1 ? (kSplitK ? "gemm_fp8_blockscale_skinny_kernel<epilogue,split>" : "gemm_fp8_blockscale_skinny_kernel<epilogue>")
                          : (kSplitK ? "gemm_fp8_blockscale_skinny_kernel<gated,split>" : "gemm_fp8_blockscale_skinny_kernel<gated>"));
    HKB_CUDA(launch_dependent(true, kern, grid, kThreads, smem, kSplitK ? p.split : 0, st, tmA, tmB0, tmB1, p));
    return check_launch("gemm_fp8_blockscale_skinny_kernel");
}

template <int NT>
int launch_out(const CUtensorMap& tmA, const CUtensorMap& tmB0, const CUtensorMap& tmB1, const BsSkinnyParams& p, const BsSkinnyOut& out, int smem,
               int grid, cudaStream_t st) {
    if (p.split > 1) return out.gated ? launch<NT, 2, true>(tmA, tmB0, tmB1, p, smem, grid, st) : launch<NT, 1, true>(tmA, tmB0, tmB1, p, smem, grid, st);
    if (out.gated) return launch<NT, 2>(tmA, tmB0, tmB1, p, smem, grid, st);
    if (out.epilogue) return launch<NT, 1>(tmA, tmB0, tmB1, p, smem, grid, st);
    return launch<NT, 0>(tmA, tmB0, tmB1, p, smem, grid, st);
}

// How many CTAs share a tile.  A K step (two blocks) takes about 0.32 us (0.41 with 32 token columns) on the MMA thread and its
// hand-off and 8 ns more per KB of weights, or the time in which an SM pulls them (45 bytes per ns when all SMs do); a split adds
// about 2 us: the clusters' barriers and the partial sums.  The split that this puts ahead is taken, if all its clusters fit the device at once.
// 16 tokens, us, whole / 2 / 4 / 8 CTAs per tile: N = 1024, K = 1024 4.9 / 5.4 / 5.1 / 4.9, K = 4096 9.2 / 7.7 / 6.4 / 6.4, K = 14336
// 23.9 / 15.8 / 10.3 / 8.3; N = 4096, K = 1024 5.0 / 5.5 / 5.7 / -, K = 4096 9.5 / 7.8 / 7.1 / -, K = 14336 25.4 / 18.0 / 15.1 / -.
void plan_split(bool nt16, const BsSkinnyOut& out, int64_t units, int parts, int ksteps, int64_t rounds, BsSkinnyParams& p) {
    const void* const kern = nt16 ? (out.gated ? (const void*)gemm_fp8_blockscale_skinny_kernel<16, 2, true> : (const void*)gemm_fp8_blockscale_skinny_kernel<16, 1, true>)
                                  : (out.gated ? (const void*)gemm_fp8_blockscale_skinny_kernel<32, 2, true> : (const void*)gemm_fp8_blockscale_skinny_kernel<32, 1, true>);
    auto step_us = [&](int64_t height) {
        const double kb = 4.0 * height * parts, pull = kb / 44, hand_off = (nt16 ? 0.32 : 0.41) + 0.008 * kb;
        return pull > hand_off ? pull : hand_off;
    };
    double best = rounds * ksteps * step_us((units + p.tiles - 1) / p.tiles);
    for (int split = 2; split <= 8 && split <= ksteps && best > 2; split *= 2) {
        const int64_t clusters = max_clusters(kern, kThreads, kSmemLimit, split);
        if (clusters == 0) break;
        const int64_t tiles = units < clusters ? units : clusters, height = (units + tiles - 1) / tiles;
        if (height * parts > kMaxUnits) break;
        const double us = (ksteps + split - 1) / split * step_us(height) + 2;
        if (us < best) {
            best = us;
            p.split = split;
            p.tiles = (int)tiles;
        }
    }
}

}  // namespace

// Host side: called for M <= 32 and 128-column weight-scale groups (arguments already validated).
int launch_gemm_fp8_blockscale_skinny(const void* A, const void* B, const float* sa, const float* sb, const BsSkinnyOut& out, int64_t M,
                                      int64_t N, int64_t K, uint32_t* status, cudaStream_t st) {
    const int sms = sm_count();
    HKB_REQUIRE(sms > 0, HKB_ERR_CUDA, "no CUDA device");
    BsSkinnyParams p{};
    p.M = (int)M; p.N = (int)N; p.K = (int)K; p.ldc = out.ldc;
    p.sa = sa; p.sb = sb; p.C = (__nv_bfloat16*)out.C; p.c_a = (const __nv_bfloat16*)out.c_a; p.c_b = (const __nv_bfloat16*)out.c_b; p.status = status;
    p.bias = (const __nv_bfloat16*)out.bias; p.act = out.act; p.residual = (const __nv_bfloat16*)out.residual; p.f32 = out.f32;
    p.a_box_rows = (int)((M + 7) / 8 * 8);
    const int nt = (int)((M + 15) / 16 * 16);
    const int64_t units = N / 16;
    const int parts = out.gated ? 2 : 1;                  // gate and up rows share the 128 MMA rows
    const int max_units = kMaxUnits / parts;
    const int64_t rounds = (units + (int64_t)max_units * sms - 1) / ((int64_t)max_units * sms);
    p.split = 1;
    p.tiles = (int)(units < rounds * sms ? units : rounds * sms);
    if (out.gated || out.epilogue) plan_split(nt == 16, out, units, parts, (int)((K / 128 + kStep - 1) / kStep), rounds, p);
    p.base = (int)(units / p.tiles);
    p.rem = (int)(units % p.tiles);
    const int maxu = p.base + (p.rem ? 1 : 0);
    HKB_REQUIRE(maxu >= 1 && maxu <= max_units, HKB_ERR_UNSUPPORTED, "gemm_fp8_blockscale (skinny): internal tile height %d out of range", maxu);
    p.a_off = parts * maxu * 2048;
    p.sub_bytes = p.a_off + nt * 128;
    const int head = kHeadBytes + (out.gated ? kXchgBytes : 0);
    p.stages = (kSmemLimit - 1024 - head - kTailPad) / (kStep * p.sub_bytes);
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    const int smem = 1024 + head + p.stages * kStep * p.sub_bytes + kTailPad;
    CUtensorMap tmA, tmB0, tmB1;
    int rc = make_tmap_bytes(&tmA, A, (uint64_t)K, (uint64_t)M, 1, (uint32_t)p.a_box_rows);
    if (rc != HKB_OK) return rc;
    rc = make_tmap_bytes(&tmB0, B, (uint64_t)K, (uint64_t)(parts * N), 1, (uint32_t)p.base * 16);
    if (rc != HKB_OK) return rc;
    rc = make_tmap_bytes(&tmB1, B, (uint64_t)K, (uint64_t)(parts * N), 1, (uint32_t)maxu * 16);
    if (rc != HKB_OK) return rc;
    const int grid = p.split > 1 ? p.tiles * p.split : p.tiles < sms ? p.tiles : sms;
    if (nt == 16) return launch_out<16>(tmA, tmB0, tmB1, p, out, smem, grid, st);
    return launch_out<32>(tmA, tmB0, tmB1, p, out, smem, grid, st);
}

}  // namespace hkb
