// y[M, N] = x . w^T with 8-bit operands on the fifth-generation tensor cores (tcgen05, kind::f8f6f4), for rows x and weights w as e4m3
// with float32 scales per 128 columns of a row and per 128 x 128 of the weight (fp8.cuh):
//
//   y[t, n] = sum_b sx[t, b] sw[n / 128, b] P_b[t, n],   P_b = the float32 product of block b's 128 k's.
//
// The scales differ from block to block of K, so no accumulator can run over all of K: the tensor core makes P_b alone (four
// MMAs over 32 k's each) in tensor memory, and eight warps multiply it by its scales and add it to float32 sums in registers while the
// next P_b is being made.
//
// Two kernels.  Pairs of SMs make tiles of 256 x 256 (below); they carry the large products and the gated one.  Where those tiles would
// be too few, single SMs make tiles of 128 x 128, and with fewer still K is cut into shares whose float32 sums a third kernel adds in
// order (2048 x 6144 x 4096: pairs 51 us, which is 2.0 PFLOP/s; 61 x 4096 x 4096 in 4 shares: 11 us with the rows' rounding and the join).
//
// Warps of the 128 x 128 kernel: 0 fetches (TMA, 128-byte swizzle: a row of 128 e4m3 is one swizzle row), 1 and 2 issue MMAs in turn, 3 to
// 10 sum.  A summing thread owns one row and half of the tile's columns, within one block of 128 weight rows, so that a block's scale
// is one number per thread (two for interleaved gate and up rows).  Persistent: one block of threads per SM walks over tiles, row
// tiles fastest.  A block of K costs it 0.37 us, bound by the way wait - MMA - commit - read of tensor memory, not by the MMAs.
//
// GATED: w's rows are gate and up interleaved by eight, a pair's 256 columns make 128 outputs act(gate) * up, one scale block
// of the next product's rows, so they leave as e4m3 with their scale.
//
// Waits are bounded as in gemm_tcgen05.cu.  The kernels start while the one ahead still runs (programmatic dependent launch): every role waits for
// its end before its first bounded wait.
#include <cuda.h>

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace tllm {

constexpr int kQM = 128, kQK = 128;              // tile rows; k's per stage = one scale block = one 128-byte swizzle row
constexpr int kQSumWarps = 8, kQThreads = (3 + kQSumWarps) * 32;
constexpr int kQPad = 64 + 16;                   // bytes of a staging row: 64 of output, padded against bank conflicts
constexpr uint32_t kQTmemCols = 512;
constexpr int kQStages = 6;                      // of 32 KB

// Instruction descriptor, kind::f8f6f4: D float32 (bits 4-5 = 1), A and B e4m3 (0), K-major, N / 8 in bits 17-22, M / 16 in 24-28.
__host__ __device__ constexpr uint32_t instr_desc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Issued by the lane that says so; the warp goes through it as one, its descriptors in uniform registers.
__device__ __forceinline__ void umma_e4m3_if(uint32_t issue, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
__device__ __forceinline__ void umma_commit_if(uint32_t issue, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(cvta_shared(bar)),
        "r"(issue)
        : "memory");
}
// Two sums at a time: (a, b) += (x, y) * (s, t).
__device__ __forceinline__ void fma_pair(float& a, float& b, uint32_t x, uint32_t y, uint64_t st) {
    uint64_t v, d;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "r"(x), "r"(y));
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "f"(a), "f"(b));
    asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(d) : "l"(v), "l"(st));
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(d));
}
__device__ __forceinline__ uint64_t twice(float s) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %1};\n" : "=l"(d) : "f"(s));
    return d;
}

// A wait by all lanes of a warp in a loop whose length is what the kernel's speed hangs on: unlike warp_wait it does not read the block's
// flag (some 100 cycles a wait); where another warp has given up, this one's own limit runs out.
__device__ __forceinline__ bool quick_wait(uint64_t* bar, uint32_t parity, volatile int* aborted, int* error_word, int code) {
    if (__all_sync(0xffffffffu, mbar_wait(bar, parity))) return true;
    atomicExch(error_word, code);
    *aborted = 1;
    return false;
}

// What the tile's sums become.
enum Fp8Out : int { kOutBf16 = 0, kOutShare = 1, kOutGated = 2 };

struct Fp8Product {
    const float *sx, *sw;
    void* y;                     // bfloat16 [M, N], float32 shares [splits][M][N], or e4m3 [M, N / 2]
    float* y_scales;             // gated: [M, ceil(N / 2 / 128)]
    int M, N, K, kb_all;         // N: weight rows
    int tiles_m, tiles_n, splits, kb_per_split;
    int act;
    GateConst gc;
};

// A summing warp's 32 rows (from row0) of kCols sums a thread (from col0) become what the product is asked for, through the warp's staging
// rows, so that an instruction stores whole 64-byte pieces of eight rows.  The two warps of a gated tile's rows exchange their largest
// magnitudes through `meet` (a barrier per four of them, waited for with a limit; two buffers, by the tile's parity).  False: given up.
struct Fp8Meeting {
    float largest[2][2][kQM];
    uint64_t bar[4];
};
template <int OUT, int kCols>
__device__ __forceinline__ bool finish_tile(float (&acc)[kCols], const Fp8Product& p, unsigned char* stage_out, Fp8Meeting* meet, int row0,
                                            int col0, int tile_n, int half, int quad, int lane, int split, int parity, volatile int* aborted,
                                            int* error_word) {
    const int row = row0 + lane;
    if constexpr (OUT == kOutGated) {
        // the thread's columns are 8 gate, 8 up, ...: kCols / 2 outputs, half of the 128 that share a scale
        float largest = 0.0f;
#pragma unroll
        for (int j = 0; j < kCols; j += 16)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = gated_unit(acc[j + e], acc[j + 8 + e], p.act, p.gc);
                acc[j / 2 + e] = v;
                largest = fmaxf(largest, fabsf(v));
            }
        meet->largest[parity][half][quad * 32 + lane] = largest;
        __syncwarp();
        if (lane == 0) mbar_arrive(&meet->bar[quad]);
        if (!warp_wait(&meet->bar[quad], parity, aborted, error_word, 5)) return false;
        const float scale = fp8_scale(fmaxf(largest, meet->largest[parity][half ^ 1][quad * 32 + lane])), inv = 1.0f / scale;
        const int out_n = p.N / 2;
        if (half == 0 && row < p.M) p.y_scales[(size_t)row * ((out_n + kFp8Block - 1) / kFp8Block) + tile_n] = scale;
        __syncwarp();
#pragma unroll
        for (int j = 0; j < kCols / 2; j += 16) {
            uint4 v;
            v.x = to_e4m3x4(acc[j] * inv, acc[j + 1] * inv, acc[j + 2] * inv, acc[j + 3] * inv);
            v.y = to_e4m3x4(acc[j + 4] * inv, acc[j + 5] * inv, acc[j + 6] * inv, acc[j + 7] * inv);
            v.z = to_e4m3x4(acc[j + 8] * inv, acc[j + 9] * inv, acc[j + 10] * inv, acc[j + 11] * inv);
            v.w = to_e4m3x4(acc[j + 12] * inv, acc[j + 13] * inv, acc[j + 14] * inv, acc[j + 15] * inv);
            *reinterpret_cast<uint4*>(stage_out + lane * kQPad + j) = v;
        }
        __syncwarp();
        // whole 64-byte pieces of rows: eight rows per instruction; out_n is a multiple of 16
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = j * 8 + (lane >> 2), col = tile_n * 128 + half * 64 + (lane & 3) * 16;
            if (row0 + r < p.M && col < out_n)
                *reinterpret_cast<uint4*>((uint8_t*)p.y + (size_t)(row0 + r) * out_n + col) =
                    *reinterpret_cast<const uint4*>(stage_out + r * kQPad + (lane & 3) * 16);
        }
    } else if constexpr (OUT == kOutShare) {
        float* y = (float*)p.y + (size_t)split * p.M * p.N;
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 16; j += 4)
                *reinterpret_cast<float4*>(stage_out + lane * kQPad + j * 4) = make_float4(acc[c + j], acc[c + j + 1], acc[c + j + 2], acc[c + j + 3]);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = j * 8 + (lane >> 2), col = col0 + c + (lane & 3) * 4;
                if (row0 + r >= p.M || col >= p.N) continue;
                const float4 v = *reinterpret_cast<const float4*>(stage_out + r * kQPad + (lane & 3) * 16);
                float* dst = y + (size_t)(row0 + r) * p.N + col;
                if ((p.N & 3) == 0) {
                    *reinterpret_cast<float4*>(dst) = v;
                } else {
                    const float e[4] = {v.x, v.y, v.z, v.w};
                    for (int i = 0; i < 4 && col + i < p.N; ++i) dst[i] = e[i];
                }
            }
        }
    } else {
#pragma unroll
        for (int c = 0; c < kCols; c += 32) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; j += 8) {
                uint4 v;
                __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(acc[c + j + 2 * i], acc[c + j + 2 * i + 1]);
                *reinterpret_cast<uint4*>(stage_out + lane * kQPad + j * 2) = v;
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = j * 8 + (lane >> 2), col = col0 + c + (lane & 3) * 8;
                if (row0 + r >= p.M || col >= p.N) continue;
                const uint4 v = *reinterpret_cast<const uint4*>(stage_out + r * kQPad + (lane & 3) * 16);
                bf16* dst = (bf16*)p.y + (size_t)(row0 + r) * p.N + col;
                if ((p.N & 7) == 0) {
                    *reinterpret_cast<uint4*>(dst) = v;
                } else {
                    const bf16* e = reinterpret_cast<const bf16*>(&v);
                    for (int i = 0; i < 8 && col + i < p.N; ++i) dst[i] = e[i];
                }
            }
        }
    }
    return true;
}

// INTER: the weight's rows are interleaved gate and up rows, with two rows of scales per 256.
template <int OUT, bool INTER>
__global__ void __launch_bounds__(kQThreads, 1)
fp8_tcgen05_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Product p,
                   int* __restrict__ error_word) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    constexpr int BN = 128, kStageA = kQM * kQK, kStageB = BN * kQK, kStage = kStageA + kStageB;
    constexpr int kStages = kQStages, kBufs = 512 / BN;
    constexpr int kCols = BN / 2;                               // of a summing thread
    // a stage's data are there; its MMAs are done (the stage is free again, the block's products are there); a quarter of tensor memory is read
    __shared__ __align__(8) uint64_t full_bar[kStages], done_bar[kStages], part_empty[kBufs];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int total = p.tiles_m * p.tiles_n * p.splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&done_bar[s], 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&part_empty[b], kQSumWarps);
        }
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(cvta_shared(&tmem_base_slot)), "r"(kQTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem_base = tmem_base_slot;
    volatile int* aborted = &abort_flag;
    // tile t: row tile fastest, then column tile, then share of K
    auto blocks_of = [&](int split, int& kb0) {
        kb0 = split * p.kb_per_split;
        return min(p.kb_all - kb0, p.kb_per_split);
    };

    TLLM_PDL_TRIGGER();
    if (warp == 0) {
        if (lane == 0) {
            TLLM_PDL_WAIT();                                    // x is the kernel ahead's
            int it = 0;
            for (int t = blockIdx.x; t < total && !*aborted; t += gridDim.x) {
                const int tile_m = t % p.tiles_m, rest = t / p.tiles_m, tile_n = rest % p.tiles_n;
                int kb0;
                const int n = blocks_of(rest / p.tiles_n, kb0);
                for (int kb = 0; kb < n; ++kb, ++it) {
                    const int s = it % kStages;
                    if (it >= kStages && !mbar_wait(&done_bar[s], ((it / kStages) - 1) & 1)) {
                        atomicExch(error_word, 1);
                        *aborted = 1;
                    }
                    if (*aborted) break;
                    unsigned char* a = tiles + (size_t)s * kStage;
                    mbar_expect_tx(&full_bar[s], kStage);
                    tma_load_2d(a, &map_x, (kb0 + kb) * kQK, tile_m * kQM, &full_bar[s]);
                    tma_load_2d(a + kStageA, &map_w, (kb0 + kb) * kQK, tile_n * BN, &full_bar[s]);
                }
            }
            if (*aborted) {                                     // not before the copies in flight have landed
                const int first = it > kStages ? it - kStages : 0;
                for (int i = first; i < it; ++i) mbar_wait(&full_bar[i % kStages], (i / kStages) & 1);
            }
        }
    } else if (warp < 3) {
        // two warps issue in turn (see the pairs below)
        TLLM_PDL_WAIT();                                        // or the limit of the first wait runs over the kernel ahead's work
        constexpr uint32_t idesc = instr_desc_e4m3(kQM, BN);
        const uint32_t issue = lane == 0;
        int it = 0;                                              // blocks of the tiles before
        bool ok = true;
        for (int t = blockIdx.x; ok && t < total; t += gridDim.x) {
            int kb0;
            const int n = blocks_of(t / p.tiles_m / p.tiles_n, kb0);
            for (int i = it; i < it + n; ++i) {
                if ((i & 1) != warp - 1) continue;
                const int s = i % kStages, buf = i % kBufs;
                ok = quick_wait(&full_bar[s], (i / kStages) & 1, aborted, error_word, 2) &&
                     (i < kBufs || quick_wait(&part_empty[buf], ((i / kBufs) - 1) & 1, aborted, error_word, 4));
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint32_t a_addr = cvta_shared(tiles + (size_t)s * kStage);
                const uint64_t a_desc = smem_desc_sw128(a_addr), b_desc = smem_desc_sw128(a_addr + kStageA);
#pragma unroll
                for (int k = 0; k < kQK / 32; ++k)               // 32 bytes further: two units of the descriptor's address
                    umma_e4m3_if(issue, tmem_base + buf * BN, a_desc + 2 * k, b_desc + 2 * k, idesc, k > 0 ? 1u : 0u);
                umma_commit_if(issue, &done_bar[s]);
            }
            it += n;
        }
    } else {
        TLLM_PDL_WAIT();                                        // so are its scales
        const int quad = warp & 3, half = (warp - 3) >> 2;      // a warp may read TMEM lanes 32 * (warp % 4) .. + 31
        unsigned char* stage_out = tiles + (size_t)kStages * kStage + (size_t)(warp - 3) * 32 * kQPad;
        int it = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x) {
            const int tile_m = t % p.tiles_m, rest = t / p.tiles_m, tile_n = rest % p.tiles_n, split = rest / p.tiles_n;
            int kb0;
            const int n = blocks_of(split, kb0);
            const int row0 = tile_m * kQM + quad * 32, row = row0 + lane, col0 = tile_n * BN + half * kCols;
            const float* sx = p.sx + (size_t)min(row, p.M - 1) * p.kb_all + kb0;
            // INTER: 256 weight rows are a block of gate and a block of up rows, interleaved; their scales are two rows
            const int last_block = (p.N - 1) / kFp8Block;
            const float* sw = p.sw + (size_t)(INTER ? 2 * (tile_n * BN / 256) : min(col0 / kFp8Block, last_block)) * p.kb_all + kb0;
            float acc[kCols];
#pragma unroll
            for (int j = 0; j < kCols; ++j) acc[j] = 0.0f;
            float s_x = sx[0], s_w = sw[0], s_u = INTER ? sw[p.kb_all] : 0.0f;
            bool ok = true;
            for (int kb = 0; kb < n; ++kb, ++it) {
                const int buf = it % kBufs;
                const uint64_t s = twice(s_x * s_w), s_up = INTER ? twice(s_x * s_u) : s;
                if (kb + 1 < n) {
                    s_x = sx[kb + 1];
                    s_w = sw[kb + 1];
                    if (INTER) s_u = sw[p.kb_all + kb + 1];
                }
                ok = quick_wait(&done_bar[it % kStages], (it / kStages) & 1, aborted, error_word, 3);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint32_t addr = tmem_base + buf * BN + half * kCols + ((uint32_t)(quad * 32) << 16);
                uint32_t r[2][32];
                tmem_ld32_issue(addr, r[0]);
                tmem_ld32_issue(addr + 32, r[1]);
                tmem_ld_wait();
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&part_empty[buf]);
#pragma unroll
                for (int j = 0; j < kCols; j += 2)
                    fma_pair(acc[j], acc[j + 1], r[j >> 5][j & 31], r[j >> 5][(j & 31) + 1], INTER && (j & 8) ? s_up : s);
            }
            if (!ok) break;
            finish_tile<OUT, kCols>(acc, p, stage_out, nullptr, row0, col0, tile_n, half, quad, lane, split, 0, aborted, error_word);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kQTmemCols) : "memory");
}

// ---------------------------------------------------------------- pairs of SMs
// Tiles of 256 x 256 by two SMs (cta_group::2): each holds 128 rows of x and half of the 256 weight rows, and the tensor cores of both
// read both halves, so a block of K costs an SM 32 KB from L2 in place of 48 for the same MMAs.  Two warps of the first SM issue for
// both; sums of 128 x 256 stay with each SM, whose eight summing warps read 64 columns at a time and take two numbers per
// instruction (fma.f32x2).  Those warps hold 128 sums a thread: registers go to them from the warpgroup that
// fetches and issues (384 threads of 168 at launch: 4 warps of 40 and 8 of 232).
// A block of K takes 0.47 us, of which the MMAs are 0.27: tensor memory holds two blocks' products, so a block's way through wait, MMAs,
// commit and read is what bounds it (the tensor pipe is active for 55% of the time).  A block's MMAs cut in halves of 128 columns, each
// with a commit of its own, took 63 us where this takes 57 (2048 x 6144 x 4096 with the rows' rounding).
constexpr int kPairThreads = 384, kPairStages = 6, kPairStage = 2 * 128 * kQK;
constexpr int kPairFetchRegs = 40, kPairSumRegs = 232;

// The address of the first SM's copy of something in shared memory.
__device__ __forceinline__ uint32_t in_first(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(a) : "r"(cvta_shared(p)));
    return a;
}
__device__ __forceinline__ void tma_load_pair(void* smem_dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n" ::"r"(
            cvta_shared(smem_dst)),
        "l"(map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void umma_pair_if(uint32_t issue, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issue)
        : "memory");
}
// Arrives at the barrier's place in both SMs once the MMAs issued so far are done.
__device__ __forceinline__ void umma_commit_pair_if(uint32_t issue, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}\n" ::"r"(cvta_shared(bar)),
        "r"(issue), "h"((uint16_t)3)
        : "memory");
}
template <int OUT>
__global__ void __launch_bounds__(kPairThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Product p,
                int* __restrict__ error_word) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    constexpr bool INTER = OUT == kOutGated;
    constexpr int kCols = 128;                                  // of a summing thread
    // a stage's data are there; its MMAs are done (the stage is free again, the block's products are there); a half of tensor memory is read
    __shared__ __align__(8) uint64_t full_bar[kPairStages], done_bar[kPairStages], part_empty[2];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ Fp8Meeting meet;
    // both SMs round up alike: descriptors made by the first serve both
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_rank(), total = p.tiles_m * p.tiles_n;
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&done_bar[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&part_empty[b], 2 * kQSumWarps);          // of both SMs
        }
        for (int q = 0; q < 4; ++q) mbar_init(&meet.bar[q], 2);
        abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(cvta_shared(&tmem_base_slot)), "r"(kQTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    cluster_sync();                                             // the other SM's barriers exist
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem_base = tmem_base_slot;
    volatile int* aborted = &abort_flag;
    TLLM_PDL_TRIGGER();

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kPairFetchRegs));
        if (warp == 0 && lane == 0) {
            TLLM_PDL_WAIT();                                    // x is the kernel ahead's
            int it = 0;
            for (int t = pair; t < total && !*aborted; t += pairs) {
                const int row = (t % p.tiles_m) * 256 + rank * 128, col = (t / p.tiles_m) * 256 + rank * 128;
                for (int kb = 0; kb < p.kb_all; ++kb, ++it) {
                    const int s = it % kPairStages;
                    if (it >= kPairStages && !mbar_wait(&done_bar[s], ((it / kPairStages) - 1) & 1)) {
                        atomicExch(error_word, 1);
                        *aborted = 1;
                    }
                    if (*aborted) break;
                    unsigned char* a = tiles + (size_t)s * kPairStage;
                    if (rank == 0) mbar_expect_tx(&full_bar[s], 2 * kPairStage);        // the bytes of both SMs
                    const uint32_t bar = in_first(&full_bar[s]);
                    tma_load_pair(a, &map_x, kb * kQK, row, bar);
                    tma_load_pair(a + 128 * kQK, &map_w, kb * kQK, col, bar);
                }
            }
            // not before the copies in flight have landed: the first SM waits for both, the second leaves with it
            if (*aborted && rank == 0) {
                const int first = it > kPairStages ? it - kPairStages : 0;
                for (int i = first; i < it; ++i) mbar_wait(&full_bar[i % kPairStages], (i / kPairStages) & 1);
            }
        } else if ((warp == 1 || warp == 2) && rank == 0) {
            // two warps issue in turn, one for each half of tensor memory: a warp's waits, issue and commit take as long as a block's MMAs
            TLLM_PDL_WAIT();                                    // or the limit of the first wait runs over the kernel ahead's work
            constexpr uint32_t idesc = instr_desc_e4m3(256, 256);
            const uint32_t issue = lane == 0, acc = tmem_base + (warp - 1) * 256;
            const int blocks = (total - pair + pairs - 1) / pairs * p.kb_all;       // of all of this pair's tiles
            for (int it = warp - 1; it < blocks; it += 2) {
                const int s = it % kPairStages;
                if (!quick_wait(&full_bar[s], (it / kPairStages) & 1, aborted, error_word, 2)) break;
                if (it >= 2 && !quick_wait(&part_empty[warp - 1], ((it >> 1) - 1) & 1, aborted, error_word, 4)) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint32_t a_addr = cvta_shared(tiles + (size_t)s * kPairStage);
                const uint64_t a_desc = smem_desc_sw128(a_addr), b_desc = smem_desc_sw128(a_addr + 128 * kQK);
#pragma unroll
                for (int k = 0; k < kQK / 32; ++k)               // 32 bytes further: two units of the descriptor's address
                    umma_pair_if(issue, acc, a_desc + 2 * k, b_desc + 2 * k, idesc, k > 0 ? 1u : 0u);
                umma_commit_pair_if(issue, &done_bar[s]);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kPairSumRegs));
        TLLM_PDL_WAIT();                                        // so are its scales
        const int quad = warp & 3, half = (warp - 4) >> 2;
        unsigned char* stage_out = tiles + (size_t)kPairStages * kPairStage + (size_t)(warp - 4) * 32 * kQPad;
        const uint32_t lane_addr = tmem_base + half * kCols + ((uint32_t)(quad * 32) << 16);
        const uint32_t empty0 = in_first(&part_empty[0]), empty1 = in_first(&part_empty[1]);
        const int last_block = (p.N - 1) / kFp8Block;
        int it = 0, parity = 0;
        for (int t = pair; t < total; t += pairs, parity ^= 1) {
            const int tile_m = t % p.tiles_m, tile_n = t / p.tiles_m;
            const int row0 = tile_m * 256 + rank * 128 + quad * 32, row = row0 + lane, col0 = tile_n * 256 + half * kCols;
            const float* sx = p.sx + (size_t)min(row, p.M - 1) * p.kb_all;
            const float* sw = p.sw + (size_t)(INTER ? 2 * tile_n : min(col0 / kFp8Block, last_block)) * p.kb_all;
            float acc[kCols];
#pragma unroll
            for (int j = 0; j < kCols; ++j) acc[j] = 0.0f;
            float s_x = sx[0], s_w = sw[0], s_u = INTER ? sw[p.kb_all] : 0.0f;
            bool ok = true;
            for (int kb = 0; kb < p.kb_all; ++kb, ++it) {
                const int buf = it & 1;
                const uint64_t s = twice(s_x * s_w), s_up = INTER ? twice(s_x * s_u) : s;
                if (kb + 1 < p.kb_all) {
                    s_x = sx[kb + 1];
                    s_w = sw[kb + 1];
                    if (INTER) s_u = sw[p.kb_all + kb + 1];
                }
                ok = quick_wait(&done_bar[it % kPairStages], (it / kPairStages) & 1, aborted, error_word, 3);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
#pragma unroll
                for (int c = 0; c < kCols; c += 64) {
                    uint32_t r[2][32];
                    tmem_ld32_issue(lane_addr + buf * 256 + c, r[0]);
                    tmem_ld32_issue(lane_addr + buf * 256 + c + 32, r[1]);
                    tmem_ld_wait();
                    if (c + 64 == kCols) {                       // all of this warp's numbers are in registers
                        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                        __syncwarp();
                        if (lane == 0) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];\n" ::"r"(buf ? empty1 : empty0) : "memory");
                    }
#pragma unroll
                    for (int j = 0; j < 64; j += 2)
                        fma_pair(acc[c + j], acc[c + j + 1], r[j >> 5][j & 31], r[j >> 5][(j & 31) + 1], INTER && (j & 8) ? s_up : s);
                }
            }
            if (!ok) break;
            if (!finish_tile<OUT, kCols>(acc, p, stage_out, &meet, row0, col0, tile_n, half, quad, lane, 0, parity, aborted, error_word)) break;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    cluster_sync();                                             // neither SM leaves while the other may signal it or read its memory
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kQTmemCols) : "memory");
}

// The shares of K added in order, as TOut.
template <typename TOut>
__global__ void __launch_bounds__(256) fp8_join_kernel(const float* shares, int splits, long long n, TOut* __restrict__ y) {
    TLLM_PDL_ENTER();
    const long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) * 4;
    if (i >= n) return;
    if ((n & 3) == 0) {
        float4 a = *reinterpret_cast<const float4*>(shares + i);
        for (int s = 1; s < splits; ++s) {
            const float4 b = *reinterpret_cast<const float4*>(shares + s * n + i);
            a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
        }
        const float e[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) y[i + j] = from_f32<TOut>(e[j]);
    } else {
        for (int j = 0; j < 4 && i + j < n; ++j) {
            float a = shares[i + j];
            for (int s = 1; s < splits; ++s) a += shares[s * n + i + j];
            y[i + j] = from_f32<TOut>(a);
        }
    }
}

using Fp8EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static Fp8EncodeFn fp8_encode_fn() {
    static Fp8EncodeFn fn = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            return (Fp8EncodeFn) nullptr;
        return (Fp8EncodeFn)ptr;
    }();
    return fn;
}
// Boxes of 128 rows x 128 bytes; what lies outside the matrix reads as zeros, so K and N need not fill their last blocks.
static bool fp8_map(CUtensorMap* map, const void* base, long long rows, long long k) {
    Fp8EncodeFn fn = fp8_encode_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)k, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)k};
    const cuuint32_t box[2] = {(cuuint32_t)kQK, 128u};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int OUT, bool INTER>
static int launch_fp8_tcgen05(const CUtensorMap& mx, const CUtensorMap& mw, Fp8Product p, int* error_word, cudaStream_t stream) {
    constexpr size_t smem = (size_t)kQStages * (kQM + 128) * kQK + 1024 + (size_t)kQSumWarps * 32 * kQPad;
    static OncePerDevice configured;
    if (configured.first()) {
        cudaError_t e = cudaFuncSetAttribute(fp8_tcgen05_kernel<OUT, INTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) { set_error("fp8_tcgen05: %s", cudaGetErrorString(e)); return (int)e; }
        configured.done();
    }
    p.tiles_m = (p.M + kQM - 1) / kQM;
    p.tiles_n = (p.N + 127) / 128;
    const long long total = (long long)p.tiles_m * p.tiles_n * p.splits;
    TLLM_REQUIRE(total <= 0x7fffffff, "fp8_tcgen05: too many tiles");
    int sms = sm_count_cached();
    if (sms <= 0) sms = 148;
    launch_pdl(kPdlAlways, fp8_tcgen05_kernel<OUT, INTER>, dim3((unsigned)(total < sms ? total : sms)), dim3(kQThreads), smem, stream, mx, mw, p, error_word);
    return finish_launch("fp8_tcgen05");
}

template <int OUT>
static int launch_fp8_pair(const CUtensorMap& mx, const CUtensorMap& mw, Fp8Product p, int* error_word, cudaStream_t stream) {
    constexpr size_t smem = (size_t)kPairStages * kPairStage + 1024 + (size_t)kQSumWarps * 32 * kQPad;
    static OncePerDevice configured;
    if (configured.first()) {
        cudaError_t e = cudaFuncSetAttribute(fp8_pair_kernel<OUT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        cudaFuncAttributes got = {};
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&got, fp8_pair_kernel<OUT>);
        if (e != cudaSuccess) { set_error("fp8_pair: %s", cudaGetErrorString(e)); return (int)e; }
        // what the summing warps ask for has to be what the block was launched with: more would never be given
        TLLM_REQUIRE(got.numRegs * kPairThreads >= 128 * kPairFetchRegs + 256 * kPairSumRegs, "fp8_pair: built with %d registers a thread", got.numRegs);
        configured.done();
    }
    p.tiles_m = (p.M + 255) / 256;
    p.tiles_n = (p.N + 255) / 256;
    const long long total = (long long)p.tiles_m * p.tiles_n;
    TLLM_REQUIRE(total <= 0x3fffffff, "fp8_pair: too many tiles");
    int sms = sm_count_cached();
    if (sms <= 1) sms = 148;
    const int pairs = (int)(total < sms / 2 ? total : sms / 2);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(kPairThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, fp8_pair_kernel<OUT>, mx, mw, p, error_word);
    if (e != cudaSuccess) { set_error("fp8_pair: %s", cudaGetErrorString(e)); return (int)e; }
    return finish_launch("fp8_pair");
}

}  // namespace tllm

using namespace tllm;

// x [M, K] e4m3 with sx [M, ceil(K / 128)], w [N, K] e4m3 with sw; K a multiple of 16, operands 16-byte aligned.
// form 0: y = x . w^T, bfloat16 [M, N], from tiles of 128 x 128, or with `pairs` of 256 x 256.
// form 1: `splits` shares of K (of `kb_per_split` blocks of 128, none empty) as float32 [splits][M][N], from tiles of 128 x 128.
// form 2: gated: w = N / 2 gate and as many up rows interleaved by eight (sw [2 ceil(N / 2 / 128), ceil(K / 128)]), y e4m3 [M, N / 2] with
// y_scales; N / 2 a multiple of 16, `pairs`.
// interleaved: the weight is one of form 2 (its scales lie so) whatever the form.
extern "C" int tllm_fp8_tcgen05(const void* x, const float* sx, const void* w, const float* sw, void* y, float* y_scales, int M, int N, int K,
                                int form, int interleaved, int pairs, int splits, int kb_per_split, int act, float limit, float slope,
                                int* error_word, cudaStream_t stream) {
    TLLM_REQUIRE(M > 0 && N > 0 && K > 0 && K % 16 == 0, "fp8_tcgen05: %d x %d x %d (K a multiple of 16)", M, N, K);
    TLLM_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0,
                 "fp8_tcgen05: operands must be 16-byte aligned");
    TLLM_REQUIRE(sx && sw && error_word, "fp8_tcgen05: missing scales or error word");
    TLLM_REQUIRE(!interleaved || N % 16 == 0, "fp8_tcgen05: interleaved gate and up rows come in sixteens, N = %d", N);
    const int kb_all = (K + kFp8Block - 1) / kFp8Block;
    if (form != 1) splits = 1, kb_per_split = kb_all;
    TLLM_REQUIRE(splits >= 1 && kb_per_split >= 1 && (long long)(splits - 1) * kb_per_split < kb_all && (long long)splits * kb_per_split >= kb_all,
                 "fp8_tcgen05: %d shares of %d blocks for %d", splits, kb_per_split, kb_all);
    CUtensorMap mx, mw;
    TLLM_REQUIRE(fp8_map(&mx, x, M, K) && fp8_map(&mw, w, N, K), "fp8_tcgen05: cuTensorMapEncodeTiled failed or is not available");
    Fp8Product p{sx, sw, y, y_scales, M, N, K, kb_all, 0, 0, splits, kb_per_split, act, GateConst{limit, slope}};
    if (form == 2) {
        TLLM_REQUIRE(interleaved && (N / 2) % 16 == 0 && y_scales && pairs && gated_act_ok(act, limit), "fp8_tcgen05: bad gated product");
        return launch_fp8_pair<kOutGated>(mx, mw, p, error_word, stream);
    }
    if (form == 1)
        return interleaved ? launch_fp8_tcgen05<kOutShare, true>(mx, mw, p, error_word, stream) : launch_fp8_tcgen05<kOutShare, false>(mx, mw, p, error_word, stream);
    TLLM_REQUIRE(form == 0 && !interleaved, "fp8_tcgen05: form %d", form);
    return pairs ? launch_fp8_pair<kOutBf16>(mx, mw, p, error_word, stream) : launch_fp8_tcgen05<kOutBf16, false>(mx, mw, p, error_word, stream);
}

// y[n] (out_dtype) = the sum over `splits` shares of n float32 numbers each.
extern "C" int tllm_fp8_join(const float* shares, int splits, long long n, void* y, int out_dtype, cudaStream_t stream) {
    TLLM_REQUIRE(splits >= 1 && n > 0 && shares && y, "fp8_join: bad arguments");
    TLLM_REQUIRE(out_dtype == kBF16 || out_dtype == kF32, "fp8_join: unknown output dtype");
    TLLM_REQUIRE((reinterpret_cast<uintptr_t>(shares) & 15u) == 0, "fp8_join: shares must be 16-byte aligned");
    const long long grid = (n + 1023) / 1024;
    TLLM_REQUIRE(grid <= 0x7fffffff, "fp8_join: too many numbers");
    if (out_dtype == kBF16)
        launch_pdl(kPdlAlways, fp8_join_kernel<bf16>, dim3((unsigned)grid), dim3(256), 0, stream, shares, splits, n, (bf16*)y);
    else
        launch_pdl(kPdlAlways, fp8_join_kernel<float>, dim3((unsigned)grid), dim3(256), 0, stream, shares, splits, n, (float*)y);
    return finish_launch("fp8_join");
}
