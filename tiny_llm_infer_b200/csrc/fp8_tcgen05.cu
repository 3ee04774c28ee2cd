// y[M, N] = x . w^T with 8-bit operands on the fifth-generation tensor cores (tcgen05, kind::f8f6f4), for rows x and weights w as e4m3
// with float32 scales per 128 columns of a row and per 128 x 128 of the weight (fp8.cuh):
//
//   y[t, n] = sum_b sx[t, b] sw[n / 128, b] P_b[t, n],   P_b = the float32 product of block b's 128 k's.
//
// The scales differ from block to block of K, so no accumulator can run over all of K: the tensor core makes P_b alone (four
// MMAs of 128 x BN x 32) in tensor memory, and eight warps multiply it by its scales and add it to float32 sums in registers while the
// next P_b is being made.  Per block and tile of 128 x 256 the MMAs take 512 cycles, the reads of tensor memory 256 and the
// multiply-adds 256, side by side.
//
// Warps: 0 fetches (TMA, 128-byte swizzle: a row of 128 e4m3 is one swizzle row), 1 issues MMAs and owns the tensor memory, 2 to 9 sum.
// A summing thread owns one row and half of the tile's columns, one block of 128 weight rows, so that a block's scale is one number per thread (two
// for interleaved gate and up rows).  Persistent: one block of threads per SM walks over tiles, row tiles fastest; with few tiles K is
// cut into shares whose float32 sums a second kernel adds in order.
//
// GATED: w's rows are gate and up interleaved by eight, the tile's 256 rows make 128 outputs act(gate) * up, one scale block
// of the next product's rows, so they leave as e4m3 with their scale.
//
// Waits are bounded as in gemm_tcgen05.cu.
#include <cuda.h>

#include "fp8.cuh"
#include "tcgen05.cuh"

namespace tllm {

constexpr int kQM = 128, kQK = 128;              // tile rows; k's per stage = one scale block = one 128-byte swizzle row
constexpr int kQSumWarps = 8, kQThreads = (2 + kQSumWarps) * 32;
constexpr int kQPad = 64 + 16;                   // bytes of a staging row: 64 of output, padded against bank conflicts
constexpr uint32_t kQTmemCols = 512;

// Instruction descriptor, kind::f8f6f4: D float32 (bits 4-5 = 1), A and B e4m3 (0), K-major, N / 8 in bits 17-22, M / 16 in 24-28.
__host__ __device__ constexpr uint32_t instr_desc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
        : "memory");
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

// BN: columns of a tile.  INTER: the weight's rows are interleaved gate and up rows, with two rows of scales per 256.
template <int BN, int OUT, bool INTER>
__global__ void __launch_bounds__(kQThreads, 1)
fp8_tcgen05_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const Fp8Product p,
                   int* __restrict__ error_word) {
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    constexpr int kStageA = kQM * kQK, kStageB = BN * kQK, kStage = kStageA + kStageB;
    constexpr int kStages = BN == 256 ? 4 : 6, kBufs = 512 / BN;
    constexpr int kCols = BN / 2;                               // of a summing thread
    __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages], part_full[kBufs], part_empty[kBufs];
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag;
    __shared__ float largest_of[2][kQM];
    unsigned char* tiles = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int total = p.tiles_m * p.tiles_n * p.splits;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full_bar[s], 1);
            mbar_init(&empty_bar[s], 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&part_full[b], 1);
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

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (int t = blockIdx.x; t < total && !*aborted; t += gridDim.x) {
                const int tile_m = t % p.tiles_m, rest = t / p.tiles_m, tile_n = rest % p.tiles_n;
                int kb0;
                const int n = blocks_of(rest / p.tiles_n, kb0);
                for (int kb = 0; kb < n; ++kb, ++it) {
                    const int s = it % kStages;
                    if (it >= kStages && !mbar_wait(&empty_bar[s], ((it / kStages) - 1) & 1)) {
                        atomicExch(error_word, 1);
                        *aborted = 1;
                    }
                    if (*aborted) break;
                    unsigned char* a = tiles + (size_t)s * kStage;
                    mbar_expect_tx(&full_bar[s], kStage);
                    tma_load_2d(a, &map_x, (kb0 + kb) * kQK, tile_m * kQM, &full_bar[s]);
#pragma unroll
                    for (int h = 0; h < BN / 128; ++h)
                        tma_load_2d(a + kStageA + h * 128 * kQK, &map_w, (kb0 + kb) * kQK, tile_n * BN + h * 128, &full_bar[s]);
                }
            }
            if (*aborted) {                                     // not before the copies in flight have landed
                const int first = it > kStages ? it - kStages : 0;
                for (int i = first; i < it; ++i) mbar_wait(&full_bar[i % kStages], (i / kStages) & 1);
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = instr_desc_e4m3(kQM, BN);
            int it = 0;
            for (int t = blockIdx.x; t < total && !*aborted; t += gridDim.x) {
                int kb0;
                const int n = blocks_of(t / p.tiles_m / p.tiles_n, kb0);
                for (int kb = 0; kb < n; ++kb, ++it) {
                    const int s = it % kStages, buf = it % kBufs;
                    if (it >= kBufs && !mbar_wait(&part_empty[buf], ((it / kBufs) - 1) & 1)) {
                        atomicExch(error_word, 4);
                        *aborted = 1;
                        break;
                    }
                    if (!mbar_wait(&full_bar[s], (it / kStages) & 1)) {
                        atomicExch(error_word, 2);
                        *aborted = 1;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                    const uint32_t a_addr = cvta_shared(tiles + (size_t)s * kStage), b_addr = a_addr + kStageA;
#pragma unroll
                    for (int k = 0; k < kQK / 32; ++k)
                        umma_e4m3(tmem_base + buf * BN, smem_desc_sw128(a_addr + k * 32), smem_desc_sw128(b_addr + k * 32), idesc, k > 0 ? 1u : 0u);
                    umma_commit(&empty_bar[s]);
                    umma_commit(&part_full[buf]);
                }
            }
        }
    } else {
        const int quad = warp & 3, half = (warp - 2) >> 2;      // a warp may read TMEM lanes 32 * (warp % 4) .. + 31
        unsigned char* stage_out = tiles + (size_t)kStages * kStage + (size_t)(warp - 2) * 32 * kQPad;
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
            bool ok = true;
            for (int kb = 0; kb < n; ++kb, ++it) {
                const int buf = it % kBufs;
                const float s0 = sx[kb];
                const float s = s0 * sw[kb], s_up = INTER ? s0 * sw[p.kb_all + kb] : s;
                ok = warp_wait(&part_full[buf], (it / kBufs) & 1, aborted, error_word, 3);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                const uint32_t addr = tmem_base + buf * BN + half * kCols + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                for (int c = 0; c < kCols; c += 32) {
                    uint32_t r[32];
                    tmem_ld32_issue(addr + c, r);
                    tmem_ld_wait();
                    if (c + 32 >= kCols) {                       // all of this warp's numbers are in registers
                        asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&part_empty[buf]);
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[c + j] = fmaf(__uint_as_float(r[j]), INTER && (j & 8) ? s_up : s, acc[c + j]);
                }
            }
            if (!ok) break;
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
                asm volatile("bar.sync 1, %0;\n" ::"n"(kQSumWarps * 32) : "memory");      // the tile before has been read
                largest_of[half][quad * 32 + lane] = largest;
                asm volatile("bar.sync 1, %0;\n" ::"n"(kQSumWarps * 32) : "memory");
                const float scale = fp8_scale(fmaxf(largest, largest_of[half ^ 1][quad * 32 + lane])), inv = 1.0f / scale;
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
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem_base), "r"(kQTmemCols) : "memory");
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

template <int BN, int OUT, bool INTER>
static int launch_fp8_tcgen05(const CUtensorMap& mx, const CUtensorMap& mw, Fp8Product p, int* error_word, cudaStream_t stream) {
    const size_t smem = (size_t)(BN == 256 ? 4 : 6) * (kQM + BN) * kQK + 1024 + (size_t)kQSumWarps * 32 * kQPad;
    static OncePerDevice configured;
    if (configured.first()) {
        cudaError_t e = cudaFuncSetAttribute(fp8_tcgen05_kernel<BN, OUT, INTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) { set_error("fp8_tcgen05: %s", cudaGetErrorString(e)); return (int)e; }
        configured.done();
    }
    p.tiles_m = (p.M + kQM - 1) / kQM;
    p.tiles_n = (p.N + BN - 1) / BN;
    const long long total = (long long)p.tiles_m * p.tiles_n * p.splits;
    TLLM_REQUIRE(total <= 0x7fffffff, "fp8_tcgen05: too many tiles");
    int sms = sm_count_cached();
    if (sms <= 0) sms = 148;
    fp8_tcgen05_kernel<BN, OUT, INTER><<<(int)(total < sms ? total : sms), kQThreads, smem, stream>>>(mx, mw, p, error_word);
    return finish_launch("fp8_tcgen05");
}

}  // namespace tllm

using namespace tllm;

// x [M, K] e4m3 with sx [M, ceil(K / 128)], w [N, K] e4m3 with sw; K a multiple of 16, operands 16-byte aligned.
// form 0: y = x . w^T, bfloat16 [M, N], from tiles of 128 x `columns` (128 or 256).
// form 1: `splits` shares of K (of `kb_per_split` blocks of 128, none empty) as float32 [splits][M][N].
// form 2: gated: w = N / 2 gate and as many up rows interleaved by eight (sw [2 ceil(N / 2 / 128), ceil(K / 128)]), y e4m3 [M, N / 2] with
// y_scales; N / 2 a multiple of 16, tiles of 256 columns.
// interleaved: the weight is one of form 2 (its scales lie so) whatever the form.
extern "C" int tllm_fp8_tcgen05(const void* x, const float* sx, const void* w, const float* sw, void* y, float* y_scales, int M, int N, int K,
                                int form, int interleaved, int columns, int splits, int kb_per_split, int act, float limit, float slope,
                                int* error_word, cudaStream_t stream) {
    TLLM_REQUIRE(M > 0 && N > 0 && K > 0 && K % 16 == 0, "fp8_tcgen05: %d x %d x %d (K a multiple of 16)", M, N, K);
    TLLM_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y)) & 15u) == 0,
                 "fp8_tcgen05: operands must be 16-byte aligned");
    TLLM_REQUIRE(sx && sw && error_word, "fp8_tcgen05: missing scales or error word");
    TLLM_REQUIRE(columns == 128 || columns == 256, "fp8_tcgen05: tiles of %d columns", columns);
    TLLM_REQUIRE(!interleaved || N % 16 == 0, "fp8_tcgen05: interleaved gate and up rows come in sixteens, N = %d", N);
    const int kb_all = (K + kFp8Block - 1) / kFp8Block;
    if (form != 1) splits = 1, kb_per_split = kb_all;
    TLLM_REQUIRE(splits >= 1 && kb_per_split >= 1 && (long long)(splits - 1) * kb_per_split < kb_all && (long long)splits * kb_per_split >= kb_all,
                 "fp8_tcgen05: %d shares of %d blocks for %d", splits, kb_per_split, kb_all);
    CUtensorMap mx, mw;
    TLLM_REQUIRE(fp8_map(&mx, x, M, K) && fp8_map(&mw, w, N, K), "fp8_tcgen05: cuTensorMapEncodeTiled failed or is not available");
    Fp8Product p{sx, sw, y, y_scales, M, N, K, kb_all, 0, 0, splits, kb_per_split, act, GateConst{limit, slope}};
    if (form == 2) {
        TLLM_REQUIRE(interleaved && (N / 2) % 16 == 0 && y_scales && columns == 256 && gated_act_ok(act, limit), "fp8_tcgen05: bad gated product");
        return launch_fp8_tcgen05<256, kOutGated, true>(mx, mw, p, error_word, stream);
    }
    if (form == 1) {
        if (interleaved)
            return columns == 256 ? launch_fp8_tcgen05<256, kOutShare, true>(mx, mw, p, error_word, stream)
                                  : launch_fp8_tcgen05<128, kOutShare, true>(mx, mw, p, error_word, stream);
        return columns == 256 ? launch_fp8_tcgen05<256, kOutShare, false>(mx, mw, p, error_word, stream)
                              : launch_fp8_tcgen05<128, kOutShare, false>(mx, mw, p, error_word, stream);
    }
    TLLM_REQUIRE(form == 0 && !interleaved, "fp8_tcgen05: form %d", form);
    return columns == 256 ? launch_fp8_tcgen05<256, kOutBf16, false>(mx, mw, p, error_word, stream)
                          : launch_fp8_tcgen05<128, kOutBf16, false>(mx, mw, p, error_word, stream);
}

// y[n] (out_dtype) = the sum over `splits` shares of n float32 numbers each.
extern "C" int tllm_fp8_join(const float* shares, int splits, long long n, void* y, int out_dtype, cudaStream_t stream) {
    TLLM_REQUIRE(splits >= 1 && n > 0 && shares && y, "fp8_join: bad arguments");
    TLLM_REQUIRE(out_dtype == kBF16 || out_dtype == kF32, "fp8_join: unknown output dtype");
    TLLM_REQUIRE((reinterpret_cast<uintptr_t>(shares) & 15u) == 0, "fp8_join: shares must be 16-byte aligned");
    const long long grid = (n + 1023) / 1024;
    TLLM_REQUIRE(grid <= 0x7fffffff, "fp8_join: too many numbers");
    if (out_dtype == kBF16)
        launch_pdl(kPdlOther, fp8_join_kernel<bf16>, dim3((unsigned)grid), dim3(256), 0, stream, shares, splits, n, (bf16*)y);
    else
        launch_pdl(kPdlOther, fp8_join_kernel<float>, dim3((unsigned)grid), dim3(256), 0, stream, shares, splits, n, (float*)y);
    return finish_launch("fp8_join");
}
