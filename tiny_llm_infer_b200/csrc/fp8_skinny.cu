// y[M, N] = x . w^T for a handful of rows with an 8-bit weight: x as e4m3 rows with a scale per 128 columns, w as e4m3 with a scale
// per 128 x 128 (fp8.cuh),
//
//   y[t, n] = sum_b sx[t, b] sw[n / 128, b] sum_{k in block b} qx[t, k] qw[n, k],
//
// the product of a decode step, where every weight is read once: the time is HBM's, half of what the bfloat16 weights take.
//
// A tile is 16 rows of w; the eight warps of a thread block split its K by blocks of 128.  Thread blocks stay (two per SM) and walk over tiles,
// and a warp's weights come through a ring of its own (cp.async, 2 KB per block of 128), filled across the ends of tiles: weights are on
// their way while a tile's sums are added up and written.  A block per tile that loaded ahead only within its tile had four blocks of 128
// per warp to fill its pipeline with and reached half of HBM's rate (gate and up of Qwen3-8B sizes, one row: 28.7 us).
//
// A lane's sixteen neighbouring bytes of a weight row become pairs of float16, which hold every e4m3 value exactly, and stand for the
// columns that four fragments of mma.sync m16n8k16 assign to the lane, on the side of x alike.  The 128 products of a block are summed
// in float32 (each is exact), then scaled and added to the running float32 sum.  (mma.sync on e4m3 itself gives the same sums in half as
// much time again: 43 us where float16 took 29.)
//
// The rows: where a warp has few blocks of 128 (KPW) it keeps its share of x in registers for all tiles, and can round it from bfloat16
// itself (XBF16: the quad that multiplies a block holds all of its 128 numbers of a row), which saves a launch; with more, rows in 8 bits
// come through the ring beside the weights.
//
// Launched early (programmatic dependent launch) like gemm_skinny.cu: weights are fetched before the wait, x after it.
#include "fp8.cuh"
#include "mma_tiles.cuh"

namespace tllm {

constexpr int kFp8Warps = 8, kFp8TileRows = 16;
constexpr int kFp8TileBytes = kFp8TileRows * kFp8Block;

__device__ __forceinline__ uint4 ld_rows(const void* p) {     // what the kernel ahead has written: ordinary loads, after the wait
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float ld_scale(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];\n" : "=f"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src));
}
// A ring stage: the weights, the rows (KPW 0), and their scales: two of the weight's, then those of the rows.  The rings of two thread
// blocks fill an SM's shared memory with 80 KB of weights on their way beside rows in registers, 48 KB with rows in the ring; sixteen rows (NT 2)
// leave room for one block with 80 KB.
template <int NT, int KPW>
struct Fp8Ring {
    static constexpr int kX = KPW == 0 ? NT * 8 * kFp8Block : 0, kScales = 16 + (KPW == 0 ? NT * 8 * 4 : 0);
    static constexpr int kStage = kFp8TileBytes + kX + kScales;
    static constexpr int kBlocks = NT == 1 ? 2 : 1, kStages = NT == 1 && KPW == 0 ? 4 : 6;
    static constexpr size_t kBytes = (size_t)kFp8Warps * kStages * kStage;
};

// Where 16-byte chunk `chunk` of row `row` of a tile lies: reads of four chunks of eight rows meet every bank once.
__device__ __forceinline__ int tile_at(int row, int chunk) { return row * kFp8Block + ((chunk ^ ((row & 1) << 2)) << 4); }

// GATED: w holds N gate and N up rows interleaved by eight, y [M, N] is act(gate) * up; a tile's upper half are eight gate rows,
// its lower half their up rows, whose scales lie in neighbouring rows of `sw`.  KPW: blocks of 128 per warp whose rows stay in registers
// (at least the number there are), 0: rows through the ring.
template <int NT, int KPW, bool XBF16, bool GATED, typename TOut>
__global__ void __launch_bounds__(kFp8Warps * 32, Fp8Ring<NT, KPW>::kBlocks)
fp8_skinny_kernel(const void* x, const float* sx, const uint8_t* __restrict__ w, const float* __restrict__ sw, TOut* y, int M, int N,
                  int K, int tiles, int act, GateConst gc) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float red[2][kFp8Warps][kFp8TileRows][NT * 8 + 1];
    TLLM_PDL_TRIGGER();
    using Ring = Fp8Ring<NT, KPW>;
    constexpr int stages = Ring::kStages;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, rq = lane >> 2;
    const int kb_all = (K + kFp8Block - 1) / kFp8Block, last_row = (GATED ? 2 * N : N) - 1;
    const int per_warp = (kb_all + kFp8Warps - 1) / kFp8Warps;
    const int kb0 = min(warp * per_warp, kb_all), n_kb = min(kb_all - kb0, per_warp);
    const uint32_t ring = smem_u32(smem) + warp * stages * Ring::kStage;
    const unsigned char* ring_p = smem + (size_t)warp * stages * Ring::kStage;

    // ---- the next block of 128 to fetch: of tile f_tile, the f_kb-th of this warp's
    int f_tile = blockIdx.x, f_kb = 0, f_stage = 0;
    const int l_row = lane >> 3, l_chunk = lane & 7;            // this lane's four pieces: rows l_row + 4 i
    auto fetch = [&](bool rows) {
        if (f_tile < tiles && n_kb > 0) {
            const int kb = kb0 + f_kb, k = kb * kFp8Block + l_chunk * 16;
            const uint32_t dst = ring + f_stage * Ring::kStage;
            const uint8_t* src = w + (size_t)(f_tile * kFp8TileRows + l_row) * K + k;
            const bool ok = k < K;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = f_tile * kFp8TileRows + l_row + 4 * i;
                cp_async_16(dst + tile_at(l_row + 4 * i, l_chunk), ok && row <= last_row ? src + (size_t)(4 * i) * K : w, ok && row <= last_row);
            }
            const uint32_t scales = dst + kFp8TileBytes + Ring::kX;
            if (lane < (GATED ? 2 : 1)) {
                const size_t block = GATED ? (size_t)(f_tile * 8 / kFp8Block) * 2 + lane : (size_t)(f_tile * kFp8TileRows / kFp8Block);
                cp_async_4(scales + lane * 4, sw + block * kb_all + kb);
            }
            if (KPW == 0 && rows) {
#pragma unroll
                for (int i = 0; i < NT * 2; ++i) {
                    const int tok = l_row + 4 * i;
                    if (tok < M) cp_async_16(dst + kFp8TileBytes + tile_at(tok, l_chunk), ok ? (const uint8_t*)x + (size_t)tok * K + k : x, ok);
                }
                if (lane < NT * 8) cp_async_4(scales + 16 + lane * 4, sx + (size_t)min(lane, M - 1) * kb_all + kb);
            }
            if (++f_kb == n_kb) f_kb = 0, f_tile += gridDim.x;
            if (++f_stage == stages) f_stage = 0;
        }
        if (rows || KPW != 0) cp_async_commit();                 // one group per call, empty past the end
    };
    // Before the wait nothing may be read that the kernel ahead writes.  Rows through the ring go with their weights, after it.
    if (KPW != 0)
        for (int i = 0; i < stages - 1; ++i) fetch(false);
    TLLM_PDL_WAIT();
    if (KPW == 0)
        for (int i = 0; i < stages - 1; ++i) fetch(true);

    // ---- this warp's share of x, in registers
    constexpr int kHeld = KPW == 0 ? 1 : KPW;
    uint32_t held[kHeld][NT][8];
    float held_s[kHeld][NT][2];
    if constexpr (KPW != 0) {
#pragma unroll
        for (int j = 0; j < KPW; ++j)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int tok = nt * 8 + rq, kb = kb0 + j;
                const uint4 zero = make_uint4(0, 0, 0, 0);
                if constexpr (XBF16) {
                    uint4 raw[4];
                    uint32_t m = 0;                              // largest magnitudes of the pairs
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int k = kb * kFp8Block + (i >> 1) * 64 + c * 16 + (i & 1) * 8;
                        raw[i] = j < n_kb && tok < M && k < K ? ld_rows((const bf16*)x + (size_t)tok * K + k) : zero;
                        const uint32_t p[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t a = p[e] & 0x7fff7fffu;
                            const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&m));
                            m = *reinterpret_cast<const uint32_t*>(&r);
                        }
                    }
                    float largest = fmaxf(low_float(m), high_float(m));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                    largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                    const float scale = fp8_scale(largest), inv = 1.0f / scale;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t p[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            held[j][nt][2 * i + e] = to_e4m3x4(low_float(p[2 * e]) * inv, high_float(p[2 * e]) * inv,
                                                               low_float(p[2 * e + 1]) * inv, high_float(p[2 * e + 1]) * inv);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) held_s[j][nt][e] = __shfl_sync(0xffffffffu, scale, (c * 2 + e) * 4);
                } else {
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int k = kb * kFp8Block + u * 64 + c * 16;
                        const uint4 raw = j < n_kb && tok < M && k < K ? ld_rows((const uint8_t*)x + (size_t)tok * K + k) : zero;
                        held[j][nt][4 * u] = raw.x; held[j][nt][4 * u + 1] = raw.y; held[j][nt][4 * u + 2] = raw.z; held[j][nt][4 * u + 3] = raw.w;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        held_s[j][nt][e] = j < n_kb ? ld_scale(sx + (size_t)min(nt * 8 + c * 2 + e, M - 1) * kb_all + kb) : 0.0f;
                }
            }
    }

    float acc[NT][4];
    int stage = 0;
    // the block of 128 in the oldest stage, against `xq` and `ts` (or the rows beside it)
    auto multiply = [&](const uint32_t (&hx)[NT][8], const float (&hs)[NT][2]) {
        __syncwarp();                                            // the stage refilled now has been read by all lanes
        fetch(true);
        cp_async_wait<stages - 1>();
        __syncwarp();
        const unsigned char* tile = ring_p + (size_t)stage * Ring::kStage;
        if (++stage == stages) stage = 0;
        const float* scales = reinterpret_cast<const float*>(tile + kFp8TileBytes + Ring::kX);
        const float w_lo = scales[0], w_hi = GATED ? scales[1] : w_lo;
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) part[nt][0] = part[nt][1] = part[nt][2] = part[nt][3] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint4 lo = *reinterpret_cast<const uint4*>(tile + tile_at(rq, 4 * u + c));
            const uint4 hi = *reinterpret_cast<const uint4*>(tile + tile_at(rq + 8, 4 * u + c));
            const uint32_t l[4] = {lo.x, lo.y, lo.z, lo.w}, h[4] = {hi.x, hi.y, hi.z, hi.w};
            uint32_t xw[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                if (KPW != 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) xw[nt][i] = hx[nt][4 * u + i];
                } else {
                    const uint4 raw = *reinterpret_cast<const uint4*>(tile + kFp8TileBytes + tile_at(nt * 8 + rq, 4 * u + c));
                    xw[nt][0] = raw.x; xw[nt][1] = raw.y; xw[nt][2] = raw.z; xw[nt][3] = raw.w;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t a[4];
                e4m3x4_to_half2(l[i], a[0], a[2]);
                e4m3x4_to_half2(h[i], a[1], a[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t b[2];
                    e4m3x4_to_half2(xw[nt][i], b[0], b[1]);
                    mma_f16_16816(part[nt], a, b);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const float t0 = KPW != 0 ? hs[nt][0] : scales[4 + nt * 8 + c * 2], t1 = KPW != 0 ? hs[nt][1] : scales[4 + nt * 8 + c * 2 + 1];
            acc[nt][0] = fmaf(part[nt][0], w_lo * t0, acc[nt][0]);
            acc[nt][1] = fmaf(part[nt][1], w_lo * t1, acc[nt][1]);
            acc[nt][2] = fmaf(part[nt][2], w_hi * t0, acc[nt][2]);
            acc[nt][3] = fmaf(part[nt][3], w_hi * t1, acc[nt][3]);
        }
    };

    int buf = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, buf ^= 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
        if constexpr (KPW != 0) {
#pragma unroll
            for (int j = 0; j < KPW; ++j)
                if (j < n_kb) multiply(held[j], held_s[j]);
        } else {
            for (int j = 0; j < n_kb; ++j) multiply(held[0], held_s[0]);
        }
        // ---- the warps' sums, added in warp order (two buffers: the next tile's sums may come while these are read)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            red[buf][warp][rq][nt * 8 + c * 2] = acc[nt][0];
            red[buf][warp][rq][nt * 8 + c * 2 + 1] = acc[nt][1];
            red[buf][warp][rq + 8][nt * 8 + c * 2] = acc[nt][2];
            red[buf][warp][rq + 8][nt * 8 + c * 2 + 1] = acc[nt][3];
        }
        __syncthreads();
        constexpr int kCols = GATED ? 8 : 16;
        for (int idx = threadIdx.x; idx < kCols * NT * 8; idx += blockDim.x) {
            const int row = idx % kCols, tok = idx / kCols, col = tile * kCols + row;
            if (tok < M && col < N) {
                float s = 0.0f;
#pragma unroll
                for (int ww = 0; ww < kFp8Warps; ++ww) s += red[buf][ww][row][tok];
                if (GATED) {
                    float up = 0.0f;
#pragma unroll
                    for (int ww = 0; ww < kFp8Warps; ++ww) up += red[buf][ww][row + 8][tok];
                    s = gated_unit(s, up, act, gc);
                }
                y[(size_t)tok * N + col] = from_f32<TOut>(s);
            }
        }
    }
    cp_async_wait<0>();
}

template <int NT, int KPW, bool XBF16, bool GATED, typename TOut>
static int launch_fp8_skinny(const void* x, const float* sx, const void* w, const float* sw, void* y, int M, int N, int K, int act,
                             GateConst gc, cudaStream_t stream) {
    using Ring = Fp8Ring<NT, KPW>;
    constexpr size_t smem = Ring::kBytes;
    auto kernel = fp8_skinny_kernel<NT, KPW, XBF16, GATED, TOut>;
    static OncePerDevice configured;
    if (configured.first()) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) { set_error("fp8_skinny: %s", cudaGetErrorString(e)); return (int)e; }
        configured.done();
    }
    const long long tiles = ((GATED ? 2ll * N : N) + kFp8TileRows - 1) / kFp8TileRows;
    int sms = sm_count_cached();
    if (sms <= 0) sms = 148;
    const long long resident = (long long)Ring::kBlocks * sms;
    const unsigned grid = (unsigned)(tiles < resident ? tiles : resident);
    launch_pdl(kPdlAlways, kernel, dim3(grid), dim3(kFp8Warps * 32), smem, stream, x, sx, (const uint8_t*)w, sw, (TOut*)y, M, N, K, (int)tiles,
               act, gc);
    return finish_launch("fp8_skinny");
}

template <bool GATED, typename TOut>
static int dispatch_fp8_skinny(const void* x, const float* sx, const void* w, const float* sw, void* y, int M, int N, int K, int act,
                               GateConst gc, cudaStream_t stream) {
    const int per_warp = ((K + kFp8Block - 1) / kFp8Block + kFp8Warps - 1) / kFp8Warps;
#define SKINNY(NT, KPW, XB) return launch_fp8_skinny<NT, KPW, XB, GATED, TOut>(x, sx, w, sw, y, M, N, K, act, gc, stream)
    if (sx == nullptr) {
        if (per_warp <= 2) SKINNY(1, 2, true);
        SKINNY(1, 4, true);
    }
    if (M <= 8) {
        if (per_warp <= 2) SKINNY(1, 2, false);
        if (per_warp <= 4) SKINNY(1, 4, false);
        SKINNY(1, 0, false);
    }
    SKINNY(2, 0, false);
#undef SKINNY
}

}  // namespace tllm

using namespace tllm;

// y[M, N] (out_dtype) = x . w^T for M <= 16.  sx null: x is [M, K] bfloat16, rounded inside (M <= 8, K <= 4096); else x e4m3 with
// scales [M, ceil(K / 128)].  w [N, K] e4m3, sw [ceil(N / 128), ceil(K / 128)].  gated: w has 2 N rows, gate and up interleaved by eight, sw
// [2 ceil(N / 128), ceil(K / 128)], y float32 = act(gate) * up.  K a multiple of 16, x and w 16-byte aligned.
extern "C" int tllm_fp8_skinny(const void* x, const float* sx, const void* w, const float* sw, void* y, int out_dtype, int M, int N, int K,
                               int gated, int act, float limit, float slope, cudaStream_t stream) {
    TLLM_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 16 == 0, "fp8_skinny: %d x %d x %d (K a multiple of 16)", M, N, K);
    TLLM_REQUIRE(M <= 16 && (sx != nullptr || (M <= 8 && K <= 4096)), "fp8_skinny: %d rows, K = %d", M, K);
    TLLM_REQUIRE(N <= 0x3fffffff, "fp8_skinny: %d columns", N);
    TLLM_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15u) == 0, "fp8_skinny: operands must be 16-byte aligned");
    TLLM_REQUIRE(out_dtype == kBF16 || out_dtype == kF32, "fp8_skinny: unknown output dtype");
    TLLM_REQUIRE(!gated || (N % 8 == 0 && out_dtype == kF32 && gated_act_ok(act, limit)), "fp8_skinny: bad gated product");
    if (M == 0) return 0;
    const GateConst gc{limit, slope};
    if (gated) return dispatch_fp8_skinny<true, float>(x, sx, w, sw, y, M, N, K, act, gc, stream);
    if (out_dtype == kF32) return dispatch_fp8_skinny<false, float>(x, sx, w, sw, y, M, N, K, act, gc, stream);
    return dispatch_fp8_skinny<false, bf16>(x, sx, w, sw, y, M, N, K, act, gc, stream);
}
