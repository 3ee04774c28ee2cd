// y[M, N] = x . w^T for a handful of rows with an 8-bit weight: x as e4m3 rows with a scale per 128 columns, w as e4m3 with a scale
// per 128 x 128 (fp8.cuh),
//
//   y[t, n] = sum_b sx[t, b] sw[n / 128, b] sum_{k in block b} qx[t, k] qw[n, k],
//
// the product of a decode step, where every weight is read once: the time is HBM's, half of what the bfloat16 weights take
// (gemm_skinny.cu, whose layout this kernel shares).  A thread block owns 16 rows of w and its eight warps split K.  A lane reads 16
// contiguous bytes of a weight row, sixteen k's, and turns them into pairs of float16, which hold every e4m3 value exactly; the four
// lanes of a quad cover 64 k's, two such reads a block of 128.  The k's of a lane stand for the columns that the fragment layout of
// mma.sync m16n8k16 assigns to it, on both sides alike.  The 128 products of a block are summed in float32 (each is exact), then
// scaled and added to the running float32 sum.
//
// Rows may come in bfloat16 (XBF16): the quad that multiplies a block of a row holds all of its 128 numbers, so it finds the scale
// and rounds them itself, which saves a launch; every thread block repeats that for all of x.
//
// Launched early (programmatic dependent launch) like gemm_skinny.cu: weights are fetched before the wait, x after it.
#include "fp8.cuh"
#include "mma_tiles.cuh"

namespace tllm {

constexpr int kFp8Warps = 8;

__device__ __forceinline__ uint4 ld_weights(const void* p) {
    uint4 v;
    asm volatile("ld.global.cs.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
// What the kernel ahead has written: ordinary loads, after the wait.
__device__ __forceinline__ uint4 ld_rows(const void* p) {
    uint4 v;
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ float ld_scale(const float* p) {
    float v;
    asm volatile("ld.global.f32 %0, [%1];\n" : "=f"(v) : "l"(p) : "memory");
    return v;
}

template <int NT, bool XBF16>
struct Fp8Stage {
    uint4 lo[2], hi[2];                         // two reads of 64 k's: row rq and row rq + 8 of the block's sixteen
    uint4 x[NT][XBF16 ? 4 : 2];
    float w_lo, w_hi, s[NT][XBF16 ? 1 : 2];     // scales of the weight rows; of the tokens whose sums this lane holds
};

// GATED: w holds N gate and N up rows interleaved by eight, y [M, N] is act(gate) * up; the tile's upper half are eight gate rows,
// its lower half their up rows, whose scales lie in neighbouring rows of `sw`.
template <int NT, bool XBF16, bool GATED, int STAGES, typename TOut>
__global__ void __launch_bounds__(kFp8Warps * 32)
fp8_skinny_kernel(const void* x, const float* sx, const uint8_t* __restrict__ w, const float* __restrict__ sw, TOut* y, int M, int N,
                  int K, int act, GateConst gc) {
    __shared__ float red[kFp8Warps][16][NT * 8 + 1];
    TLLM_PDL_TRIGGER();
    const int r0 = blockIdx.x * (GATED ? 8 : 16);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, rq = lane >> 2;
    const size_t lo_row = GATED ? (size_t)2 * r0 + rq : (size_t)min(r0 + rq, N - 1);
    const size_t hi_row = GATED ? lo_row + 8 : (size_t)min(r0 + rq + 8, N - 1);
    const uint8_t *w_lo = w + lo_row * K, *w_hi = w + hi_row * K;
    const int kb_all = (K + kFp8Block - 1) / kFp8Block;
    // sixteen rows never straddle a block of 128; of a gated weight the gate block's scales are followed by the up block's
    const float* sw_lo = sw + (size_t)(r0 / kFp8Block) * (GATED ? 2 : 1) * kb_all;
    const float* sw_hi = GATED ? sw_lo + kb_all : sw_lo;
    const uint8_t* xr[NT];
    bool xv[NT];
    const float* sxr[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int tok = nt * 8 + rq;
        xv[nt] = tok < M;
        xr[nt] = (const uint8_t*)x + (size_t)(xv[nt] ? tok : 0) * K * (XBF16 ? 2 : 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) sxr[nt][e] = XBF16 ? nullptr : sx + (size_t)min(nt * 8 + c * 2 + e, M - 1) * kb_all;
    }
    float acc[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.0f;
    const int per_warp = (kb_all + kFp8Warps - 1) / kFp8Warps;
    const int kb0 = warp * per_warp, kb1 = min(kb_all, kb0 + per_warp);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    using Stage = Fp8Stage<NT, XBF16>;

    auto load_w = [&](Stage& s, int kb) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int k = kb * kFp8Block + u * 64 + c * 16;
            const bool ok = kb < kb1 && k < K;
            s.lo[u] = ok ? ld_weights(w_lo + k) : zero;
            s.hi[u] = ok ? ld_weights(w_hi + k) : zero;
        }
        s.w_lo = kb < kb1 ? sw_lo[kb] : 0.0f;
        s.w_hi = GATED ? (kb < kb1 ? sw_hi[kb] : 0.0f) : s.w_lo;
    };
    auto load_x = [&](Stage& s, int kb) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int k = kb * kFp8Block + u * 64 + c * 16;
                const bool ok = kb < kb1 && k < K && xv[nt];
                if (XBF16) {
                    s.x[nt][2 * u] = ok ? ld_rows(xr[nt] + 2 * k) : zero;
                    s.x[nt][(2 * u + 1) % (XBF16 ? 4 : 2)] = ok ? ld_rows(xr[nt] + 2 * k + 16) : zero;
                } else {
                    s.x[nt][u] = ok ? ld_rows(xr[nt] + k) : zero;
                }
            }
            if constexpr (!XBF16) {
#pragma unroll
                for (int e = 0; e < 2; ++e) s.s[nt][e] = kb < kb1 ? ld_scale(sxr[nt][e] + kb) : 0.0f;
            }
        }
    };
    auto multiply = [&](Stage& s) {
        uint32_t xq[NT][8];                     // this lane's k's of a token: eight words of four e4m3
        float ts[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if constexpr (XBF16) {
                uint32_t m = 0;                 // largest magnitudes of the pairs
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t p[4] = {s.x[nt][i].x, s.x[nt][i].y, s.x[nt][i].z, s.x[nt][i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t a = p[j] & 0x7fff7fffu;
                        __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&m));
                        m = *reinterpret_cast<uint32_t*>(&r);
                    }
                }
                float largest = fmaxf(low_float(m), high_float(m));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                const float scale = fp8_scale(largest), inv = 1.0f / scale;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t p[4] = {s.x[nt][i].x, s.x[nt][i].y, s.x[nt][i].z, s.x[nt][i].w};
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        xq[nt][2 * i + j] = to_e4m3x4(low_float(p[2 * j]) * inv, high_float(p[2 * j]) * inv,
                                                      low_float(p[2 * j + 1]) * inv, high_float(p[2 * j + 1]) * inv);
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) ts[nt][e] = __shfl_sync(0xffffffffu, scale, (c * 2 + e) * 4);
            } else {
                const uint32_t p[8] = {s.x[nt][0].x, s.x[nt][0].y, s.x[nt][0].z, s.x[nt][0].w,
                                       s.x[nt][1].x, s.x[nt][1].y, s.x[nt][1].z, s.x[nt][1].w};
#pragma unroll
                for (int i = 0; i < 8; ++i) xq[nt][i] = p[i];
#pragma unroll
                for (int e = 0; e < 2; ++e) ts[nt][e] = s.s[nt][e];
            }
        }
        float part[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) part[nt][0] = part[nt][1] = part[nt][2] = part[nt][3] = 0.0f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t l[4] = {s.lo[u].x, s.lo[u].y, s.lo[u].z, s.lo[u].w}, h[4] = {s.hi[u].x, s.hi[u].y, s.hi[u].z, s.hi[u].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a[4] = {e4m3x2_to_half2(l[i]), e4m3x2_to_half2(h[i]), e4m3x2_to_half2(l[i] >> 16), e4m3x2_to_half2(h[i] >> 16)};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const uint32_t xw = xq[nt][4 * u + i];
                    const uint32_t b[2] = {e4m3x2_to_half2(xw), e4m3x2_to_half2(xw >> 16)};
                    mma_f16_16816(part[nt], a, b);
                }
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            acc[nt][0] = fmaf(part[nt][0], s.w_lo * ts[nt][0], acc[nt][0]);
            acc[nt][1] = fmaf(part[nt][1], s.w_lo * ts[nt][1], acc[nt][1]);
            acc[nt][2] = fmaf(part[nt][2], s.w_hi * ts[nt][0], acc[nt][2]);
            acc[nt][3] = fmaf(part[nt][3], s.w_hi * ts[nt][1], acc[nt][3]);
        }
    };

    Stage st[STAGES];
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) load_w(st[i], kb0 + i);
    TLLM_PDL_WAIT();                             // from here on x may be read, y written
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) load_x(st[i], kb0 + i);
    for (int kb = kb0; kb < kb1; kb += STAGES) {
#pragma unroll
        for (int i = 0; i < STAGES; ++i) {
            constexpr int kLast = STAGES - 1;
            load_w(st[(i + kLast) % STAGES], kb + i + kLast);
            load_x(st[(i + kLast) % STAGES], kb + i + kLast);
            if (kb + i < kb1) multiply(st[i]);   // past its share a stage's scales need not be finite
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        red[warp][rq][nt * 8 + c * 2] = acc[nt][0];
        red[warp][rq][nt * 8 + c * 2 + 1] = acc[nt][1];
        red[warp][rq + 8][nt * 8 + c * 2] = acc[nt][2];
        red[warp][rq + 8][nt * 8 + c * 2 + 1] = acc[nt][3];
    }
    __syncthreads();
    constexpr int kCols = GATED ? 8 : 16;
    for (int idx = threadIdx.x; idx < kCols * NT * 8; idx += blockDim.x) {
        const int row = idx % kCols, tok = idx / kCols;
        if (tok < M && r0 + row < N) {
            float s = 0.0f;
#pragma unroll
            for (int ww = 0; ww < kFp8Warps; ++ww) s += red[ww][row][tok];
            if (GATED) {
                float up = 0.0f;
#pragma unroll
                for (int ww = 0; ww < kFp8Warps; ++ww) up += red[ww][row + 8][tok];
                s = gated_unit(s, up, act, gc);
            }
            y[(size_t)tok * N + r0 + row] = from_f32<TOut>(s);
        }
    }
}

template <int NT, bool XBF16, bool GATED, int STAGES, typename TOut>
static int launch_fp8_skinny(const void* x, const float* sx, const void* w, const float* sw, void* y, int M, int N, int K, int act,
                             GateConst gc, cudaStream_t stream) {
    launch_pdl(kPdlAlways, fp8_skinny_kernel<NT, XBF16, GATED, STAGES, TOut>, dim3(GATED ? (N + 7) / 8 : (N + 15) / 16),
               dim3(kFp8Warps * 32), 0, stream, x, sx, (const uint8_t*)w, sw, (TOut*)y, M, N, K, act, gc);
    return finish_launch("fp8_skinny");
}

}  // namespace tllm

using namespace tllm;

// y[M, N] (out_dtype) = x . w^T for M <= 32.  sx null: x is [M, K] bfloat16, rounded inside (M <= 8); else x e4m3 with scales
// [M, ceil(K / 128)].  w [N, K] e4m3, sw [ceil(N / 128), ceil(K / 128)].  gated: w has 2 N rows, gate and up interleaved by eight, sw
// [2 ceil(N / 128), ceil(K / 128)], y float32 = act(gate) * up.  K a multiple of 16, x and w 16-byte aligned.
extern "C" int tllm_fp8_skinny(const void* x, const float* sx, const void* w, const float* sw, void* y, int out_dtype, int M, int N, int K,
                               int gated, int act, float limit, float slope, cudaStream_t stream) {
    TLLM_REQUIRE(M >= 0 && N > 0 && K > 0 && K % 16 == 0, "fp8_skinny: %d x %d x %d (K a multiple of 16)", M, N, K);
    TLLM_REQUIRE(M <= 32 && (sx != nullptr || M <= 8), "fp8_skinny: %d rows", M);
    TLLM_REQUIRE(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15u) == 0, "fp8_skinny: operands must be 16-byte aligned");
    TLLM_REQUIRE(out_dtype == kBF16 || out_dtype == kF32, "fp8_skinny: unknown output dtype");
    TLLM_REQUIRE(!gated || (N % 8 == 0 && out_dtype == kF32 && gated_act_ok(act, limit)), "fp8_skinny: bad gated product");
    if (M == 0) return 0;
    const GateConst gc{limit, slope};
#define SKINNY(NT, XB, G, ST, T) return launch_fp8_skinny<NT, XB, G, ST, T>(x, sx, w, sw, y, M, N, K, act, gc, stream)
    if (gated) {
        if (sx == nullptr) SKINNY(1, true, true, 3, float);
        if (M <= 8) SKINNY(1, false, true, 3, float);
        if (M <= 16) SKINNY(2, false, true, 3, float);
        SKINNY(4, false, true, 2, float);
    }
    if (out_dtype == kF32) {
        if (sx == nullptr) SKINNY(1, true, false, 3, float);
        if (M <= 8) SKINNY(1, false, false, 3, float);
        if (M <= 16) SKINNY(2, false, false, 3, float);
        SKINNY(4, false, false, 2, float);
    }
    if (sx == nullptr) SKINNY(1, true, false, 3, bf16);
    if (M <= 8) SKINNY(1, false, false, 3, bf16);
    if (M <= 16) SKINNY(2, false, false, 3, bf16);
    SKINNY(4, false, false, 2, bf16);
#undef SKINNY
}
