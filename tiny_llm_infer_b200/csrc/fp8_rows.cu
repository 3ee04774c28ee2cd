// Rows and weights in 8 bits: e4m3 values with a float32 scale per 128 columns of a row, or per 128 x 128 of a weight (fp8.cuh has
// the scale).  Three kernels make rows for the products of fp8_skinny.cu and fp8_tcgen05.cu: from rows as they are, from the
// residual stream (sum and RMSNorm in the same pass), and from gate and up sums (the activation in the same pass); what they round
// is float32, never first bfloat16.
#include "fp8.cuh"

namespace tllm {

template <typename T> __device__ __forceinline__ void load8(const T* p, float (&v)[8]);
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&v)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
template <> __device__ __forceinline__ void load8<bf16>(const bf16* p, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// Sixteen lanes make one block of 128: eight columns each, one 16-byte read (bfloat16), one 8-byte write; PER blocks, all their reads on their
// way at once.  Bound by HBM or, for a few rows, by its launch.
template <typename T, int PER>
__global__ void __launch_bounds__(256) fp8_rows_kernel(const T* x, uint8_t* __restrict__ q, float* __restrict__ scales, int K, unsigned kb,
                                                       unsigned blocks) {
    TLLM_PDL_ENTER();
    const int lane16 = threadIdx.x & 15;
    const unsigned first = blockIdx.x * PER * (blockDim.x >> 4) + (threadIdx.x >> 4);
    float v[PER][8];
    long long at[PER];                                           // of the lane's columns; negative: none
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const unsigned b = first + i * (blockDim.x >> 4), row = b / kb;
        const int col = (int)(b - row * kb) * kFp8Block + lane16 * 8;
        at[i] = b < blocks && col < K ? (long long)row * K + col : -1;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
        if (at[i] >= 0) load8<T>(x + at[i], v[i]);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const unsigned b = first + i * (blockDim.x >> 4);
        const float s = fp8_scale(half_warp_max(largest8(v[i])));
        if (at[i] >= 0) *reinterpret_cast<uint2*>(q + at[i]) = to_e4m3x8(v[i], 1.0f / s);
        if (lane16 == 0 && b < blocks) scales[b] = s;
    }
}

// act(gate) * up of sums that lie interleaved by eight ([rows][2 I]: eight gate, their eight up, ...), summed over `splits` shares of
// K one after the other, as 8-bit rows.  Sixteen lanes make a block of 128 outputs, eight each, from sixteen neighbouring sums.
__global__ void __launch_bounds__(256) fp8_gated_rows_kernel(const float* sums, int splits, long long share, uint8_t* __restrict__ q,
                                                             float* __restrict__ scales, int inter, unsigned ib, unsigned blocks, int act,
                                                             GateConst gc) {
    TLLM_PDL_ENTER();
    const int lane16 = threadIdx.x & 15;
    const unsigned b = blockIdx.x * (blockDim.x >> 4) + (threadIdx.x >> 4), in_row = b / ib;
    const size_t row = in_row;
    const int col = (int)(b - in_row * ib) * kFp8Block + lane16 * 8;
    const bool live = b < blocks && col < inter;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live) {
        const float* p = sums + (row * inter + col) * 2;
        float g[8], u[8], t[8];
        load8<float>(p, g);
        load8<float>(p + 8, u);
        for (int i = 1; i < splits; ++i) {
            load8<float>(p + i * share, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] += t[e];
            load8<float>(p + i * share + 8, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) u[e] += t[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = gated_unit(g[e], u[e], act, gc);
    }
    const float s = fp8_scale(half_warp_max(largest8(v)));
    const float inv = 1.0f / s;
    if (live) *reinterpret_cast<uint2*>(q + row * inter + col) = to_e4m3x8(v, inv);
    if (lane16 == 0 && b < blocks) scales[b] = s;
}

// h[r] += delta[r] (float32, written back), then the row gain * h / sqrt(mean(h^2) + eps) in 8 bits.  One thread block per row, the
// row in registers between its sum and its scaling (CHUNKS groups of eight columns per thread); sixteen neighbouring threads hold a
// block of 128 columns, so its largest magnitude takes four shuffles.
template <typename TD, typename TG, int CHUNKS>
__global__ void __launch_bounds__(CHUNKS == 4 ? 1024 : 512)
add_rmsnorm_fp8_kernel(float* h, const TD* delta, const TG* __restrict__ gain, float eps, uint8_t* __restrict__ q,
                       float* __restrict__ scales, int width) {
    __shared__ float scratch[32];
    TLLM_PDL_ENTER();
    const int r = blockIdx.x, n_chunks = width >> 3, kb = (width + kFp8Block - 1) / kFp8Block;
    float* hr = h + (size_t)r * width;
    const TD* dr = delta ? delta + (size_t)r * width : nullptr;
    float v[CHUNKS][8], d[CHUNKS][8];
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        if (c < n_chunks) {
            load8<float>(hr + c * 8, v[j]);
            if (dr) load8<TD>(dr + c * 8, d[j]);
        }
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        if (c < n_chunks) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (dr) v[j][e] += d[j][e];
                sum += v[j][e] * v[j][e];
            }
            if (dr) {
                *reinterpret_cast<float4*>(hr + c * 8) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
                *reinterpret_cast<float4*>(hr + c * 8 + 4) = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
            }
        }
    }
    sum = block_sum(sum, scratch);
    const float scale = 1.0f / sqrtf(sum / (float)width + eps);
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j) {
        const int c = threadIdx.x + j * blockDim.x;
        const bool live = c < n_chunks;
        float g[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (live) {
            load8<TG>(gain + c * 8, g);
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = g[e] * v[j][e] * scale;
        }
        const float s = fp8_scale(half_warp_max(largest8(g)));   // every thread of the block takes part
        if (live) {
            *reinterpret_cast<uint2*>(q + (size_t)r * width + c * 8) = to_e4m3x8(g, 1.0f / s);
            if ((c & 15) == 0) scales[(size_t)r * kb + (c >> 4)] = s;
        }
    }
}

// One block of 128 x 128 of a weight per thread block.  GATED: q's rows are gate and up rows interleaved by eight (x has them so already); the
// scales' rows are a block of 128 gate rows, the block of their up rows, and so on.
template <typename T>
__global__ void __launch_bounds__(256) fp8_weight_kernel(const T* __restrict__ w, uint8_t* __restrict__ q, float* __restrict__ scales, int N,
                                                         int K, int kb, int gated) {
    __shared__ float scratch[8];
    const int b = blockIdx.y, k0 = blockIdx.x * kFp8Block;
    const int warp = threadIdx.x >> 5, lane16 = threadIdx.x & 15, half = threadIdx.x >> 4;       // 16 rows at a time, 8 columns a thread
    const int col = k0 + lane16 * 8;
    auto row_of = [&](int i) {                                  // i-th row of the block's 128, or N for none
        if (!gated) return min(b * kFp8Block + i, N);
        const int j = (b >> 1) * kFp8Block + i;                 // index among the gate (or up) rows
        return j < N / 2 ? 16 * (j >> 3) + (j & 7) + 8 * (b & 1) : N;
    };
    float largest = 0.0f, v[8];
    for (int i = half; i < kFp8Block; i += 16) {
        const int row = row_of(i);
        if (row < N && col < K) {
            load8<T>(w + (size_t)row * K + col, v);
            largest = fmaxf(largest, largest8(v));
        }
    }
    largest = warp_max(largest);
    if ((threadIdx.x & 31) == 0) scratch[warp] = largest;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = fmaxf(largest, scratch[i]);
    const float s = fp8_scale(largest), inv = 1.0f / s;
    for (int i = half; i < kFp8Block; i += 16) {
        const int row = row_of(i);
        if (row < N && col < K) {
            load8<T>(w + (size_t)row * K + col, v);
            *reinterpret_cast<uint2*>(q + (size_t)row * K + col) = to_e4m3x8(v, inv);
        }
    }
    if (threadIdx.x == 0) scales[(size_t)b * kb + blockIdx.x] = s;
}

// Nothing, by an ordinary launch: it starts when all before it in the stream has ended and is in memory, and lets nothing start early.
__global__ void fp8_settle_kernel() {}

template <typename TD, typename TG>
static int launch_add_rmsnorm_fp8(float* h, const void* delta, const void* gain, float eps, void* q, float* scales, int rows, int width,
                                  cudaStream_t stream) {
    const int n_chunks = width / 8;
#define NORM8(C, BLOCK)                                                                                                  \
    launch_pdl(kPdlNorm, add_rmsnorm_fp8_kernel<TD, TG, C>, dim3(rows), dim3(BLOCK), 0, stream, h, (const TD*)delta,       \
               (const TG*)gain, eps, (uint8_t*)q, scales, width)
    const int one = (n_chunks + 31) / 32 * 32, two = ((n_chunks + 1) / 2 + 31) / 32 * 32;
    if (one <= 512) NORM8(1, one);
    else if (two <= 512) NORM8(2, two);
    else NORM8(4, 1024);
#undef NORM8
    return finish_launch("add_rmsnorm_fp8");
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace tllm

using namespace tllm;

// x [rows, K] (dtype) -> q [rows, K] e4m3, scales [rows, ceil(K / 128)] float32.  K a multiple of 16, x and q 16-byte aligned.
extern "C" int tllm_fp8_rows(const void* x, int dtype, void* q, float* scales, int rows, int K, cudaStream_t stream) {
    TLLM_REQUIRE(rows >= 0 && K > 0 && K % 16 == 0, "fp8_rows: %d rows of %d columns (a multiple of 16)", rows, K);
    TLLM_REQUIRE(dtype == kF32 || dtype == kBF16, "fp8_rows: unknown dtype %d", dtype);
    TLLM_REQUIRE(aligned16(x) && aligned16(q), "fp8_rows: operands must be 16-byte aligned");
    if (rows == 0) return 0;
    const int kb = (K + kFp8Block - 1) / kFp8Block;
    const long long blocks = (long long)rows * kb, grid = (blocks + 15) / 16;
    TLLM_REQUIRE(blocks <= 0x7fffffff, "fp8_rows: too many rows");
    // four blocks a lane once that leaves every SM four thread blocks and more
    const bool four = grid >= 4 * 4 * 148;
    const unsigned n = (unsigned)(four ? (blocks + 63) / 64 : grid);
#define ROWS8(T, PER) launch_pdl(kPdlAlways, fp8_rows_kernel<T, PER>, dim3(n), dim3(256), 0, stream, (const T*)x, (uint8_t*)q, scales, K, (unsigned)kb, (unsigned)blocks)
    if (dtype == kF32) {
        if (four) ROWS8(float, 4); else ROWS8(float, 1);
    } else {
        if (four) ROWS8(bf16, 4); else ROWS8(bf16, 1);
    }
#undef ROWS8
    return finish_launch("fp8_rows");
}

// sums float32 [splits][rows][2 inter] (gate and up interleaved by eight) -> act(gate) * up as q [rows, inter] e4m3 and scales
// [rows, ceil(inter / 128)].  inter a multiple of 8.
extern "C" int tllm_fp8_gated_rows(const float* sums, int splits, void* q, float* scales, int rows, int inter, int act, float limit,
                                   float slope, cudaStream_t stream) {
    TLLM_REQUIRE(rows >= 0 && inter > 0 && inter % 8 == 0 && splits > 0, "fp8_gated_rows: bad sizes");
    TLLM_REQUIRE(gated_act_ok(act, limit), "fp8_gated_rows: unknown activation %d", act);
    TLLM_REQUIRE(aligned16(sums) && aligned16(q), "fp8_gated_rows: operands must be 16-byte aligned");
    if (rows == 0) return 0;
    const int ib = (inter + kFp8Block - 1) / kFp8Block;
    const long long blocks = (long long)rows * ib, grid = (blocks + 15) / 16;
    TLLM_REQUIRE(blocks <= 0x7fffffff, "fp8_gated_rows: too many rows");
    launch_pdl(kPdlAlways, fp8_gated_rows_kernel, dim3((unsigned)grid), dim3(256), 0, stream, sums, splits, (long long)rows * inter * 2,
               (uint8_t*)q, scales, inter, (unsigned)ib, (unsigned)blocks, act, GateConst{limit, slope});
    return finish_launch("fp8_gated_rows");
}

// h [rows, width] float32, delta null or [rows, width] (dtype): see add_rmsnorm_fp8_kernel.  width a multiple of 16, at most 32768.
extern "C" int tllm_add_rmsnorm_fp8(float* h, const void* delta, int dtype, const void* gain, int gain_dtype, float eps, void* q,
                                    float* scales, int rows, int width, cudaStream_t stream) {
    TLLM_REQUIRE(rows >= 0 && width > 0 && width % 16 == 0 && width <= 32768,
                 "add_rmsnorm_fp8: %d rows of width %d (a multiple of 16 up to 32768)", rows, width);
    TLLM_REQUIRE(eps > 0.0f, "add_rmsnorm_fp8: eps must be positive");
    TLLM_REQUIRE((dtype == kF32 || dtype == kBF16) && (gain_dtype == kF32 || gain_dtype == kBF16), "add_rmsnorm_fp8: unknown dtype");
    TLLM_REQUIRE(aligned16(h) && aligned16(delta) && aligned16(gain) && aligned16(q), "add_rmsnorm_fp8: operands must be 16-byte aligned");
    if (rows == 0) return 0;
    if (dtype == kBF16)
        return gain_dtype == kBF16 ? launch_add_rmsnorm_fp8<bf16, bf16>(h, delta, gain, eps, q, scales, rows, width, stream)
                                   : launch_add_rmsnorm_fp8<bf16, float>(h, delta, gain, eps, q, scales, rows, width, stream);
    return gain_dtype == kBF16 ? launch_add_rmsnorm_fp8<float, bf16>(h, delta, gain, eps, q, scales, rows, width, stream)
                               : launch_add_rmsnorm_fp8<float, float>(h, delta, gain, eps, q, scales, rows, width, stream);
}

// Between what wrote a weight's tensors and its first product: the weight-streaming product fetches weights before the kernel ahead of it has
// ended, and the kernels that make rows let it start at once.
extern "C" int tllm_fp8_settle(cudaStream_t stream) {
    fp8_settle_kernel<<<1, 32, 0, stream>>>();
    return finish_launch("fp8_settle");
}

// w [N, K] (dtype) -> q [N, K] e4m3, scales [ceil(N / 128), ceil(K / 128)]; gated (N / 2 gate and N / 2 up rows interleaved by eight):
// scales [2 ceil(N / 2 / 128), ceil(K / 128)].
extern "C" int tllm_fp8_weight(const void* w, int dtype, void* q, float* scales, int N, int K, int gated, cudaStream_t stream) {
    TLLM_REQUIRE(N > 0 && K > 0 && K % 16 == 0, "fp8_weight: %d x %d (columns a multiple of 16)", N, K);
    TLLM_REQUIRE(!gated || N % 16 == 0, "fp8_weight: interleaved gate and up rows come in sixteens, N = %d", N);
    TLLM_REQUIRE(dtype == kF32 || dtype == kBF16, "fp8_weight: unknown dtype %d", dtype);
    TLLM_REQUIRE(aligned16(w) && aligned16(q), "fp8_weight: operands must be 16-byte aligned");
    const int kb = (K + kFp8Block - 1) / kFp8Block;
    const int nb = gated ? 2 * ((N / 2 + kFp8Block - 1) / kFp8Block) : (N + kFp8Block - 1) / kFp8Block;
    TLLM_REQUIRE(nb <= 65535, "fp8_weight: %d rows are too many", N);
    if (dtype == kF32)
        fp8_weight_kernel<float><<<dim3(kb, nb), 256, 0, stream>>>((const float*)w, (uint8_t*)q, scales, N, K, kb, gated);
    else
        fp8_weight_kernel<bf16><<<dim3(kb, nb), 256, 0, stream>>>((const bf16*)w, (uint8_t*)q, scales, N, K, kb, gated);
    return finish_launch("fp8_weight");
}
