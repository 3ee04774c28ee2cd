// The products with 8-bit weights as one call each: rows brought to 8 bits where they are not, the product by the kernel that the caller
// chose, its shares added.  A call from Python costs several microseconds, as long as the short kernels take.
#include "fp8.cuh"

extern "C" {
int tllm_fp8_rows(const void* x, int dtype, void* q, float* scales, int rows, int K, cudaStream_t stream);
int tllm_fp8_gated_rows(const float* sums, int splits, void* q, float* scales, int rows, int inter, int act, float limit, float slope,
                        cudaStream_t stream);
int tllm_fp8_skinny(const void* x, const float* sx, const void* w, const float* sw, void* y, int out_dtype, int M, int N, int K, int gated, int act,
                    float limit, float slope, cudaStream_t stream);
int tllm_fp8_tcgen05(const void* x, const float* sx, const void* w, const float* sw, void* y, float* y_scales, int M, int N, int K, int form,
                     int interleaved, int pairs, int splits, int kb_per_split, int act, float limit, float slope, int* error_word, cudaStream_t stream);
int tllm_fp8_join(const float* shares, int splits, long long n, void* y, int out_dtype, cudaStream_t stream);
}

using namespace tllm;

// Routes: the weight-streaming kernel, tiles of 128 x 128 (with `splits` shares of `each` blocks of K), pairs of SMs.
enum Fp8Route : int { kRouteSkinny = 0, kRouteTiles = 1, kRoutePairs = 2 };
constexpr int kRows8 = 2, kRowsInside = 3;      // x_kind beside kF32 and kBF16: rows in 8 bits; bfloat16 that the streaming kernel rounds itself

static size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

// Rows in 8 bits: as they come (sx), or made in `scratch`, which moves on behind them.
static int fp8_bring_rows(const void*& x, const float*& sx, int x_kind, int M, int K, unsigned char*& scratch, cudaStream_t stream) {
    if (x_kind == kRows8 || x_kind == kRowsInside) return 0;
    unsigned char* q = scratch;
    float* s = reinterpret_cast<float*>(q + up16((size_t)M * K));
    scratch = reinterpret_cast<unsigned char*>(s) + up16((size_t)M * ((K + kFp8Block - 1) / kFp8Block) * 4);
    const int rc = tllm_fp8_rows(x, x_kind, q, s, M, K, stream);
    x = q;
    sx = s;
    return rc;
}

// y[M, N] (out_dtype) = x . w^T.  scratch: 16-byte aligned; rows in 8 bits (x_kind float32 or bfloat16) M K + 4 M ceil(K / 128) bytes, each rounded
// up to 16, then float32 [splits][M][N] if there is more than one share or y is float32 (route kRouteTiles).
extern "C" int tllm_fp8_linear(const void* x, const float* sx, int x_kind, const void* w, const float* sw, void* y, int out_dtype, int M, int N, int K,
                               int route, int splits, int each, void* scratch, int* error_word, cudaStream_t stream) {
    TLLM_REQUIRE(M > 0 && x_kind >= kF32 && x_kind <= kRowsInside && (x_kind != kRows8 || sx), "fp8_linear: bad rows");
    TLLM_REQUIRE(x_kind == kRows8 || x_kind == kRowsInside || scratch, "fp8_linear: rows in 8 bits need scratch");
    unsigned char* at = (unsigned char*)scratch;
    if (x_kind == kRowsInside) sx = nullptr;
    int rc = fp8_bring_rows(x, sx, x_kind, M, K, at, stream);
    if (rc != 0) return rc;
    if (route == kRouteSkinny) return tllm_fp8_skinny(x, sx, w, sw, y, out_dtype, M, N, K, 0, 0, 0.0f, 0.0f, stream);
    TLLM_REQUIRE(x_kind != kRowsInside, "fp8_linear: only the streaming kernel rounds rows itself");
    const bool shares = splits > 1 || out_dtype != kBF16;
    TLLM_REQUIRE(!shares || (route == kRouteTiles && at), "fp8_linear: shares need scratch and tiles of 128 x 128");
    if (!shares) return tllm_fp8_tcgen05(x, sx, w, sw, y, nullptr, M, N, K, 0, 0, route == kRoutePairs, 1, each, 0, 0.0f, 0.0f, error_word, stream);
    rc = tllm_fp8_tcgen05(x, sx, w, sw, at, nullptr, M, N, K, 1, 0, 0, splits, each, 0, 0.0f, 0.0f, error_word, stream);
    if (rc != 0) return rc;
    return tllm_fp8_join((const float*)at, splits, (long long)M * N, y, out_dtype, stream);
}

// act(x . gate^T) * (x . up^T) as e4m3 [M, inter] with scales [M, ceil(inter / 128)], w the 2 inter interleaved rows.  scratch: rows in 8 bits as
// above, then float32 [M][inter] (route kRouteSkinny) or [splits][M][2 inter] (kRouteTiles).
extern "C" int tllm_fp8_gated(const void* x, const float* sx, int x_kind, const void* w, const float* sw, void* out, float* out_scales, int M, int inter,
                              int K, int route, int splits, int each, int act, float limit, float slope, void* scratch, int* error_word,
                              cudaStream_t stream) {
    TLLM_REQUIRE(M > 0 && x_kind >= kF32 && x_kind <= kRowsInside && (x_kind != kRows8 || sx), "fp8_gated: bad rows");
    TLLM_REQUIRE(scratch || (route == kRoutePairs && x_kind == kRows8), "fp8_gated: no scratch");
    TLLM_REQUIRE(x_kind != kRowsInside || route == kRouteSkinny, "fp8_gated: only the streaming kernel rounds rows itself");
    unsigned char* at = (unsigned char*)scratch;
    if (x_kind == kRowsInside) sx = nullptr;
    int rc = fp8_bring_rows(x, sx, x_kind, M, K, at, stream);
    if (rc != 0) return rc;
    if (route == kRouteSkinny) {
        rc = tllm_fp8_skinny(x, sx, w, sw, at, kF32, M, inter, K, 1, act, limit, slope, stream);
        return rc != 0 ? rc : tllm_fp8_rows(at, kF32, out, out_scales, M, inter, stream);
    }
    if (route == kRoutePairs)
        return tllm_fp8_tcgen05(x, sx, w, sw, out, out_scales, M, 2 * inter, K, 2, 1, 1, 1, each, act, limit, slope, error_word, stream);
    rc = tllm_fp8_tcgen05(x, sx, w, sw, at, nullptr, M, 2 * inter, K, 1, 1, 0, splits, each, 0, 0.0f, 0.0f, error_word, stream);
    return rc != 0 ? rc : tllm_fp8_gated_rows((const float*)at, splits, out, out_scales, M, inter, act, limit, slope, stream);
}
