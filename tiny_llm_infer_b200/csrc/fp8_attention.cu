// Attention of single tokens over a paged cache of 8-bit keys and values, split over the keys and joined; and the pages of prompt
// portions back in bfloat16 for the prompt kernels.
//
// A key is kept as e4m3 values k8 and a float32 scale sk, a value as v8 and sv (fp8.cuh; one scale per token and head).  With base-2
// scores s_j = (q . k8_j) sk_j scale log2(e),
//
//   out = sum_j 2^(s_j) sv_j v8_j / sum_j 2^(s_j).
//
// One block of threads owns (row, key/value head, run of keys): the query heads of the group are the rows of a 16-row tile, so a key and its
// value come from HBM once per group: 2 hd + 8 bytes, half of the bfloat16 cache's.  What bounds it is their way from HBM.  Each of
// the four warps walks every fourth tile of 16 keys: cp.async brings the tile's keys, values and scales into the warp's own ring; keys that do
// not count (behind the row's position, before its window, without a page) arrive as zeros, so that what a page held before
// meets no sum.
//
// Products run on mma.sync m16n8k16 with float16 operands, which hold every e4m3 value exactly: queries are brought to float16 by a power
// of two per head that puts the largest at 2^14 to 2^15, exact down to 2^-28 of the largest.  A lane's sixteen neighbouring
// bytes of a key stand for the columns that four fragments assign to it, on the query's side alike, so keys need no rearrangement.  For
// P V the fragments want two keys side by side: bytes of two keys are interleaved (prmt) before they become float16.
//
// The softmax is online in float32 with two maxima: M of s_j for the denominator, and D of (s_j - M) + log2 sv_j for the weights
// 2^((s_j - M) + log2 sv_j - D + 15) of the values, which are rounded to float16: relative to the heaviest term they keep 11 bits down to
// 2^-29, whatever the values' scales, and what is lost below is under 2^-40 of it per key.  (D is relative to M, so that a score of any size
// leaves the scale's logarithm its bits.)  The denominator sums unrounded numbers.
#include "fp8.cuh"
#include "mma_tiles.cuh"

namespace tllm {

constexpr int kA8Warps = 4, kA8Keys = 16;
constexpr int kA8Stages = 4;                     // tiles of a warp's ring: one in use, three on their way (12 KB of them at width 128)
constexpr float kA8Lift = 15.0f;                 // weights are 2^15 at most

template <int HD>
struct A8Tile {
    static constexpr int kPlane = kA8Keys * HD, kBytes = 2 * kPlane + kA8Keys * 8;
    // 16-byte chunk `chunk` of key `row`; both keep the reads of the main loop free of bank conflicts
    static __device__ __forceinline__ int key_at(int row, int chunk) { return HD == 128 ? row * 128 + ((chunk ^ ((row & 1) << 2)) << 4) : row * 64 + (chunk << 4); }
    static __device__ __forceinline__ int value_at(int row, int chunk) {
        const int b = row * HD + (chunk << 4);
        return (b & ~127) + ((((b >> 4) & 7) ^ (row & 6)) << 4);
    }
};

struct A8Cache {
    const uint8_t *k, *v, *scales;
    long long stride;             // bytes from one page to the next
};

// Four bytes of two keys, interleaved: the first two dims' pairs, and the last two's.
__device__ __forceinline__ uint32_t pairs_low(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5140); }
__device__ __forceinline__ uint32_t pairs_high(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7362); }

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ float quad_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// Runs of keys of one head added in order: sums and values of n runs, each with its M, D and l (`me` apart), one dim of its values (`oe`
// apart).  M = max M_s, D = max (D_s + M_s - M); acc = sum o_s 2^(D_s + M_s - M - D), total = sum l_s 2^(M_s - M).  A run without keys has
// M of -infinity and sums of zero; scores that are all NaN leave M so too, and l NaN.
template <int UNROLL>
__device__ __forceinline__ void join_runs(const float* m, int me, const float* o, int oe, int n, float& acc, float& total, float& mm, float& dn) {
    mm = dn = -INFINITY;
    acc = total = 0.0f;
#pragma unroll UNROLL
    for (int s = 0; s < n; ++s) mm = fmaxf(mm, m[s * me]);
#pragma unroll UNROLL
    for (int s = 0; s < n; ++s)
        if (m[s * me] != -INFINITY) dn = fmaxf(dn, m[s * me + 1] + (m[s * me] - mm));
#pragma unroll UNROLL
    for (int s = 0; s < n; ++s) {
        const float ms = m[s * me], l = m[s * me + 2];
        if (ms == -INFINITY) {
            total += l;
        } else {
            total += l * exp2f(ms - mm);
            const float d = m[s * me + 1] + (ms - mm);
            if (d != -INFINITY) acc += o[s * oe] * exp2f(d - dn);
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(kA8Warps * 32, 3)
attention_fp8_decode_kernel(const bf16* q, const A8Cache cache, const int* __restrict__ positions, const int* __restrict__ token_slot,
                            const int* __restrict__ rows, const int* __restrict__ block_table, int max_pages, int page_size, int q_heads,
                            int kv_heads, int window, float scale_log2e, int splits, float* __restrict__ part_o,
                            float* __restrict__ part_m, bf16* __restrict__ out) {
    extern __shared__ __align__(128) unsigned char smem[];
    TLLM_PDL_ENTER();
    using Tile = A8Tile<HD>;
    const int split = blockIdx.x, g = blockIdx.y, ridx = blockIdx.z;
    const int r = rows ? rows[ridx] : ridx;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, gr = lane >> 2;
    const int group = q_heads / kv_heads;
    const int slot = token_slot[r];
    if (slot < 0) {
        if (splits == 1)
            for (int i = threadIdx.x; i < group * HD; i += blockDim.x) out[((size_t)r * q_heads + (size_t)g * group) * HD + i] = __float2bfloat16_rn(0.0f);
        return;
    }
    const int pos = positions[r];
    const int lo = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
    const int base = lo / kA8Keys * kA8Keys;
    const int tiles_all = (pos - base) / kA8Keys + 1;
    int per = (tiles_all + splits - 1) / splits;
    per = (per + kA8Warps - 1) / kA8Warps * kA8Warps;              // whole rounds of the four warps
    const int tile0 = base / kA8Keys + split * per;
    const int tile_end = min(base / kA8Keys + tiles_all, tile0 + per);
    const int* table = block_table + (size_t)slot * max_pages;
    unsigned char* ring = smem + (size_t)warp * kA8Stages * Tile::kBytes;

    auto issue = [&](int tile, int stage) {
        if (tile < tile_end) {
            const int key0 = tile * kA8Keys;
            const int page = table[key0 / page_size];
            const size_t at = (size_t)max(page, 0) * cache.stride, token0 = (size_t)g * page_size + key0 % page_size;
            const uint8_t *kp = cache.k + at + token0 * HD, *vp = cache.v + at + token0 * HD, *sp = cache.scales + at + token0 * 8;
            const uint32_t ks = smem_u32(ring + (size_t)stage * Tile::kBytes), vs = ks + Tile::kPlane, ss = vs + Tile::kPlane;
            const bool whole = page >= 0 && key0 >= lo && key0 + kA8Keys - 1 <= pos;
#pragma unroll
            for (int i = 0; i < Tile::kPlane / 16 / 32; ++i) {
                const int n = lane + 32 * i, row = n / (HD / 16), chunk = n % (HD / 16);
                const bool ok = whole || (page >= 0 && key0 + row >= lo && key0 + row <= pos);
                cp_async_16(ks + Tile::key_at(row, chunk), kp + n * 16, ok);
                cp_async_16(vs + Tile::value_at(row, chunk), vp + n * 16, ok);
            }
            if (lane < 8) cp_async_16(ss + lane * 16, sp + lane * 16, page >= 0);       // two keys' scales: masked below
        }
        cp_async_commit();                                         // one group per call, empty past the end
    };
    int tile = tile0 + warp;
#pragma unroll
    for (int st = 0; st < kA8Stages - 1; ++st) issue(tile + st * kA8Warps, st);

    // queries in float16, each head times a power of two; fragment (h, w) has dims 64 h + 16 c + 4 w .. + 3 of this lane
    uint32_t qa[HD / 16][4];
    float to_score[2];                                             // of heads gr and gr + 8: what turns a product into s
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int head = gr + 8 * half;
        const bf16* qp = q + ((size_t)r * q_heads + (size_t)g * group + min(head, group - 1)) * HD;
        float v[HD / 4];
        float largest = 0.0f;
#pragma unroll
        for (int h = 0; h < HD / 64; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint4 raw = *reinterpret_cast<const uint4*>(qp + 64 * h + 16 * c + 8 * i);
                const uint32_t p[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[16 * h + 8 * i + 2 * j] = low_float(p[j]);
                    v[16 * h + 8 * i + 2 * j + 1] = high_float(p[j]);
                    largest = fmaxf(largest, fmaxf(fabsf(low_float(p[j])), fabsf(high_float(p[j]))));
                }
            }
        largest = quad_max(largest);
        // 2^(14 - exponent): as a product of two factors, each within float32's range for every bfloat16
        const int e = (__float_as_int(largest) >> 23) & 255;       // biased exponent; 0 for zeros and the smallest, 255 for infinities
        const int shift = e == 255 ? 0 : 14 + 127 - max(e, 1);     // -113 .. 140
        const float f0 = __int_as_float((127 + shift / 2) << 23), f1 = __int_as_float((127 + shift - shift / 2) << 23);
        const float b0 = __int_as_float((127 - shift / 2) << 23), b1 = __int_as_float((127 - (shift - shift / 2)) << 23);
        to_score[half] = scale_log2e * b0 * b1;
#pragma unroll
        for (int f = 0; f < HD / 16; ++f) {
            const float* x = v + 4 * f;
            const bool live = head < group;
            qa[f][half] = live ? pack_half(x[0] * f0 * f1, x[1] * f0 * f1) : 0u;
            qa[f][2 + half] = live ? pack_half(x[2] * f0 * f1, x[3] * f0 * f1) : 0u;
        }
    }

    float o[HD / 8][4];                                            // o[i]: dims gr' (HD / 8) + i of columns gr' = 2 c, 2 c + 1
#pragma unroll
    for (int i = 0; i < HD / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, dd[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};   // M, D, sum

    for (int stage = 0; tile < tile_end; tile += kA8Warps, stage = (stage + 1) % kA8Stages) {
        __syncwarp();                                              // the stage refilled below has been read by all lanes
        issue(tile + (kA8Stages - 1) * kA8Warps, (stage + kA8Stages - 1) % kA8Stages);
        cp_async_wait<kA8Stages - 1>();
        __syncwarp();
        const unsigned char *kt = ring + (size_t)stage * Tile::kBytes, *vt = kt + Tile::kPlane;
        const float* st = reinterpret_cast<const float*>(vt + Tile::kPlane);

        float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
                const uint4 raw = *reinterpret_cast<const uint4*>(kt + Tile::key_at(nt * 8 + gr, 4 * h + c));
                const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t b[2] = {e4m3x2_to_half2(w[i]), e4m3x2_to_half2(w[i] >> 16)};
                    mma_f16_16816(s[nt], qa[4 * h + i], b);
                }
            }
        // s[nt][e], s[nt][2 + e]: heads gr and gr + 8, key nt * 8 + 2 c + e
        float lv[2][2], tm[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            const float4 sc = *reinterpret_cast<const float4*>(st + (nt * 8 + 2 * c) * 2);
            const int j = tile * kA8Keys + nt * 8 + 2 * c;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const bool ok = j + e >= lo && j + e <= pos;
                const float sk = e ? sc.z : sc.x;
                lv[nt][e] = ok ? __log2f(e ? sc.w : sc.y) : -INFINITY;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    float& x = s[nt][2 * half + e];
                    x = ok ? x * (sk * to_score[half]) : -INFINITY;
                    tm[half] = fmaxf(tm[half], x);
                }
            }
        }
        float w[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const float mn = fmaxf(m[half], quad_max(tm[half]));
            const float ms = mn == -INFINITY ? 0.0f : mn, back = m[half] - ms;      // -infinity before the first key
            float sum = 0.0f, td = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float t = s[nt][2 * half + e] - ms;
                    sum += exp2f(t);
                    w[nt][2 * half + e] = t + lv[nt][e];
                    td = fmaxf(td, w[nt][2 * half + e]);
                }
            const float dn = fmaxf(dd[half] + back, quad_max(td)), ds = dn == -INFINITY ? 0.0f : dn;
            const float cu = exp2f(dd[half] + back - ds);
            l[half] = l[half] * exp2f(back) + sum;
            m[half] = mn;
            dd[half] = dn;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) w[nt][2 * half + e] = exp2f(w[nt][2 * half + e] - ds + kA8Lift);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                o[i][2 * half] *= cu;
                o[i][2 * half + 1] *= cu;
            }
        }
        const uint32_t pa[4] = {pack_half(w[0][0], w[0][1]), pack_half(w[0][2], w[0][3]), pack_half(w[1][0], w[1][1]), pack_half(w[1][2], w[1][3])};
        // values of keys 2 c, 2 c + 1 and eight further, dims gr (HD / 8) .. + HD / 8 - 1
        constexpr int kWords = HD / 32;
        uint32_t vw[4][kWords];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 2 * c + (i & 1) + (i >> 1) * 8;
            if constexpr (HD == 128) {
                const uint4 raw = *reinterpret_cast<const uint4*>(vt + Tile::value_at(row, gr));
                vw[i][0] = raw.x; vw[i][1] = raw.y; vw[i][2] = raw.z; vw[i][3] = raw.w;
            } else {
                const uint2 raw = *reinterpret_cast<const uint2*>(vt + Tile::value_at(row, gr >> 1) + (gr & 1) * 8);
                vw[i][0] = raw.x; vw[i][1] = raw.y;
            }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint32_t a0 = pairs_low(vw[0][i], vw[1][i]), a1 = pairs_high(vw[0][i], vw[1][i]);
            const uint32_t b0 = pairs_low(vw[2][i], vw[3][i]), b1 = pairs_high(vw[2][i], vw[3][i]);
            const uint32_t d[4][2] = {{e4m3x2_to_half2(a0), e4m3x2_to_half2(b0)}, {e4m3x2_to_half2(a0 >> 16), e4m3x2_to_half2(b0 >> 16)},
                                      {e4m3x2_to_half2(a1), e4m3x2_to_half2(b1)}, {e4m3x2_to_half2(a1 >> 16), e4m3x2_to_half2(b1 >> 16)}};
#pragma unroll
            for (int e = 0; e < 4; ++e) mma_f16_16816(o[4 * i + e], pa, d[e]);
        }
    }
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
        l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    }
    // ---- the four warps' results are added in shared memory, which the ring no longer needs
    cp_async_wait<0>();
    __syncthreads();
    float* os = reinterpret_cast<float*>(smem);                    // [warps][16][HD]
    float* ms = os + kA8Warps * 16 * HD;                           // [warps][16][3]: M, D, L
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int row = gr + 8 * half;
        if (row < group) {
            float* dst = os + ((size_t)warp * 16 + row) * HD;
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < HD / 8; i += 4)
                    *reinterpret_cast<float4*>(dst + (2 * c + e) * (HD / 8) + i) =
                        make_float4(o[i][2 * half + e], o[i + 1][2 * half + e], o[i + 2][2 * half + e], o[i + 3][2 * half + e]);
            if (c == 0) {
                ms[(warp * 16 + row) * 3] = m[half];
                ms[(warp * 16 + row) * 3 + 1] = dd[half];
                ms[(warp * 16 + row) * 3 + 2] = l[half];
            }
        }
    }
    __syncthreads();
    for (int idx = threadIdx.x; idx < group * HD; idx += blockDim.x) {
        const int row = idx / HD, d = idx - row * HD;
        float acc, total, mm, dn;
        join_runs<kA8Warps>(ms + row * 3, 16 * 3, os + (size_t)row * HD + d, 16 * HD, kA8Warps, acc, total, mm, dn);
        const int head = g * group + row;
        if (splits == 1) {
            const float up = dn == -INFINITY ? 0.0f : exp2f(dn - kA8Lift);
            out[((size_t)r * q_heads + head) * HD + d] = __float2bfloat16_rn(acc * up / total);
        } else {
            const size_t at = ((size_t)ridx * q_heads + head) * splits + split;
            part_o[at * HD + d] = acc;
            if (d == 0) { part_m[at * 3] = mm; part_m[at * 3 + 1] = dn; part_m[at * 3 + 2] = total; }
        }
    }
}

template <int HD>
__global__ void attention_fp8_join_kernel(const float* part_o, const float* part_m, const int* __restrict__ token_slot,
                                          const int* __restrict__ rows, int q_heads, int splits, bf16* __restrict__ out) {
    TLLM_PDL_ENTER();
    const int ridx = blockIdx.x, head = blockIdx.y, d = threadIdx.x;
    const int r = rows ? rows[ridx] : ridx;
    bf16* dst = out + ((size_t)r * q_heads + head) * HD;
    if (token_slot[r] < 0) { dst[d] = __float2bfloat16_rn(0.0f); return; }
    const size_t base = ((size_t)ridx * q_heads + head) * splits;
    float acc, total, mm, dn;
    join_runs<1>(part_m + base * 3, 3, part_o + base * HD + d, HD, splits, acc, total, mm, dn);
    const float up = dn == -INFINITY ? 0.0f : exp2f(dn - kA8Lift);
    dst[d] = __float2bfloat16_rn(acc * up / total);
}

template <int HD>
static int launch_attention_fp8(const void* q, const A8Cache& cache, const int* positions, const int* token_slot, const int* rows, int n_rows,
                                const int* block_table, int max_pages, int page_size, int q_heads, int kv_heads, int window, float scale,
                                int splits, float* part_o, float* part_m, void* out, cudaStream_t stream) {
    constexpr size_t ring = (size_t)kA8Warps * kA8Stages * A8Tile<HD>::kBytes, joined = (size_t)kA8Warps * 16 * (HD + 3) * sizeof(float);
    constexpr size_t smem = ring > joined ? ring : joined;
    static OncePerDevice configured;
    if (configured.first()) {
        cudaError_t e = cudaFuncSetAttribute(attention_fp8_decode_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) { set_error("attention_fp8_decode: %s", cudaGetErrorString(e)); return (int)e; }
        configured.done();
    }
    launch_pdl(kPdlAttention, attention_fp8_decode_kernel<HD>, dim3(splits, kv_heads, n_rows), dim3(kA8Warps * 32), smem, stream,
               (const bf16*)q, cache, positions, token_slot, rows, block_table, max_pages, page_size, q_heads, kv_heads, window,
               scale * 1.4426950408889634f, splits, part_o, part_m, (bf16*)out);
    const int rc = finish_launch("attention_fp8_decode");
    if (rc != 0 || splits == 1) return rc;
    launch_pdl(kPdlCombine, attention_fp8_join_kernel<HD>, dim3(n_rows, q_heads), dim3(HD), 0, stream, (const float*)part_o, (const float*)part_m,
               token_slot, rows, q_heads, splits, (bf16*)out);
    return finish_launch("attention_fp8_join");
}

// ---------------------------------------------------------------- pages back in bfloat16
// For the portions (segments of more than one token) of a step: the pages that a portion's tokens may read, from the one that holds the
// first key of its first token's window to the last token's, become pages of `pages` ([pages][keys, values][kv head][token][HD] bfloat16),
// one portion after the other, and table[slot] lists them (-1 elsewhere).  The prompt kernels then read those.  One block of threads per
// page; bound by HBM.
template <int HD>
__global__ void __launch_bounds__(256) attention_fp8_unpack_kernel(const A8Cache cache, const int* __restrict__ seg_info,
                                                                   const int* __restrict__ block_table, int max_pages, int page_size,
                                                                   int kv_heads, int window, int capacity, bf16* __restrict__ pages,
                                                                   int* __restrict__ table) {
    TLLM_PDL_ENTER();
    const int seg = blockIdx.y;
    const int slot = seg_info[4 * seg], length = seg_info[4 * seg + 2], pos0 = seg_info[4 * seg + 3], last = pos0 + length - 1;
    if (slot < 0 || length <= 1) return;
    auto first_page = [&](int p) { return window > 0 && p - window + 1 > 0 ? (p - window + 1) / page_size : 0; };
    const int first = first_page(pos0), i = first + blockIdx.x;
    if (blockIdx.x == 0)                                           // pages outside: none
        for (int n = threadIdx.x; n < max_pages; n += blockDim.x)
            if (n < first || n > last / page_size) table[(size_t)slot * max_pages + n] = -1;
    if (i > last / page_size || i >= max_pages) return;
    int to = blockIdx.x;
    for (int s = 0; s < seg; ++s)
        if (seg_info[4 * s + 2] > 1 && seg_info[4 * s] >= 0)
            to += (seg_info[4 * s + 3] + seg_info[4 * s + 2] - 1) / page_size - first_page(seg_info[4 * s + 3]) + 1;
    const int page = to < capacity ? block_table[(size_t)slot * max_pages + i] : -1;
    if (threadIdx.x == 0) table[(size_t)slot * max_pages + i] = page < 0 ? -1 : to;
    if (page < 0) return;
    const size_t at = (size_t)page * cache.stride, plane = (size_t)kv_heads * page_size;
    const float* scales = reinterpret_cast<const float*>(cache.scales + at);
    bf16* dst = pages + (size_t)to * 2 * plane * HD;
    constexpr int kPer = HD / 16;                                  // 16-byte pieces of a head
    for (int n = threadIdx.x; n < 2 * (int)plane * kPer; n += blockDim.x) {
        const int token = n / kPer, which = token >= (int)plane, t = token - which * (int)plane;
        // tokens behind the last one hold what an earlier request left, or nothing: zeros instead
        const bool ok = i * page_size + t % page_size <= last;
        const uint4 raw = ok ? *reinterpret_cast<const uint4*>((which ? cache.v : cache.k) + at + (size_t)t * HD + n % kPer * 16) : make_uint4(0, 0, 0, 0);
        const float s = ok ? scales[2 * t + which] : 0.0f;
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t h = e4m3x2_to_half2(e & 1 ? w[e >> 1] >> 16 : w[e >> 1]);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
            o[e] = pack_bf16(f.x * s, f.y * s);
        }
        uint4* d = reinterpret_cast<uint4*>(dst + (size_t)token * HD + n % kPer * 16);
        d[0] = make_uint4(o[0], o[1], o[2], o[3]);
        d[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
}

}  // namespace tllm

using namespace tllm;

static int check_a8(const char* what, const void* k, const void* v, const void* scales, long long page_bytes, int page_size, int kv_heads, int head_dim) {
    TLLM_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %d is not 64 or 128", what, head_dim);
    TLLM_REQUIRE(kv_heads > 0 && kv_heads <= 65535, "%s: %d key/value heads", what, kv_heads);
    TLLM_REQUIRE(page_size > 0 && page_size % 16 == 0, "%s: page size %d is no multiple of 16", what, page_size);
    TLLM_REQUIRE(k && v && scales && page_bytes > 0 && page_bytes % 16 == 0 &&
                     ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(scales)) & 15u) == 0,
                 "%s: planes must be 16-byte aligned", what);
    return 0;
}

// q, out [rows, q_heads * head_dim] bfloat16; planes of pages `page_bytes` apart: k, v [kv_heads][page_size][head_dim] e4m3, scales
// [kv_heads][page_size][2] float32.  rows: indices of the one-token rows, null for 0 .. n_rows - 1.  Scratch for splits > 1: part_o
// float[n_rows * q_heads * splits * head_dim], part_m float[n_rows * q_heads * splits * 3].
extern "C" int tllm_attention_fp8_decode(const void* q, const void* k, const void* v, const void* scales, long long page_bytes,
                                         const int* positions, const int* token_slot, const int* rows, int n_rows, const int* block_table,
                                         int max_pages, int page_size, int q_heads, int kv_heads, int head_dim, int window, float scale,
                                         int splits, float* part_o, float* part_m, void* out, cudaStream_t stream) {
    if (check_a8("attention_fp8_decode", k, v, scales, page_bytes, page_size, kv_heads, head_dim) != 0) return -1;
    TLLM_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16,
                 "attention_fp8_decode: %d query heads over %d key/value heads (at most 16 per group)", q_heads, kv_heads);
    TLLM_REQUIRE(splits >= 1 && splits <= 65535 && n_rows >= 0 && n_rows <= 65535 && q_heads <= 65535 && max_pages > 0, "attention_fp8_decode: bad grid");
    TLLM_REQUIRE(splits == 1 || (part_o && part_m), "attention_fp8_decode: %d runs of keys need scratch", splits);
    TLLM_REQUIRE(q && out && positions && token_slot && block_table && (reinterpret_cast<uintptr_t>(q) & 15u) == 0,
                 "attention_fp8_decode: missing or unaligned operands");
    if (n_rows == 0) return 0;
    const A8Cache cache{(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)scales, page_bytes};
    return head_dim == 64 ? launch_attention_fp8<64>(q, cache, positions, token_slot, rows, n_rows, block_table, max_pages, page_size, q_heads, kv_heads,
                                                     window, scale, splits, part_o, part_m, out, stream)
                          : launch_attention_fp8<128>(q, cache, positions, token_slot, rows, n_rows, block_table, max_pages, page_size, q_heads, kv_heads,
                                                      window, scale, splits, part_o, part_m, out, stream);
}

// seg_info [segments][4] = slot, first row, tokens, position of the first.  `per`: pages of the portion that has most; pages bfloat16
// [capacity][2][kv_heads][page_size][head_dim], room for all portions' pages; table int32 like block_table.
extern "C" int tllm_attention_fp8_unpack(const void* k, const void* v, const void* scales, long long page_bytes, const int* seg_info, int segments,
                                         const int* block_table, int max_pages, int page_size, int kv_heads, int head_dim, int window, int per,
                                         int capacity, void* pages, int* table, cudaStream_t stream) {
    if (check_a8("attention_fp8_unpack", k, v, scales, page_bytes, page_size, kv_heads, head_dim) != 0) return -1;
    TLLM_REQUIRE(segments > 0 && segments <= 65535 && per > 0 && per <= max_pages && capacity > 0, "attention_fp8_unpack: bad sizes");
    TLLM_REQUIRE(seg_info && block_table && pages && table && (reinterpret_cast<uintptr_t>(pages) & 15u) == 0, "attention_fp8_unpack: missing operands");
    TLLM_REQUIRE((long long)2 * kv_heads * page_size * (head_dim / 16) <= 0x7fffffff, "attention_fp8_unpack: too large");
    const A8Cache cache{(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)scales, page_bytes};
    if (head_dim == 64)
        launch_pdl(kPdlOther, attention_fp8_unpack_kernel<64>, dim3(per, segments), dim3(256), 0, stream, cache, seg_info, block_table, max_pages,
                   page_size, kv_heads, window, capacity, (bf16*)pages, table);
    else
        launch_pdl(kPdlOther, attention_fp8_unpack_kernel<128>, dim3(per, segments), dim3(256), 0, stream, cache, seg_info, block_table, max_pages,
                   page_size, kv_heads, window, capacity, (bf16*)pages, table);
    return finish_launch("attention_fp8_unpack");
}
