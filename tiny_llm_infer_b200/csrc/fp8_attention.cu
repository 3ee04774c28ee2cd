// Attention of single tokens over a paged cache of 8-bit keys and values, split over the keys and joined; and the pages of prompt
// portions back in bfloat16 for the prompt kernels.
//
// A key is kept as e4m3 values k8 and a float32 scale sk, a value as v8 and sv (fp8.cuh; one scale per token and head).  With base-2
// scores s_j = (q . k8_j) sk_j scale log2(e),
//
//   out = sum_j 2^(s_j) sv_j v8_j / sum_j 2^(s_j).
//
// One block of threads owns (row, key/value head, run of keys): the query heads of the group share what is read, so a key and its value
// come from HBM once per group: 2 hd + 8 bytes, half of the bfloat16 cache's.  What bounds it is their way from HBM.  The four warps take
// units of 32 keys in turn: cp.async brings a unit's keys, values and scales into the warp's own ring of two while the unit before is
// worked on; keys that do not count (behind the row's position, before its window, without a page) arrive as zeros, so that what a page
// held before meets no sum; a row left without keys becomes zeros.
//
// Products run on mma.sync m16n8k16 with float16 operands, which hold every e4m3 value exactly; keys and values are the left operands
// (16 keys, or 16 dims, by 16) and eight query heads the right one, so a group of up to eight heads wastes nothing.  Queries are brought to
// float16 by a power of two per head that puts the largest at 2^14 to 2^15, exact down to 2^-28 of the largest.  A lane's sixteen
// neighbouring bytes of a key stand for the columns that four fragments assign to it, on the query's side alike, so keys need no
// rearrangement.  For V^T P the fragments want two keys side by side: bytes of two keys are interleaved (prmt) before they become float16,
// and the weights are turned by movmatrix.
//
// The softmax is online in float32 with two maxima: M of s_j for the denominator, and D of (s_j - M) + log2 sv_j for the weights
// 2^((s_j - M) + log2 sv_j - D + 15) of the values, which are rounded to float16: relative to the heaviest term they keep 11 bits down to
// 2^-29, whatever the values' scales, and what is lost below is under 2^-40 of it per key.  (D is relative to M, so that a score of any size
// leaves the scale's logarithm its bits.)  The denominator sums unrounded numbers.  A value whose scale is zero, or below float32's normal
// numbers, adds nothing, and its key counts in the denominator; scales are not negative.
//
// With the heads as rows of a 16-row tile and 16 keys at a time a warp took 1.0 us a tile alone and 1.8 us beside eleven others (2.9 to
// 3.9 TB/s): half of every product was wasted on missing rows, and the chain of scores, maxima and weights was walked twice as often.
#include "fp8.cuh"
#include "mma_tiles.cuh"

namespace tllm {

constexpr int kA8Warps = 4, kA8Unit = 32;        // keys a warp takes at a time
constexpr int kA8Stages = 2;                     // units of a warp's ring: one in use, one on its way (8.4 KB at width 128); more of them gained nothing
constexpr float kA8Lift = 15.0f;                 // weights are 2^15 at most

// A unit in shared memory: keys, values, pairs of scales.
template <int HD>
struct A8Unit {
    static constexpr int kPlane = kA8Unit * HD, kBytes = 2 * kPlane + kA8Unit * 8;
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
    int pages;
    // a page of the table, or -1 where it names none: no other memory is read for it
    __device__ __forceinline__ int held(int page) const { return (unsigned)page < (unsigned)pages ? page : -1; }
};

// Four bytes of two keys, interleaved: the first two dims' pairs, and the last two's.
__device__ __forceinline__ uint32_t pairs_low(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5140); }
__device__ __forceinline__ uint32_t pairs_high(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7362); }

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// 2^x and log2 x by the special function unit (2 units in the last place; results below 2^-126 are zero).
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float fast_log2(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async_all(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src));
}
// The largest (the sum) over the eight lanes that hold the same heads and other keys.
__device__ __forceinline__ float keys_max(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float keys_sum(float v) {
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// An 8 x 8 matrix of 16-bit numbers, a row in four lanes, turned.
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(v));
    return d;
}

// The warps' runs of keys of one head added in order: sums and values of n runs, each with its M, D and l (`me` apart), one dim of its
// values (`oe` apart).  M = max M_s, D = max (D_s + M_s - M); acc = sum o_s 2^(D_s + M_s - M - D), total = sum l_s 2^(M_s - M).  A run without keys has
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

// One run: units [unit0, unit_end) of the keys of one (row, key/value head), by the four warps of a block in turn.  Leaves the warps' results
// in shared memory (os, ms; every thread may read them): run_sums adds them.  NT: eights of query heads per key/value head.
// lo, base: the first key that counts, and the same rounded down to 16 (16 keys never straddle a page), where unit 0 begins.
struct A8Row {
    const bf16* q;                // of the group's first head
    const int* table;
    int g, group, page_size, kv_heads, pos, lo, base;
    float scale_log2e;
};
template <int HD, int NT>
__device__ __forceinline__ void attend_run(unsigned char* smem, const A8Row& row_of, const A8Cache& cache, int unit0, int unit_end) {
    using Unit = A8Unit<HD>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = lane & 3, gr = lane >> 2;
    const int g = row_of.g, group = row_of.group, page_size = row_of.page_size, pos = row_of.pos, lo = row_of.lo, base = row_of.base;
    const int* table = row_of.table;
    int unit = unit0 + warp;
    unsigned char* ring = smem + (size_t)warp * kA8Stages * Unit::kBytes;

    // ---- the next unit to fetch: its first key and that key's place in its page
    int f_unit = unit, f_stage = 0, key0 = base + unit * kA8Unit;
    int in_page = key0 % page_size;
    constexpr int kStep = kA8Warps * kA8Unit;
    const int step_rest = kStep % page_size;
    const uint8_t* const k0 = cache.k + lane * 16;
    const uint8_t* const v0 = cache.v + lane * 16;
    const int key_dst = Unit::key_at(lane / (HD / 16), lane % (HD / 16));
    uint32_t gaps = 0;                                             // bit 2 s + h: keys 16 h .. 16 h + 15 of the unit in stage s are in no page
    // The pages of sixteen units at once, a lane each for a sixteen of keys, and of the sixteen units after them: no copy waits for the table.
    // (Looked up unit by unit, a unit ahead, a unit took a warp 1.2 us where it takes 0.9.)
    auto look_up = [&](int first) {
        const int mine = first + (lane >> 1) * kA8Warps;
        if (first >= unit_end || mine >= unit_end) return -1;
        const int key = base + mine * kA8Unit + (lane & 1) * 16;
        return key <= pos ? table[key / page_size] : -1;
    };
    constexpr int kBatch = 16 * kA8Warps;
    int listed = look_up(unit), listed_next = look_up(unit + kBatch), f_at = 0;
    auto fetch = [&]() {
        if (f_unit < unit_end) {
            const bool wraps = in_page + 16 >= page_size;
            const int page[2] = {cache.held(__shfl_sync(0xffffffffu, listed, f_at)), cache.held(__shfl_sync(0xffffffffu, listed, f_at + 1))};
            const uint32_t dst = smem_u32(ring + (size_t)f_stage * Unit::kBytes);
            gaps = (gaps & ~(3u << 2 * f_stage)) | ((uint32_t)page[0] >> 31 | (uint32_t)page[1] >> 31 << 1) << 2 * f_stage;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int first = key0 + 16 * h;
                const size_t at = (size_t)max(page[h], 0) * cache.stride, token = (size_t)g * page_size + (h == 0 ? in_page : wraps ? in_page + 16 - page_size : in_page + 16);
                const uint8_t *kp = k0 + at + token * HD, *vp = v0 + at + token * HD;
                constexpr int kPieces = 16 * HD / 16 / 32;         // per lane: 4 or 2
                if (page[h] >= 0 && first >= lo && first + 15 <= pos) {
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        const int n = lane + 32 * i;
                        cp_async_all(dst + key_dst + h * 16 * HD + i * 512, kp + i * 512);
                        cp_async_all(dst + Unit::kPlane + Unit::value_at(n / (HD / 16), n % (HD / 16)) + h * 16 * HD, vp + i * 512);
                    }
                } else {                                           // some of them do not count
#pragma unroll
                    for (int i = 0; i < kPieces; ++i) {
                        const int n = lane + 32 * i, row = n / (HD / 16);
                        const bool ok = page[h] >= 0 && first + row >= lo && first + row <= pos;
                        cp_async_16(dst + key_dst + h * 16 * HD + i * 512, kp + i * 512, ok);
                        cp_async_16(dst + Unit::kPlane + Unit::value_at(row, n % (HD / 16)) + h * 16 * HD, vp + i * 512, ok);
                    }
                }
                if (lane < 8) cp_async_16(dst + 2 * Unit::kPlane + h * 128 + lane * 16, cache.scales + at + token * 8 + lane * 16, page[h] >= 0);   // masked below
            }
            f_unit += kA8Warps;
            key0 += kStep;
            in_page += step_rest;
            if (in_page >= page_size) in_page -= page_size;
            f_stage = f_stage + 1 == kA8Stages ? 0 : f_stage + 1;
            f_at += 2;
            if (f_at == 32) f_at = 0, listed = listed_next, listed_next = look_up(f_unit + kBatch);
        }
        cp_async_commit();                                         // one group per call, empty past the end
    };
#pragma unroll
    for (int st = 0; st < kA8Stages - 1; ++st) fetch();

    // ---- queries in float16, each head times a power of two; fragment (h, i) has dims 64 h + 16 c + 4 i .. + 3 of head nt * 8 + gr
    uint32_t qb[NT][HD / 16][2];
    float to_score[NT][2];                                         // of heads nt * 8 + 2 c, + 1: what turns a product into s
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int head = nt * 8 + gr;
        const bf16* qp = row_of.q + (size_t)min(head, group - 1) * HD;
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
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // 2^(14 - exponent): as a product of two factors, each within float32's range for every bfloat16
        const int e = (__float_as_int(largest) >> 23) & 255;       // biased exponent; 0 for zeros and the smallest, 255 for infinities
        const int shift = e == 255 ? 0 : 14 + 127 - max(e, 1);     // -113 .. 140
        const float f0 = __int_as_float((127 + shift / 2) << 23), f1 = __int_as_float((127 + shift - shift / 2) << 23);
        const float b0 = __int_as_float((127 - shift / 2) << 23), b1 = __int_as_float((127 - (shift - shift / 2)) << 23);
        const float back = row_of.scale_log2e * b0 * b1;
        const bool live = head < group;
#pragma unroll
        for (int f = 0; f < HD / 16; ++f) {
            const float* x = v + 4 * f;
            qb[nt][f][0] = live ? pack_half(x[0] * f0 * f1, x[1] * f0 * f1) : 0u;
            qb[nt][f][1] = live ? pack_half(x[2] * f0 * f1, x[3] * f0 * f1) : 0u;
        }
#pragma unroll
        for (int e2 = 0; e2 < 2; ++e2) to_score[nt][e2] = __shfl_sync(0xffffffffu, back, (2 * c + e2) * 4);
    }

    constexpr int kMT = HD / 16;                                   // tiles of 16 dims; of a lane the dims gr (HD / 8) + 2 t, + 1 are rows gr, gr + 8 of tile t
    float o[NT][kMT][4];
    float m[NT][2], dd[NT][2], l[NT][2];                           // of heads nt * 8 + 2 c, + 1: M, D, sum over this lane's keys
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int t = 0; t < kMT; ++t) o[nt][t][0] = o[nt][t][1] = o[nt][t][2] = o[nt][t][3] = 0.0f;
#pragma unroll
        for (int e = 0; e < 2; ++e) m[nt][e] = dd[nt][e] = -INFINITY, l[nt][e] = 0.0f;
    }

    for (int stage = 0; unit < unit_end; unit += kA8Warps, stage = stage + 1 == kA8Stages ? 0 : stage + 1) {
        __syncwarp();                                              // the stage refilled below has been read by all lanes
        fetch();
        cp_async_wait<kA8Stages - 1>();
        __syncwarp();
        const unsigned char *kt = ring + (size_t)stage * Unit::kBytes, *vt = kt + Unit::kPlane;
        const float2* st = reinterpret_cast<const float2*>(vt + Unit::kPlane);

        // ---- scores: s[nt][h][e], s[nt][h][2 + e]: keys 16 h + gr and 16 h + gr + 8, head nt * 8 + 2 c + e
        float s[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[nt][h][0] = s[nt][h][1] = s[nt][h][2] = s[nt][h][3] = 0.0f;
#pragma unroll
        for (int f = 0; f < HD / 64; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 ra = *reinterpret_cast<const uint4*>(kt + Unit::key_at(16 * h + gr, 4 * f + c));
                const uint4 rb = *reinterpret_cast<const uint4*>(kt + Unit::key_at(16 * h + gr + 8, 4 * f + c));
                const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t a[4];
                    e4m3x4_to_half2(wa[i], a[0], a[2]);
                    e4m3x4_to_half2(wb[i], a[1], a[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_f16_16816(s[nt][h], a, qb[nt][4 * f + i]);
                }
            }
        const int first = base + unit * kA8Unit + gr;
        const uint32_t missing = gaps >> 2 * stage & 3u;
        const bool whole = base + unit * kA8Unit >= lo && base + unit * kA8Unit + kA8Unit - 1 <= pos && missing == 0;
        float lv[2][2];                                            // log2 of the values' scales, keys 16 h + gr + 8 e
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 sc = st[16 * h + 8 * e + gr];
                lv[h][e] = fast_log2(sc.y);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int n = 0; n < 2; ++n) s[nt][h][2 * e + n] *= sc.x * to_score[nt][n];
            }
        if (!whole)                                                // keys that do not count
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int j = first + 16 * h + 8 * e;
                    if (j >= lo && j <= pos && !(missing >> h & 1)) continue;
                    lv[h][e] = -INFINITY;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int n = 0; n < 2; ++n) s[nt][h][2 * e + n] = -INFINITY;
                }
        // ---- maxima, sums and weights, head by head
        uint32_t pb[NT][2][2];                                     // weights as the right operand: keys 2 c, + 1 (and 8 further) of sixteen h, head gr
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float w[2][4], cu[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float mn = fmaxf(m[nt][n], keys_max(fmaxf(fmaxf(s[nt][0][n], s[nt][0][2 + n]), fmaxf(s[nt][1][n], s[nt][1][2 + n]))));
                const float ms = mn == -INFINITY ? 0.0f : mn, back = m[nt][n] - ms;        // -infinity before the first key
                float sum = 0.0f, td = -INFINITY;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float t = s[nt][h][2 * e + n] - ms;
                        sum += fast_exp2(t);
                        w[h][2 * e + n] = t + lv[h][e];
                        td = fmaxf(td, w[h][2 * e + n]);
                    }
                const float dn = fmaxf(dd[nt][n] + back, keys_max(td)), ds = dn == -INFINITY ? 0.0f : dn;
                cu[n] = fast_exp2(dd[nt][n] + back - ds);
                l[nt][n] = l[nt][n] * fast_exp2(back) + sum;
                m[nt][n] = mn;
                dd[nt][n] = dn;
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) w[h][2 * e + n] = fast_exp2(w[h][2 * e + n] - ds + kA8Lift);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 2; ++e) pb[nt][h][e] = turned(pack_half(w[h][2 * e], w[h][2 * e + 1]));
            if (__any_sync(0xffffffffu, cu[0] != 1.0f || cu[1] != 1.0f)) {                 // seldom after the first units
#pragma unroll
                for (int t = 0; t < kMT; ++t) {
                    o[nt][t][0] *= cu[0];
                    o[nt][t][1] *= cu[1];
                    o[nt][t][2] *= cu[0];
                    o[nt][t][3] *= cu[1];
                }
            }
        }
        // ---- values of keys 2 c, 2 c + 1 and eight further of each sixteen, dims gr (HD / 8) .. + HD / 8 - 1
        constexpr int kWords = HD / 32;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t vw[4][kWords];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = 16 * h + 2 * c + (i & 1) + (i >> 1) * 8;
                if constexpr (HD == 128) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(vt + Unit::value_at(row, gr));
                    vw[i][0] = raw.x; vw[i][1] = raw.y; vw[i][2] = raw.z; vw[i][3] = raw.w;
                } else {
                    const uint2 raw = *reinterpret_cast<const uint2*>(vt + Unit::value_at(row, gr >> 1) + (gr & 1) * 8);
                    vw[i][0] = raw.x; vw[i][1] = raw.y;
                }
            }
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const uint32_t x0 = pairs_low(vw[0][i], vw[1][i]), x1 = pairs_high(vw[0][i], vw[1][i]);
                const uint32_t y0 = pairs_low(vw[2][i], vw[3][i]), y1 = pairs_high(vw[2][i], vw[3][i]);
                uint32_t a0[4], a1[4];
                e4m3x4_to_half2(x0, a0[0], a0[1]);
                e4m3x4_to_half2(y0, a0[2], a0[3]);
                e4m3x4_to_half2(x1, a1[0], a1[1]);
                e4m3x4_to_half2(y1, a1[2], a1[3]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    mma_f16_16816(o[nt][2 * i], a0, pb[nt][h]);
                    mma_f16_16816(o[nt][2 * i + 1], a1, pb[nt][h]);
                }
            }
        }
    }
    // ---- the four warps' results are added in shared memory, which the ring no longer needs
    cp_async_wait<0>();
    __syncthreads();
    float* os = reinterpret_cast<float*>(smem);                    // [warps][8 NT][HD]
    float* ms = os + kA8Warps * 8 * NT * HD;                       // [warps][8 NT][3]: M, D, sum
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int row = nt * 8 + 2 * c + n;
            const float sum = keys_sum(l[nt][n]);
            if (row < group) {
                float* dst = os + ((size_t)warp * 8 * NT + row) * HD + gr * (HD / 8);
#pragma unroll
                for (int t = 0; t < kMT; t += 2)
                    *reinterpret_cast<float4*>(dst + 2 * t) = make_float4(o[nt][t][n], o[nt][t][2 + n], o[nt][t + 1][n], o[nt][t + 1][2 + n]);
                if (gr == 0) {
                    ms[(warp * 8 * NT + row) * 3] = m[nt][n];
                    ms[(warp * 8 * NT + row) * 3 + 1] = dd[nt][n];
                    ms[(warp * 8 * NT + row) * 3 + 2] = sum;
                }
            }
        }
    __syncthreads();
}

// Head `row` of the group and dim d of a run: the warps' results added (join_runs).
template <int HD, int NT>
__device__ __forceinline__ void run_sums(const unsigned char* smem, int row, int d, float& acc, float& total, float& mm, float& dn) {
    const float* os = reinterpret_cast<const float*>(smem);
    const float* ms = os + kA8Warps * 8 * NT * HD;
    join_runs<kA8Warps>(ms + row * 3, 8 * NT * 3, os + (size_t)row * HD + d, 8 * NT * HD, kA8Warps, acc, total, mm, dn);
}

// Units of 32 keys that a row's position and window give it.
__device__ __forceinline__ int first_key(int pos, int window) { return window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0; }
__device__ __forceinline__ int units_of(int pos, int window) { return (pos - first_key(pos, window) / 16 * 16) / kA8Unit + 1; }

struct A8Step {
    const bf16* q;
    A8Cache cache;
    const int *positions, *token_slot, *rows, *block_table;
    int n_rows, slots, max_pages, page_size, q_heads, kv_heads, window, room;       // room: max_pages * page_size
    float scale_log2e;
};
// A caller's mistake reads no other memory: a row's position is held within what its row of the block table has room for, and a slot without
// a row of the table, or a position before the first key, is no request.
__device__ __forceinline__ int position_of(const A8Step& st, int r) { return min(st.positions[r], st.room - 1); }
__device__ __forceinline__ int slot_of(const A8Step& st, int r) {
    const int slot = st.token_slot[r];
    return slot < st.slots && st.positions[r] >= 0 ? slot : -1;
}
// Sums in float32 brought to an output; nothing where no key counted.
__device__ __forceinline__ bf16 weighed(float acc, float dn, float total) {
    return __float2bfloat16_rn(total == 0.0f ? 0.0f : acc * (dn == -INFINITY ? 0.0f : exp2f(dn - kA8Lift)) / total);
}
template <int HD>
__device__ __forceinline__ A8Row row_at(const A8Step& st, int r, int slot, int g) {
    A8Row x;
    x.group = st.q_heads / st.kv_heads;
    x.g = g;
    x.q = st.q + ((size_t)r * st.q_heads + (size_t)g * x.group) * HD;
    x.table = st.block_table + (size_t)slot * st.max_pages;
    x.page_size = st.page_size;
    x.kv_heads = st.kv_heads;
    x.pos = position_of(st, r);
    x.lo = first_key(x.pos, st.window);
    x.base = x.lo / 16 * 16;
    x.scale_log2e = st.scale_log2e;
    return x;
}

// A block of threads per (row, key/value head), the whole of it one run.  No kernel that follows may start before this one ends (and the same for clusters
// below): bfloat16 products that start early hold their places and fetch beside it (eight layers of Qwen3-8B widths, 8 rows of 4096 keys: 1.39 ms
// a step where it takes 0.89; one row 1.00 and 0.73).  ORDERED, for more blocks than are resident at once: the rows with most
// keys first, so that what starts late is short (64 rows of 1024 to 4096 keys, 8 heads of
// 128: 62 us where equal shares take 72; 64 rows all of 4096, which shares do better, 119 and 99).
constexpr int kA8MaxOrdered = 256;
template <int HD, int NT, bool ORDERED>
__global__ void __launch_bounds__(kA8Warps * 32, NT == 1 ? 3 : 2) attention_fp8_whole_kernel(const A8Step st, bf16* __restrict__ out) {
    extern __shared__ __align__(128) unsigned char smem[];
    TLLM_PDL_WAIT();
    const int g = blockIdx.x;
    int ridx = blockIdx.y;
    if constexpr (ORDERED) {
        __shared__ int units[kA8MaxOrdered], mine;
        for (int i = threadIdx.x; i < st.n_rows; i += kA8Warps * 32) {
            const int r = st.rows ? st.rows[i] : i;
            units[i] = slot_of(st, r) >= 0 ? units_of(position_of(st, r), st.window) : 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < st.n_rows; i += kA8Warps * 32) {
            const int n = units[i];
            int ahead = 0;                                         // rows before this one: no two have as many
            for (int j = 0; j < st.n_rows; ++j) ahead += units[j] > n || (units[j] == n && j < i);
            if (ahead == (int)blockIdx.y) mine = i;
        }
        __syncthreads();
        ridx = mine;
    }
    const int r = st.rows ? st.rows[ridx] : ridx, group = st.q_heads / st.kv_heads;
    const int slot = slot_of(st, r);
    bf16* dst = out + ((size_t)r * st.q_heads + (size_t)g * group) * HD;
    if (slot < 0) {
        for (int i = threadIdx.x; i < group * HD; i += blockDim.x) dst[i] = __float2bfloat16_rn(0.0f);
        return;
    }
    const A8Row x = row_at<HD>(st, r, slot, g);
    attend_run<HD, NT>(smem, x, st.cache, 0, units_of(x.pos, st.window));
    for (int i = threadIdx.x; i < group * HD; i += blockDim.x) {
        float acc, total, mm, dn;
        run_sums<HD, NT>(smem, i / HD, i % HD, acc, total, mm, dn);
        dst[i] = weighed(acc, dn, total);
    }
}

// Longer ones of few rows: a cluster of `size` blocks per (row, key/value head), each with an equal run of its keys, whose sums are added in
// the order of the keys through distributed shared memory.  One kernel, no scratch, and no plan to be made before the first key is fetched.
// (One row of 4095 keys for 32 heads on 8: 10.7 us, in shares 13.1, a block per head 34; 8 rows of up to 4096: 17 to 18, 20 to 23 and 34.)
constexpr int kA8MaxCluster = 8;
__device__ __forceinline__ float peer_float(uint32_t address, int rank) {
    float v;
    asm volatile("{\n\t.reg .b32 a;\n\t"
                 "mapa.shared::cluster.u32 a, %1, %2;\n\t"
                 "ld.shared::cluster.f32 %0, [a];\n\t}\n"
                 : "=f"(v)
                 : "r"(address), "r"(rank)
                 : "memory");
    return v;
}
template <int HD, int NT>
__global__ void __launch_bounds__(kA8Warps * 32, NT == 1 ? 3 : 2) attention_fp8_cluster_kernel(const A8Step st, int size, bf16* __restrict__ out) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr size_t kJoined = (size_t)kA8Warps * 8 * NT * (HD + 3) * sizeof(float), kSums = (size_t)8 * NT * (HD + 3) * sizeof(float);
    static_assert(kJoined + kSums <= (size_t)kA8Warps * kA8Stages * A8Unit<HD>::kBytes, "a block's sums lie behind its warps'");
    TLLM_PDL_WAIT();
    const int g = blockIdx.x / size, rank = (int)cluster_rank(), ridx = blockIdx.y;
    const int r = st.rows ? st.rows[ridx] : ridx, group = st.q_heads / st.kv_heads;
    const int slot = slot_of(st, r);
    bf16* dst = out + ((size_t)r * st.q_heads + (size_t)g * group) * HD;
    if (slot < 0) {                                                // for all of the cluster
        for (int i = rank * blockDim.x + threadIdx.x; i < group * HD; i += size * blockDim.x) dst[i] = __float2bfloat16_rn(0.0f);
        return;
    }
    const A8Row x = row_at<HD>(st, r, slot, g);
    const int units = units_of(x.pos, st.window), each = ((units + size - 1) / size + kA8Warps - 1) / kA8Warps * kA8Warps;
    const int u0 = min((long long)rank * each, (long long)units), u1 = min(u0 + each, units);
    attend_run<HD, NT>(smem, x, st.cache, u0, u1);
    float* o = reinterpret_cast<float*>(smem + kJoined);           // [8 NT][HD], then [8 NT][3]: M, D, sum
    float* m = o + 8 * NT * HD;
    for (int i = threadIdx.x; i < group * HD; i += kA8Warps * 32) {
        float acc, total, mm, dn;
        run_sums<HD, NT>(smem, i / HD, i % HD, acc, total, mm, dn);
        o[i] = acc;
        if (i % HD == 0) {
            float* to = m + i / HD * 3;
            to[0] = mm; to[1] = dn; to[2] = total;
        }
    }
    __syncwarp();
    cluster_sync();
    const uint32_t o_at = smem_u32(o), m_at = smem_u32(m);
    for (int i = rank * (kA8Warps * 32) + threadIdx.x; i < group * HD; i += size * kA8Warps * 32) {
        float runs[kA8MaxCluster * 3], sums[kA8MaxCluster];
#pragma unroll
        for (int s = 0; s < kA8MaxCluster; ++s) {
            const bool there = s < size;
            sums[s] = there ? peer_float(o_at + i * 4, s) : 0.0f;
#pragma unroll
            for (int e = 0; e < 3; ++e) runs[3 * s + e] = there ? peer_float(m_at + (i / HD * 3 + e) * 4, s) : e == 2 ? 0.0f : -INFINITY;
        }
        float acc, total, mm, dn;
        join_runs<kA8MaxCluster>(runs, 3, sums, 1, kA8MaxCluster, acc, total, mm, dn);
        dst[i] = weighed(acc, dn, total);
    }
    __syncwarp();
    cluster_sync();                                                // no block leaves while its sums are read
}

// Longer ones: the keys of all rows shared by all blocks of threads, whatever the rows' lengths, in one of two ways.
//   Chunks, where there are two blocks and more for every (row, head): each is cut into chunks of `each` units, the shortest that leave no chunk
//   without a block, and a block takes one.
//   Shares, where there are more (rows, heads) than that: all units in a row, (row, head, unit), are cut into equal shares; a share is the end of
//   one (row, head), whole ones, and the beginning of another.
// A (row, head) that one block has whole is written; pieces go to scratch.  Place of a chunk: its block; of the piece of (row, head) i in share b:
// i + b (no two pieces have the same, as every next piece is of the next pair, the next share or both).  Chunks and shares are whole rounds of the
// four warps.  plan: the chunks (units) of a head before each row, then 0 (the length of a share): the first block leaves it for the kernel
// that adds the pieces.  (A grid of equal runs per row, whose lengths differ: 64 rows of 1000 to 4096 keys 86 us however finely cut, in shares 73;
// shares alone, 8 rows of 500 to 2000 keys 21 us, as some blocks work on two pieces one after the other, in chunks 16.)
constexpr int kA8MaxRows = 512, kA8MaxShares = 512;
template <int HD, int NT>
__global__ void __launch_bounds__(kA8Warps * 32, NT == 1 ? 3 : 2)
attention_fp8_share_kernel(const A8Step st, int* __restrict__ plan, float* __restrict__ part_o, float* __restrict__ part_m, bf16* __restrict__ out) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int before[kA8MaxRows + 1], units[kA8MaxRows], sums[2][kA8Warps];
    TLLM_PDL_ENTER();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = st.q_heads / st.kv_heads, blocks = gridDim.x;
    int some = 0, rows_here = 0;
    for (int ridx = threadIdx.x; ridx < st.n_rows; ridx += kA8Warps * 32) {
        const int r = st.rows ? st.rows[ridx] : ridx;
        const int pos = position_of(st, r), slot = slot_of(st, r);
        const int n = slot >= 0 ? units_of(pos, st.window) : 0;
        units[ridx] = n;                                           // read back by this thread alone
        some += n;
        rows_here += n > 0;
    }
    int turn = 0;
    auto block_total = [&](int v) {
        v = __reduce_add_sync(0xffffffffu, v);
        if (lane == 0) sums[turn][warp] = v;
        __syncthreads();
        int t = 0;
#pragma unroll
        for (int i = 0; i < kA8Warps; ++i) t += sums[turn][i];
        turn ^= 1;
        return t;
    };
    const int total = block_total(some) * st.kv_heads;            // below 2^31 - 2^13: see the entry point
    int each = ((total + blocks - 1) / blocks + kA8Warps - 1) / kA8Warps * kA8Warps;
    if (each == 0) each = kA8Warps;
    const bool chunks = block_total(rows_here) * st.kv_heads * 2 <= blocks;
    if (chunks) {
        // the shortest of a few lengths, a sixteenth longer each time: with twice as many blocks as pairs, twice the mean length always does
        for (;;) {
            int c = 0;
            for (int ridx = threadIdx.x; ridx < st.n_rows; ridx += kA8Warps * 32) c += (units[ridx] + each - 1) / each;
            if (block_total(c) * st.kv_heads <= blocks) break;
            each += max(each / 16 / kA8Warps, 1) * kA8Warps;
        }
    }
    // chunks or units of a head before each row
    int all = 0;
    for (int first = 0; first < st.n_rows; first += kA8Warps * 32) {
        const int ridx = first + threadIdx.x;
        const int n = ridx < st.n_rows ? (chunks ? (units[ridx] + each - 1) / each : units[ridx]) : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        if (lane == 31) sums[turn][warp] = upto;
        __syncthreads();
        int offset = all + upto - n;
#pragma unroll
        for (int i = 0; i < kA8Warps; ++i) {
            if (i < warp) offset += sums[turn][i];
            all += sums[turn][i];
        }
        turn ^= 1;
        if (ridx < st.n_rows) before[ridx] = offset;
    }
    if (threadIdx.x == 0) before[st.n_rows] = all;
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int i = threadIdx.x; i <= st.n_rows; i += blockDim.x) plan[i] = before[i];
        if (threadIdx.x == 0) plan[st.n_rows + 1] = chunks ? 0 : each;
    }
    // in chunks or units, of all heads: this block's first and the one behind its last
    const int here = all * st.kv_heads;
    if ((long long)blockIdx.x * (chunks ? 1 : each) >= here) return;
    int at = blockIdx.x * (chunks ? 1 : each);
    const int end = chunks ? at + 1 : min(at + each, here);
    // the row that holds it: the last one with before * kv_heads <= at (rows with nothing are passed over)
    int ridx = 0;
    for (int step = st.n_rows > 64 ? kA8MaxRows / 2 : 32; step > 0; step >>= 1)
        if (ridx + step < st.n_rows && before[ridx + step] * st.kv_heads <= at) ridx += step;
    while (at < end) {
        const int n = before[ridx + 1] - before[ridx];
        if (n == 0) { ++ridx; continue; }
        const int in_row = at - before[ridx] * st.kv_heads, g = in_row / n, first = in_row - g * n;
        const int r = st.rows ? st.rows[ridx] : ridx;
        const A8Row x = row_at<HD>(st, r, st.token_slot[r], g);
        const int u0 = chunks ? first * each : first;
        const int u1 = chunks ? min(u0 + each, units_of(x.pos, st.window)) : min(n, u0 + end - at);
        attend_run<HD, NT>(smem, x, st.cache, u0, u1);
        const bool whole = chunks ? n == 1 : u0 == 0 && u1 == n;
        const size_t place = ((chunks ? (size_t)0 : (size_t)ridx * st.kv_heads + g) + blockIdx.x) * group;
        for (int i = threadIdx.x; i < group * HD; i += blockDim.x) {
            const int row = i / HD, d = i % HD;
            float acc, sum, mm, dn;
            run_sums<HD, NT>(smem, row, d, acc, sum, mm, dn);
            if (whole) {
                out[((size_t)r * st.q_heads + (size_t)g * group) * HD + i] = weighed(acc, dn, sum);
            } else {
                part_o[(place + row) * HD + d] = acc;
                if (d == 0) { part_m[(place + row) * 3] = mm; part_m[(place + row) * 3 + 1] = dn; part_m[(place + row) * 3 + 2] = sum; }
            }
        }
        if (chunks) return;
        at += u1 - u0;
        if (g == st.kv_heads - 1 && u1 == n) ++ridx;
        __syncthreads();                                           // the ring may be filled again
    }
}

// The pieces of a (row, head) added in the order of their keys.  A warp's lanes find the pieces' factors, 32 at a time, and add HD / 32 dims
// each, four pieces on their way at once.  WIDE (few heads of many pieces): the warps of a block share a head's pieces, and their sums are
// added in order; else each takes a head of the group.  Rows of no request become zeros here.  (512 threads per head, whatever the pieces,
// took 18 us for 2048 heads of two pieces each.)
constexpr int kA8JoinWarps = 8;
template <int HD, bool WIDE>
__global__ void __launch_bounds__(kA8JoinWarps * 32)
attention_fp8_join_kernel(const A8Step st, const int* plan, const float* part_o, const float* part_m, bf16* __restrict__ out) {
    constexpr int kDims = HD / 32;
    __shared__ float sums[WIDE ? kA8JoinWarps : 1][HD];
    TLLM_PDL_ENTER();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, ridx = blockIdx.y;       // WIDE: kA8JoinWarps warps
    const int r = st.rows ? st.rows[ridx] : ridx, group = st.q_heads / st.kv_heads, slot = slot_of(st, r);
    const int before = plan[ridx], n = plan[ridx + 1] - before, each = plan[st.n_rows + 1];
    const int g = WIDE ? blockIdx.x / group : blockIdx.x;
    const int start = before * st.kv_heads + g * n, b0 = each == 0 ? start : start / each;
    const int pieces = each == 0 ? n : (start + n - 1) / each - b0 + 1;
    if (slot >= 0 && pieces == 1) return;                          // written where it was made
    const int first = WIDE ? blockIdx.x % group : warp, step = WIDE ? group : warps;
    for (int h = first; h < group; h += step) {
        bf16* dst = out + ((size_t)r * st.q_heads + g * group + h) * HD + lane * kDims;
        if (slot < 0) {
            if (!WIDE || warp == 0)
#pragma unroll
                for (int i = 0; i < kDims; ++i) dst[i] = __float2bfloat16_rn(0.0f);
            continue;
        }
        const size_t base = ((each == 0 ? (size_t)0 : (size_t)ridx * st.kv_heads + g) + b0) * group + h;      // the first piece's place
        const float* me = part_m + base * 3;
        const float* oe = part_o + base * HD + lane * kDims;
        // the first pieces' numbers and values, all on their way at once
        constexpr int kAhead = 4, kApart = WIDE ? kA8JoinWarps : 1;
        const int mine = WIDE ? warp : 0;
        const bool there = lane < pieces;
        const float m0 = there ? me[lane * group * 3] : -INFINITY, d0 = there ? me[lane * group * 3 + 1] : -INFINITY;
        const float l0 = there ? me[lane * group * 3 + 2] : 0.0f;
        float ahead[kAhead][kDims];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
#pragma unroll
            for (int e = 0; e < kDims; ++e) ahead[i][e] = mine + i * kApart < pieces ? oe[(size_t)(mine + i * kApart) * group * HD + e] : 0.0f;
        float mm = m0, dn = -INFINITY, total = 0.0f;
        for (int p = lane + 32; p < pieces; p += 32) mm = fmaxf(mm, me[p * group * 3]);
        mm = warp_max(mm);
        // a piece without keys has M of -infinity and sums of zero; scores that are all NaN leave M so too, and l NaN
        auto take = [&](float m, float d, float l) {
            total += m == -INFINITY ? l : l * exp2f(m - mm);
            if (m != -INFINITY) dn = fmaxf(dn, d + (m - mm));
        };
        take(m0, d0, l0);
        for (int p = lane + 32; p < pieces; p += 32) take(me[p * group * 3], me[p * group * 3 + 1], me[p * group * 3 + 2]);
        dn = warp_max(dn);
        total = warp_sum(total);
        auto factor_of = [&](float m, float d) {
            const float of = m == -INFINITY ? -INFINITY : d + (m - mm);
            return of == -INFINITY ? 0.0f : exp2f(of - dn);
        };
        float acc[kDims];
#pragma unroll
        for (int i = 0; i < kDims; ++i) acc[i] = 0.0f;
        float factor = factor_of(m0, d0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const float f = __shfl_sync(0xffffffffu, factor, mine + i * kApart);                 // at most piece 31
#pragma unroll
            for (int e = 0; e < kDims; ++e) acc[e] = fmaf(ahead[i][e], f, acc[e]);
        }
        for (int p0 = 0, from = mine + kAhead * kApart; p0 < pieces; p0 += 32, from = mine) {
            if (p0 > 0) {
                const int p = p0 + lane;
                factor = p < pieces ? factor_of(me[p * group * 3], me[p * group * 3 + 1]) : 0.0f;
            }
            const int count = min(32, pieces - p0);
#pragma unroll 4
            for (int i = from; i < count; i += kApart) {
                const float f = __shfl_sync(0xffffffffu, factor, i);
                const float* o = oe + (size_t)(p0 + i) * group * HD;
#pragma unroll
                for (int e = 0; e < kDims; ++e) acc[e] = fmaf(o[e], f, acc[e]);
            }
        }
        if (WIDE) {
#pragma unroll
            for (int e = 0; e < kDims; ++e) sums[warp][lane * kDims + e] = acc[e];
            __syncthreads();
            if (warp != 0) return;
#pragma unroll
            for (int i = 1; i < kA8JoinWarps; ++i)
#pragma unroll
                for (int e = 0; e < kDims; ++e) acc[e] += sums[i][lane * kDims + e];
        }
#pragma unroll
        for (int e = 0; e < kDims; ++e) dst[e] = weighed(acc[e], dn, total);
        if (WIDE) return;
    }
}

template <int HD, int NT>
static int launch_attention_fp8(const A8Step& st, int blocks, int cluster, int* plan, float* part_o, float* part_m, void* out, cudaStream_t stream) {
    constexpr size_t ring = (size_t)kA8Warps * kA8Stages * A8Unit<HD>::kBytes, joined = (size_t)kA8Warps * 8 * NT * (HD + 3) * sizeof(float);
    constexpr size_t smem = ring > joined ? ring : joined;
    static OncePerDevice configured;
    if (configured.first()) {
        cudaError_t e = cudaFuncSetAttribute(attention_fp8_whole_kernel<HD, NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_fp8_whole_kernel<HD, NT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_fp8_cluster_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(attention_fp8_share_kernel<HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) { set_error("attention_fp8_decode: %s", cudaGetErrorString(e)); return (int)e; }
        configured.done();
    }
    if (cluster > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(cluster * st.kv_heads, st.n_rows);
        cfg.blockDim = dim3(kA8Warps * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = cluster;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t e = cudaLaunchKernelEx(&cfg, attention_fp8_cluster_kernel<HD, NT>, st, cluster, (bf16*)out);
        if (e != cudaSuccess) { set_error("attention_fp8_cluster: %s", cudaGetErrorString(e)); return (int)e; }
        return finish_launch("attention_fp8_cluster");
    }
    if (blocks == 0) {
        int sms = sm_count_cached();
        if (sms <= 0) sms = 148;
        auto kernel = st.n_rows <= kA8MaxOrdered && (long long)st.n_rows * st.kv_heads > (NT == 1 ? 3 : 2) * sms ? attention_fp8_whole_kernel<HD, NT, true>
                                                                                                           : attention_fp8_whole_kernel<HD, NT, false>;
        launch_pdl(kPdlAttention, kernel, dim3(st.kv_heads, st.n_rows), dim3(kA8Warps * 32), smem, stream, st, (bf16*)out);
        return finish_launch("attention_fp8_whole");
    }
    launch_pdl(kPdlAttention, attention_fp8_share_kernel<HD, NT>, dim3(blocks), dim3(kA8Warps * 32), smem, stream, st, plan, part_o, part_m, (bf16*)out);
    const int rc = finish_launch("attention_fp8_share");
    if (rc != 0) return rc;
    const int group = st.q_heads / st.kv_heads;
    if ((long long)st.n_rows * st.kv_heads * 8 <= blocks)         // eight pieces a head and more, on average
        launch_pdl(kPdlCombine, attention_fp8_join_kernel<HD, true>, dim3(st.q_heads, st.n_rows), dim3(kA8JoinWarps * 32), 0, stream, st,
                   (const int*)plan, (const float*)part_o, (const float*)part_m, (bf16*)out);
    else
        launch_pdl(kPdlCombine, attention_fp8_join_kernel<HD, false>, dim3(st.kv_heads, st.n_rows), dim3((group < kA8JoinWarps ? group : kA8JoinWarps) * 32),
                   0, stream, st, (const int*)plan, (const float*)part_o, (const float*)part_m, (bf16*)out);
    return finish_launch("attention_fp8_join");
}

// ---------------------------------------------------------------- pages back in bfloat16
// For the portions (segments of more than one token) of a step: the pages that a portion's tokens may read, from the one that holds the
// first key of its first token's window to the last token's, become pages of `pages` ([pages][keys, values][kv head][token][HD] bfloat16),
// one portion after the other, and table[slot] lists them (-1 elsewhere).  The prompt kernels then read those.  One block of threads per
// page; bound by HBM.
// Portions that share pages (a common prefix) may list many times more than the cache has: then a page goes to the place of its own
// number, `pages` as many as the cache's (kTails, kTokens).  Its tokens up to the last that any portion counts are written, all alike by
// whichever portions list it; behind a portion's last token come zeros first, by a launch of their own, as another portion may go on there.
enum A8Unpack : int { kInTurn = 0, kTails = 1, kTokens = 2 };
template <int HD>
__global__ void __launch_bounds__(256) attention_fp8_unpack_kernel(const A8Cache cache, const int* __restrict__ seg_info,
                                                                   const int* __restrict__ block_table, int max_pages, int page_size,
                                                                   int kv_heads, int window, int capacity, int places, bf16* __restrict__ pages,
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
    const int listed = cache.held(block_table[(size_t)slot * max_pages + i]);
    int to = listed;
    if (places == kInTurn) {
        to = blockIdx.x;
        for (int s = 0; s < seg; ++s)
            if (seg_info[4 * s + 2] > 1 && seg_info[4 * s] >= 0)
                to += (seg_info[4 * s + 3] + seg_info[4 * s + 2] - 1) / page_size - first_page(seg_info[4 * s + 3]) + 1;
    }
    const int page = to < capacity ? listed : -1;
    if (threadIdx.x == 0) table[(size_t)slot * max_pages + i] = page < 0 ? -1 : to;
    if (page < 0 || (places == kTails && (i + 1) * page_size - 1 <= last)) return;
    const size_t at = (size_t)page * cache.stride, plane = (size_t)kv_heads * page_size;
    const float* scales = reinterpret_cast<const float*>(cache.scales + at);
    bf16* dst = pages + (size_t)to * 2 * plane * HD;
    constexpr int kPer = HD / 16;                                  // 16-byte pieces of a head
    for (int n = threadIdx.x; n < 2 * (int)plane * kPer; n += blockDim.x) {
        const int token = n / kPer, which = token >= (int)plane, t = token - which * (int)plane;
        // tokens behind the last one hold what an earlier request left, or nothing: zeros instead
        const bool ok = i * page_size + t % page_size <= last;
        if (places == (ok ? kTails : kTokens)) continue;
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

static int check_a8(const char* what, const void* k, const void* v, const void* scales, long long page_bytes, int pages, int page_size, int kv_heads, int head_dim) {
    TLLM_REQUIRE(pages > 0, "%s: %d pages", what, pages);
    TLLM_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim %d is not 64 or 128", what, head_dim);
    TLLM_REQUIRE(kv_heads > 0 && kv_heads <= 65535, "%s: %d key/value heads", what, kv_heads);
    TLLM_REQUIRE(page_size > 0 && page_size % 16 == 0, "%s: page size %d is no multiple of 16", what, page_size);
    TLLM_REQUIRE(k && v && scales && page_bytes > 0 && page_bytes % 16 == 0 &&
                     ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(scales)) & 15u) == 0,
                 "%s: planes must be 16-byte aligned", what);
    return 0;
}

// q, out [rows, q_heads * head_dim] bfloat16; block_table [slots][max_pages]; planes of `pages` pages `page_bytes` apart: k, v [kv_heads][page_size][head_dim] e4m3, scales
// [kv_heads][page_size][2] float32.  rows: indices of the one-token rows, null for 0 .. n_rows - 1.  blocks: 0 for a block of threads per (row,
// key/value head), or with `cluster` (2, 4, 8) a cluster of them; else how many share all rows' keys (at most 512 rows and 512 blocks); then scratch, 16-byte aligned: float [(n_rows * kv_heads + blocks) *
// (q_heads / kv_heads) * (head_dim + 3)], int [n_rows + 2].
extern "C" int tllm_attention_fp8_decode(const void* q, const void* k, const void* v, const void* scales, long long page_bytes,
                                         int pages, const int* positions, const int* token_slot, const int* rows, int n_rows,
                                         const int* block_table, int slots, int max_pages, int page_size, int q_heads, int kv_heads, int head_dim, int window, float scale,
                                         int blocks, int cluster, float* scratch, void* out, cudaStream_t stream) {
    if (check_a8("attention_fp8_decode", k, v, scales, page_bytes, pages, page_size, kv_heads, head_dim) != 0) return -1;
    TLLM_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16,
                 "attention_fp8_decode: %d query heads over %d key/value heads (at most 16 per group)", q_heads, kv_heads);
    TLLM_REQUIRE(n_rows >= 0 && n_rows <= 65535 && q_heads <= 65535 && max_pages > 0 && window >= 0 && (long long)max_pages * page_size <= 0x7fffffff,
                 "attention_fp8_decode: bad grid");
    TLLM_REQUIRE(blocks >= 0 && blocks <= kA8MaxShares && (blocks == 0 || (n_rows <= kA8MaxRows && scratch)),
                 "attention_fp8_decode: %d rows shared by %d blocks (at most 512 and 512, with scratch)", n_rows, blocks);
    TLLM_REQUIRE(cluster == 1 || (blocks == 0 && (cluster == 2 || cluster == 4 || cluster == kA8MaxCluster)),
                 "attention_fp8_decode: clusters of %d blocks (1, 2, 4 or 8, without shares)", cluster);
    TLLM_REQUIRE(blocks == 0 || (long long)n_rows * kv_heads * ((long long)max_pages * page_size / kA8Unit + 1) < 0x7fffffff - (1 << 13),
                 "attention_fp8_decode: too many keys for shares");
    TLLM_REQUIRE(q && out && positions && token_slot && block_table && ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(scratch)) & 15u) == 0,
                 "attention_fp8_decode: missing or unaligned operands");
    if (n_rows == 0) return 0;
    const A8Step st{(const bf16*)q, A8Cache{(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)scales, page_bytes, pages}, positions, token_slot, rows,
                    block_table, n_rows, slots, max_pages, page_size, q_heads, kv_heads, window, max_pages * page_size, scale * 1.4426950408889634f};
    const int group = q_heads / kv_heads;
    const size_t places = ((size_t)n_rows * kv_heads + blocks) * group;
    float *part_o = scratch, *part_m = scratch + places * head_dim;
    int* plan = reinterpret_cast<int*>(part_m + places * 3);
#define ATTEND(HD, NT) return launch_attention_fp8<HD, NT>(st, blocks, cluster, plan, part_o, part_m, out, stream)
    if (head_dim == 64) {
        if (group <= 8) ATTEND(64, 1);
        ATTEND(64, 2);
    }
    if (group <= 8) ATTEND(128, 1);
    ATTEND(128, 2);
#undef ATTEND
}

// `held`: pages of the cache.  seg_info [segments][4] = slot, first row, tokens, position of the first.  `per`: pages of the portion that has most; pages bfloat16
// [capacity][2][kv_heads][page_size][head_dim], room for all portions' pages, or with `by_page` for as many as the cache has; table int32 like block_table.
extern "C" int tllm_attention_fp8_unpack(const void* k, const void* v, const void* scales, long long page_bytes, int held, const int* seg_info, int segments,
                                         const int* block_table, int max_pages, int page_size, int kv_heads, int head_dim, int window, int per,
                                         int capacity, int by_page, void* pages, int* table, cudaStream_t stream) {
    if (check_a8("attention_fp8_unpack", k, v, scales, page_bytes, held, page_size, kv_heads, head_dim) != 0) return -1;
    TLLM_REQUIRE(segments > 0 && segments <= 65535 && per > 0 && per <= max_pages && capacity > 0, "attention_fp8_unpack: bad sizes");
    TLLM_REQUIRE(seg_info && block_table && pages && table && (reinterpret_cast<uintptr_t>(pages) & 15u) == 0, "attention_fp8_unpack: missing operands");
    TLLM_REQUIRE((long long)2 * kv_heads * page_size * (head_dim / 16) <= 0x7fffffff && (long long)max_pages * page_size <= 0x7fffffff, "attention_fp8_unpack: too large");
    TLLM_REQUIRE(!by_page || capacity == held, "attention_fp8_unpack: %d places for the cache's %d pages", capacity, held);
    const A8Cache cache{(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)scales, page_bytes, held};
    auto kernel = head_dim == 64 ? attention_fp8_unpack_kernel<64> : attention_fp8_unpack_kernel<128>;
    for (int places = by_page ? kTails : kInTurn; places <= (by_page ? kTokens : kInTurn); ++places) {
        launch_pdl(kPdlOther, kernel, dim3(per, segments), dim3(256), 0, stream, cache, seg_info, block_table, max_pages, page_size, kv_heads, window,
                   capacity, places, (bf16*)pages, table);
        const int rc = finish_launch("attention_fp8_unpack");
        if (rc != 0) return rc;
    }
    return 0;
}
