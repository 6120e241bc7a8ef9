// Attention of new rows over the paged 8-bit cache (kv8.hpp has its format).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = log2(e) / sqrt(128) * scale_k * (q . u_j)
//
// over the rows j <= place of the query and, with a window, j > place - window or j < sinks.  The queries that share a kv head (n_rep of each new row) are
// the columns of both products, S^T = U_k Q^T and O^T = U_v^T P^T (v_mfma_f32_16x16x32_f16): codes are exact in fp16, a block's scale multiplies the fp32
// scores, one of V the weights, so that the one thing rounded below 32 bits is a weight, to fp16 (half a step: 2^-11 of it), before it counts in either sum.
// Softmax state (m, l) and sums are fp32; the running form lets a block be read once.
//
// Bound: HBM for a few queries a head (256 bytes a row and kv head), the matrix cores for many.
#include "kv8.hpp"

namespace smh {

struct Kv8AttnParams {
    const half_t *q;
    half_t *out;
    long q_stride;
    const int32_t *lens, *cu;
    Kv8Cache c;
    int T, B, H, Hkv, max_new, window, sinks, splits;
    float *part_o;                                 // [splits][T * H][128], not normalised
    float2 *part_ml;                               // [splits][T * H]
};

// What a run of rows sees of its sequence: blocks 0 .. sink_blocks - 1 and first .. last, `count` in all, of which the last may be the open one.
struct Kv8Span {
    int whole, open_rows;                          // whole blocks, rows of the open one
    int sink_blocks, first, count;
    __device__ __forceinline__ int block(int i) const { return i < sink_blocks ? i : first + i - sink_blocks; }
};
__device__ __forceinline__ Kv8Span kv8_span(const Kv8AttnParams &p, const Kv8Seq &s, int lo, int hi) {      // lo, hi: places of the first and last query
    Kv8Span v;
    const int total = kv8_kept(s.old + s.n, p.c.cols);
    v.whole = total >> 6;
    v.open_rows = total & 63;
    const int last = min(hi, total - 1) >> 6;
    v.first = 0;
    v.sink_blocks = 0;
    if (p.window > 0) {
        v.first = min(max(lo - p.window + 1, 0) >> 6, last + 1);
        v.sink_blocks = min(min((p.sinks + 63) >> 6, v.first), last + 1);
    }
    v.count = v.sink_blocks + last - v.first + 1;
    return v;
}

// The largest of the four lane groups' values, in all of them
__device__ __forceinline__ float max_of_groups(float v) {
    typedef float v2 __attribute__((ext_vector_type(2)));
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    v2 r = __builtin_bit_cast(v2, __builtin_amdgcn_permlane32_swap(u, u, false, false));      // (lower half twice, upper half twice)
    u = __builtin_bit_cast(uint32_t, fmaxf(r[0], r[1]));
    r = __builtin_bit_cast(v2, __builtin_amdgcn_permlane16_swap(u, u, false, false));
    return fmaxf(r[0], r[1]);
}

// A wave's queries: QT tiles of 16 columns, lane l has column l % 16.
template <int QT>
struct Kv8Wave {
    h8 q[QT][4];
    f4 o[QT][8];                                   // in units of `unit`
    float m[QT], l[QT];                            // the weights' reference, at most LAZY below the largest score; l: of the lane's own rows
    float unit;                                    // 1 .. 2^FALL times the scale of V that the wave had last; 0: none yet
    int at[QT];                                    // place of the query, -1: none
    int lo, hi;                                    // least and largest place of the wave's queries

    __device__ __forceinline__ void init(const Kv8AttnParams &p, const Kv8Seq &s, int kvh, int row0, int n_rep) {
        const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, rows = s.n * n_rep;
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            const int r = row0 + t * 16 + col;
            const int i = r / n_rep;
            at[t] = r < rows ? s.old + i : -1;
            const half_t *src = p.q + (long)(s.t0 + i) * p.q_stride + (long)(kvh * n_rep + r - i * n_rep) * KV8_DIM;
#pragma unroll
            for (int k = 0; k < 4; ++k) q[t][k] = r < rows ? *reinterpret_cast<const h8 *>(src + (k >> 1) * 64 + g * 16 + (k & 1) * 8) : h8{0, 0, 0, 0, 0, 0, 0, 0};
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[t][d] = f4{0, 0, 0, 0};
        }
        unit = 0.0f;
        lo = s.old + row0 / n_rep;
        hi = s.old + min(row0 + QT * 16 - 1, rows - 1) / n_rep;
    }

    // Scores of 64 rows -> weights, as the second product takes them: p * f, f = v_scale / unit, with the factor in the exponent and taken out of l again, so that
    // the product adds up in `unit`s by itself.  l must not lose a row because its V is small, so f stays in 2^-FALL .. 1: the unit goes up to a larger scale, and down to a far smaller
    // one by a power of two, and the sums go with it (exactly, where blocks of large and of small values take turns).  A block of zeros has no scale: its weights count in l alone.
    // masked: some row of the block may be out of some query's sight.  seen[t]: the lane's query sees a row of the block.
    // The reference follows the largest score only when that is 2^LAZY of weight ahead, and stands for a weight of 2^RAISE: weights are at most 2^14, and fp16's least exponent takes bits only
    // from those below 2^-22 / f of the largest, which is 2^-20 at most.  l adds up the rounded weights, so that what the sums are divided by is what they were made with.
    static constexpr float LAZY = 6.0f, RAISE = 8.0f;
    static constexpr int FALL = 2;
    __device__ __forceinline__ void softmax(f4 (&x)[QT][4], float scale, float v_scale, int block, bool masked, int limit, int window, int sinks, h8 (&w)[QT][2], bool (&seen)[QT]) {
        const int g = (threadIdx.x & 63) >> 4;
        // (compared as bits, which order as positive numbers do: as numbers the two bounds cost the reads 1 % of their rate)
        const uint32_t above = __builtin_bit_cast(uint32_t, v_scale) - (__builtin_bit_cast(uint32_t, unit) - ((uint32_t)FALL << 23));
        if (above > (uint32_t)FALL << 23 && v_scale > 0.0f) {
            float now = v_scale;
            if (v_scale < unit) {
                now = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, unit) & 0x7FFFFFu) | (__builtin_bit_cast(uint32_t, v_scale) & 0x7F800000u));
                if (now < v_scale) now *= 2.0f;
            }
            const float by = unit / now;
#pragma unroll
            for (int t = 0; t < QT; ++t)
#pragma unroll
                for (int d = 0; d < 8; ++d) o[t][d] *= by;
            unit = now;
        }
        // v_scale / unit: Markstein's correction of the quotient by an approximate reciprocal with its remainder (NaN stays NaN)
        const float inverse = __builtin_amdgcn_rcpf(unit), about = v_scale * inverse;
        const float f = v_scale == 0.0f ? 1.0f : __builtin_fmaf(__builtin_fmaf(-about, unit, v_scale), inverse, about);
        const float log_f = __builtin_amdgcn_logf(f), inverse_f = __builtin_amdgcn_rcpf(f);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            seen[t] = true;
            float by_scale = scale;
            if (masked) {
                const int top = min(at[t], limit - 1) - block * KV8_ROWS, low = window > 0 ? at[t] - window - block * KV8_ROWS : -1, first = sinks - block * KV8_ROWS;
                seen[t] = top >= 0 && (low < min(top, KV8_ROWS - 1) || first > 0);
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = k * 16 + g * 4 + i;
                        x[t][k][i] = r <= top && (r > low || r < first) ? x[t][k][i] * scale : -INFINITY;
                    }
                by_scale = 1.0f;
            }
            float top = x[t][0][0];
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = fmaxf(top, x[t][k][i]);
            top *= by_scale;                       // (a scale is not negative)
            if (__any(top > m[t] + LAZY)) {
                const float now = fmaxf(m[t], max_of_groups(top)), by = now == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m[t] - now);
                l[t] *= by;
#pragma unroll
                for (int d = 0; d < 8; ++d) o[t][d] *= by;
                m[t] = now;
            }
            const float off = RAISE + (seen[t] ? log_f : 0.0f) - (m[t] == -INFINITY ? 0.0f : m[t]);      // (nothing seen yet: weights of 0, not of -inf + inf)
            float sum = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const h2 e = {(half_t)__builtin_amdgcn_exp2f(__builtin_fmaf(x[t][k][i], by_scale, off)), (half_t)__builtin_amdgcn_exp2f(__builtin_fmaf(x[t][k][i + 1], by_scale, off))};
                    sum = __builtin_amdgcn_fdot2(e, h2{(half_t)1.0f, (half_t)1.0f}, sum, false);
                    w[t][k >> 1][(k & 1) * 4 + i] = e[0];
                    w[t][k >> 1][(k & 1) * 4 + i + 1] = e[1];
                }
            l[t] += sum * (seen[t] ? inverse_f : 1.0f);
        }
    }

    // l over the lane groups that share a query, sums in units of 1.  Scores that are all NaN leave no maximum: the lowest number stands in, so that the NaN in l is
    // not passed over.
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            l[t] += __shfl_xor(l[t], 16, 64);
            l[t] += __shfl_xor(l[t], 32, 64);
            if (l[t] != l[t] && m[t] == -INFINITY) m[t] = -3.0e38f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[t][d] *= unit;
        }
    }
};

__device__ __forceinline__ bool kv8_masked(const Kv8AttnParams &p, int block, int lo, int hi, int rows) {
    if (block * KV8_ROWS + 63 > lo || rows < KV8_ROWS) return true;
    return p.window > 0 && block * KV8_ROWS <= hi - p.window && (block + 1) * KV8_ROWS > p.sinks;
}

constexpr int KV8_MAX_SPLITS = 256;
constexpr float KV8_SCORE_SCALE = 0.08838834764831845f * 1.4426950408889634f;       // log2(e) / sqrt(128)

// The open block from memory: fp16 values, rows past its end absent.
template <int QT>
__device__ __forceinline__ void kv8_open_block(Kv8Wave<QT> &w, const Kv8AttnParams &p, const half_t *k, const half_t *v, int block, int rows) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    f4 x[QT][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        h8 a[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) a[s] = *reinterpret_cast<const h8 *>(k + (t * 16 + col) * KV8_DIM + (s >> 1) * 64 + g * 16 + (s & 1) * 8);
#pragma unroll
        for (int u = 0; u < QT; ++u) {
            x[u][t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 4; ++s) x[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[s], w.q[u][s], x[u][t], 0, 0, 0);
        }
    }
    h8 pr[QT][2];
    bool seen[QT];
    if (w.unit == 0.0f) w.unit = 1.0f;
    w.softmax(x, KV8_SCORE_SCALE, w.unit, block, true, block * KV8_ROWS + rows, p.window, p.sinks, pr, seen);
    const float by = 1.0f / w.unit;                // (V's values are in units of 1; a scale is 2^-24 / 127 at least)
#pragma unroll
    for (int d = 0; d < 8; ++d) {
        h8 a[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            a[u] = *reinterpret_cast<const h8 *>(v + (d * 16 + col) * KV8_ROWS + g * 16 + u * 8);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (u * 32 + (i >> 2) * 16 + g * 4 + (i & 3) >= rows) a[u][i] = (half_t)0.0f;      // (what is there may be anything)
        }
#pragma unroll
        for (int t = 0; t < QT; ++t) {
            f4 s = {0, 0, 0, 0};
#pragma unroll
            for (int u = 0; u < 2; ++u) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[u], pr[t][u], s, 0, 0, 0);
            if (seen[t]) w.o[t][d] += s * by;
        }
    }
}

// ---- up to 32 queries a sequence and kv head ------------------------------------------------------------------------------------
// The four waves of a workgroup take alternate blocks of their part of the sequence, each for all queries (QT tiles), straight from memory into the operands: K of the
// next block is asked for behind the products with this one's, V ahead of them.  Their states meet in LDS.
// Bound by HBM: 80 sequences of up to 8192 rows, 64 heads over 8, 187 us (926 MB, 4.96 TB/s: uneven lengths, of one length 5.8 .. 6.05); 16 windows of 4096 rows of 32 heads 100 us (538 MB, 5.4 TB/s).
// Two waves a SIMD: with three the registers do not suffice (us, two and three: 194 and 202, 108 and 117).
template <int QT>
__global__ __launch_bounds__(256, 2) void kv8_attn_few_kernel(Kv8AttnParams p) {
    extern __shared__ float lds[];
    const int kvh = blockIdx.x, split = blockIdx.y, b = blockIdx.z;
    const Kv8Seq s = kv8_seq(p.lens, p.cu, b, p.T, p.max_new);
    if (s.n == 0) return;
    const int n_rep = p.H / p.Hkv, lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4, rows = s.n * n_rep;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    Kv8Wave<QT> w;
    w.init(p, s, kvh, 0, n_rep);
    const Kv8Span v = kv8_span(p, s, w.lo, w.hi);
    const int per = (v.count + p.splits - 1) / p.splits, begin = split * per, end = min(begin + per, v.count);
    const bool has_open = v.count > 0 && v.open_rows > 0 && v.block(v.count - 1) == v.whole;
    const int end8 = min(end, v.count - (has_open ? 1 : 0));
    const int32_t *pages = p.c.pages + (long)b * p.c.pages_stride;
    auto tile_of = [&](int i) { return min(max((long)pages[v.block(i)], 0L), p.c.n_pages - 1) * p.Hkv + kvh; };

    u32x4 kw[4][2], vw[8];
    auto ask_k = [&](long tile) {
        const uint8_t *k = p.c.k + tile * KV8_TILE + col * KV8_DIM + g * 16;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) kw[t][h] = *reinterpret_cast<const u32x4 *>(k + t * 16 * KV8_DIM + h * 64);
    };
    int i = begin + wave;
    long tile = 0;
    float2 sc = make_float2(0, 0);
    if (i < end8) {
        tile = tile_of(i);
        ask_k(tile);
        sc = *reinterpret_cast<const float2 *>(p.c.scales + tile * 2);
    }
    for (; i < end8; i += 4) {
        const uint8_t *vp = p.c.v + tile * KV8_TILE + col * KV8_ROWS + g * 16;
#pragma unroll
        for (int d = 0; d < 8; ++d) vw[d] = *reinterpret_cast<const u32x4 *>(vp + d * 16 * KV8_ROWS);
        f4 x[QT][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int u = 0; u < QT; ++u) x[u][t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const h8 a = kv8_codes8(kw[t][k >> 1][(k & 1) * 2], kw[t][k >> 1][(k & 1) * 2 + 1]);
#pragma unroll
                for (int u = 0; u < QT; ++u) x[u][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w.q[u][k], x[u][t], 0, 0, 0);
            }
        }
        const float2 sc_now = sc;
        const int block = v.block(i);
        if (i + 4 < end8) {
            tile = tile_of(i + 4);
            ask_k(tile);
            sc = *reinterpret_cast<const float2 *>(p.c.scales + tile * 2);
        }
        h8 pr[QT][2];
        bool seen[QT];
        w.softmax(x, sc_now.x * KV8_SCORE_SCALE, sc_now.y, block, kv8_masked(p, block, w.lo, w.hi, KV8_ROWS), (block + 1) * KV8_ROWS, p.window, p.sinks, pr, seen);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const h8 a0 = kv8_codes8(vw[d][0], vw[d][1]), a1 = kv8_codes8(vw[d][2], vw[d][3]);
#pragma unroll
            for (int t = 0; t < QT; ++t) {
                w.o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pr[t][0], w.o[t][d], 0, 0, 0);
                w.o[t][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pr[t][1], w.o[t][d], 0, 0, 0);
            }
        }
    }
    if (has_open && v.count - 1 >= begin && v.count - 1 < end && ((v.count - 1 - begin) & 3) == wave) {
        const long head = (long)b * p.Hkv + kvh;
        kv8_open_block<QT>(w, p, p.c.open_k + head * KV8_TILE, p.c.open_v + head * KV8_TILE, v.whole, v.open_rows);
    }
    w.finish();
    // the waves' states: [wave][16 queries][128 + 4] and (m, l)
    constexpr int PITCH = KV8_DIM + 4;
    float *lo = lds;
    float2 *ml = reinterpret_cast<float2 *>(lds + 4 * 16 * PITCH);
    const int row = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 8;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
        if (t > 0) __syncthreads();
#pragma unroll
        for (int d = 0; d < 8; ++d) *reinterpret_cast<f4 *>(lo + (wave * 16 + col) * PITCH + d * 16 + g * 4) = w.o[t][d];
        if (g == 0) ml[wave * 16 + col] = make_float2(w.m[t], w.l[t]);
        __syncthreads();
        const int r = t * 16 + row;
        if (r >= rows) continue;
        float top = -INFINITY, l = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = fmaxf(top, ml[k * 16 + row].x);
        const float zero = top == -INFINITY ? 0.0f : top;
        f4 a = {0, 0, 0, 0}, c = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float by = __builtin_amdgcn_exp2f(ml[k * 16 + row].x - zero);
            l += ml[k * 16 + row].y * by;
            a += *reinterpret_cast<const f4 *>(lo + (k * 16 + row) * PITCH + d0) * by;
            c += *reinterpret_cast<const f4 *>(lo + (k * 16 + row) * PITCH + d0 + 4) * by;
        }
        const int tok = r / n_rep;
        const long out = (long)(s.t0 + tok) * p.H + kvh * n_rep + r - tok * n_rep;
        if (p.splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            h8 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) { y[e] = (half_t)(a[e] * inv); y[4 + e] = (half_t)(c[e] * inv); }
            *reinterpret_cast<h8 *>(p.out + out * KV8_DIM + d0) = y;
        } else {
            const long at = (long)split * p.T * p.H + out;
            if ((threadIdx.x & 15) == 0) p.part_ml[at] = make_float2(top, l);
            if (top != -INFINITY) {
                *reinterpret_cast<f4 *>(p.part_o + at * KV8_DIM + d0) = a;
                *reinterpret_cast<f4 *>(p.part_o + at * KV8_DIM + d0 + 4) = c;
            }
        }
    }
}

// ---- many queries -------------------------------------------------------------------------------------------------------------
// Four waves have QT * 16 queries each and go through the same blocks; a block's codes become fp16 once for all of them, in LDS, in the order in which the lanes
// read their operands (1 KB a read, no bank twice).  AHEAD blocks of codes are on their way in registers; with two BUFFERS a block costs one barrier.
// Bound by the sum of LDS reads (32 KB a wave and block), exponentials and MFMAs, each about half of the time: a chunk of 2048 tokens of 64 heads over 8 behind 6144 rows
// 494 us (974 TFLOP/s; an 8192^3 fp16 library product reaches 1182).  Steps there, us: 980 as first written; 495 with two waves a SIMD (the register limit in the launch bounds), the scale
// of V in the exponent instead of 64 multiply-adds a block, a reference that follows lazily, one barrier instead of two.  Wave priorities around the products: 500 to 515.
template <int QT, int AHEAD, int BUFFERS>
__global__ __launch_bounds__(256, QT == 1 ? 4 : 2) void kv8_attn_many_kernel(Kv8AttnParams p) {
    extern __shared__ float lds[];
    const int kvh = blockIdx.x % p.Hkv, b = blockIdx.x / p.Hkv, split = blockIdx.z;
    const Kv8Seq s = kv8_seq(p.lens, p.cu, b, p.T, p.max_new);
    const int n_rep = p.H / p.Hkv, rows = s.n * n_rep;
    // The last queries have the most to see: they begin first.  Where all workgroups run at a time, two a compute unit, the second half goes the other way round.
    const int groups = gridDim.y, half = (groups + 1) / 2, all = gridDim.x * groups * gridDim.z;
    const int row0 = (all > 256 && all <= 512 && (int)blockIdx.y >= half ? (int)blockIdx.y - half : groups - 1 - (int)blockIdx.y) * (QT * 64);
    if (row0 >= rows) return;
    const int t = threadIdx.x, lane = t & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    Kv8Wave<QT> w;
    w.init(p, s, kvh, row0 + wave * QT * 16, n_rep);
    const bool idle = row0 + wave * QT * 16 >= rows;
    const Kv8Span v = kv8_span(p, s, s.old + row0 / n_rep, s.old + min(row0 + QT * 64 - 1, rows - 1) / n_rep);
    const int per = (v.count + p.splits - 1) / p.splits, begin = split * per, end = min(begin + per, v.count);
    const bool has_open = v.count > 0 && v.open_rows > 0 && v.block(v.count - 1) == v.whole;
    const int end8 = min(end, v.count - (has_open ? 1 : 0));
    const int32_t *pages = p.c.pages + (long)b * p.c.pages_stride;
    auto tile_of = [&](int i) { return min(max((long)pages[v.block(i)], 0L), p.c.n_pages - 1) * p.Hkv + kvh; };
    u32x4 kw[AHEAD][2], vw[AHEAD][2];
    float2 sc[AHEAD];
    auto ask = [&](int i, u32x4 (&kw)[2], u32x4 (&vw)[2], float2 &sc) {
        const long tile = tile_of(i);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                                  // wave: tile of 16 rows; two halves of their dims
            kw[h] = *reinterpret_cast<const u32x4 *>(p.c.k + tile * KV8_TILE + (wave * 16 + col) * KV8_DIM + h * 64 + g * 16);
            vw[h] = *reinterpret_cast<const u32x4 *>(p.c.v + tile * KV8_TILE + ((wave * 2 + h) * 16 + col) * KV8_ROWS + g * 16);
        }
        sc = *reinterpret_cast<const float2 *>(p.c.scales + tile * 2);
    };
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
        sc[a] = make_float2(0, 0);
        if (begin + a < end8) ask(begin + a, kw[a], vw[a], sc[a]);
    }
    for (int i0 = begin; i0 < end8; i0 += AHEAD)
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) {
        const int i = i0 + a;
        if (i >= end8) break;
        // two buffers: who writes one has passed the barrier behind the last reads of it
        if (BUFFERS == 1) __syncthreads();
        h8 *kl = reinterpret_cast<h8 *>(lds) + (BUFFERS == 1 ? 0 : (i - begin) & 1) * 2048, *vl = kl + 1024;      // [tile][k step][lane], [dims of 16][half][lane]
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                kl[(wave * 4 + h * 2 + e) * 64 + lane] = kv8_codes8(kw[a][h][e * 2], kw[a][h][e * 2 + 1]);
                vl[((wave * 2 + h) * 2 + e) * 64 + lane] = kv8_codes8(vw[a][h][e * 2], vw[a][h][e * 2 + 1]);
            }
        const float2 sc_now = sc[a];
        const int block = v.block(i);
        if (i + AHEAD < end8) ask(i + AHEAD, kw[a], vw[a], sc[a]);
        __syncthreads();
        if (idle || block * KV8_ROWS > w.hi) continue;                 // (nothing there for this wave)
        f4 x[QT][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
#pragma unroll
            for (int u = 0; u < QT; ++u) x[u][k] = f4{0, 0, 0, 0};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const h8 a = kl[(k * 4 + e) * 64 + lane];
#pragma unroll
                for (int u = 0; u < QT; ++u) x[u][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, w.q[u][e], x[u][k], 0, 0, 0);
            }
        }
        h8 pr[QT][2];
        bool seen[QT];
        w.softmax(x, sc_now.x * KV8_SCORE_SCALE, sc_now.y, block, kv8_masked(p, block, w.lo, w.hi, KV8_ROWS), (block + 1) * KV8_ROWS, p.window, p.sinks, pr, seen);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
            const h8 a0 = vl[(d * 2) * 64 + lane], a1 = vl[(d * 2 + 1) * 64 + lane];
#pragma unroll
            for (int u = 0; u < QT; ++u) {
                w.o[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a0, pr[u][0], w.o[u][d], 0, 0, 0);
                w.o[u][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a1, pr[u][1], w.o[u][d], 0, 0, 0);
            }
        }
    }
    if (idle) return;
    if (has_open && v.count - 1 >= begin && v.count - 1 < end && v.whole * KV8_ROWS <= w.hi) {
        const long head = (long)b * p.Hkv + kvh;
        kv8_open_block<QT>(w, p, p.c.open_k + head * KV8_TILE, p.c.open_v + head * KV8_TILE, v.whole, v.open_rows);
    }
    w.finish();
#pragma unroll
    for (int u = 0; u < QT; ++u) {
        const int r = row0 + (wave * QT + u) * 16 + col;
        if (r >= rows) continue;
        const int tok = r / n_rep;
        const long out = (long)(s.t0 + tok) * p.H + kvh * n_rep + r - tok * n_rep;
        if (p.splits == 1) {
            const float inv = w.l[u] == 0.0f ? 0.0f : 1.0f / w.l[u];
#pragma unroll
            for (int d = 0; d < 8; ++d) {
                h4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (half_t)(w.o[u][d][e] * inv);
                *reinterpret_cast<h4 *>(p.out + out * KV8_DIM + d * 16 + g * 4) = y;
            }
        } else {
            const long at = (long)split * p.T * p.H + out;
            if (g == 0) p.part_ml[at] = make_float2(w.m[u], w.l[u]);
            if (w.m[u] != -INFINITY) {
#pragma unroll
                for (int d = 0; d < 8; ++d) *reinterpret_cast<f4 *>(p.part_o + at * KV8_DIM + d * 16 + g * 4) = w.o[u][d];
            }
        }
    }
}

// The parts of each query: half a wave a query, four dims a lane.  Everything is asked for at once - the sequence that the row belongs to, (m, l), the sums of the first
// parts - and what turns out to be none's is not used (32768 queries in two parts: 10.3 us, 25.8 where each waited for the one before).
__global__ __launch_bounds__(256) void kv8_attn_merge_kernel(Kv8AttnParams p) {
    __shared__ float weights[8][KV8_MAX_SPLITS];
    const long rows = (long)p.T * p.H, r0 = (long)blockIdx.x * 8 + (threadIdx.x >> 5), r = min(r0, rows - 1);
    const int lane = threadIdx.x & 31, n = p.splits;
    float *weight = weights[threadIdx.x >> 5];
    const float *o = p.part_o + r * KV8_DIM + lane * 4;
    f4 x[8];
    auto ask = [&](int s0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (s0 + i < n) x[i] = *reinterpret_cast<const f4 *>(o + (s0 + i) * rows * KV8_DIM);
    };
    const float2 mine = p.part_ml[min(lane, n - 1) * rows + r];        // of the first 32 parts
    ask(0);
    bool there = r0 < rows;
    if (p.cu != nullptr) {                         // rows of no sequence (behind the last one, past max_new) have no parts
        const int tok = (int)(r / p.H);
        int lo = 0, hi = p.B;                      // the last sequence that begins at or before the row
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.cu[mid] <= tok) lo = mid;
            else hi = mid;
        }
        const Kv8Seq s = kv8_seq(p.lens, p.cu, lo, p.T, p.max_new);
        there = there && tok >= s.t0 && tok < s.t0 + s.n;
    }
    float top = lane < n ? mine.x : -INFINITY, l = 0.0f;
    for (int s = lane + 32; s < n; s += 32) top = fmaxf(top, p.part_ml[s * rows + r].x);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 32));
    const float zero = top == -INFINITY ? 0.0f : top;
    for (int s = lane; s < n; s += 32) {
        const float2 ml = s < 32 ? mine : p.part_ml[s * rows + r];
        const bool none = ml.x == -INFINITY;       // a part that saw nothing left no sums
        const float by = none ? 0.0f : __builtin_amdgcn_exp2f(ml.x - zero);
        l += none ? 0.0f : ml.y * by;
        weight[s] = by;
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) l += __shfl_xor(l, s, 32);
    __syncthreads();
    f4 a = {0, 0, 0, 0};
    for (int s0 = 0; s0 < n; s0 += 8) {
        if (s0 > 0) ask(s0);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float by = s0 + i < n ? weight[s0 + i] : 0.0f;
            if (by != 0.0f) a += x[i] * by;
        }
    }
    if (!there) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    h4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (half_t)(a[e] * inv);
    *reinterpret_cast<h4 *>(p.out + r * KV8_DIM + lane * 4) = y;
}

}  // namespace smh

using namespace smh;

namespace {
struct Kv8Plan { int tiles, rows, splits; long groups; };  // tiles of 16 queries of a wave (0: many), queries a workgroup has then, parts of a sequence
// Blocks that a sequence of up to max_len rows shows its queries, from above
long kv8_blocks(int max_new, long max_len, int window, int sinks) {
    long n = (max_len + 63) / 64;
    if (window > 0) {
        const long w = ((long)window + max_new + 62) / 64 + 1 + (sinks + 63) / 64;
        n = n < w ? n : w;
    }
    return n < 1 ? 1 : n;
}
// Parts of a sequence: as many as fill the compute units once with what runs there at a time (2 workgroups, of 64 queries 4), of four blocks at least; more parts are
// more sums to write and merge.  us with 512 / 1024 / 2048 / 4096 workgroups wanted: 3 sequences of 130000 rows, 64 heads over 8, one token each, 102 / 109 / 116 / 128;
// 12 of 8000, four tokens, 39 / 42 / 48 / 55; one of 4095, 32 heads, 13 each; with 256: 113, 46, 14.
// With 128 workgroups and more without parts those are of eight blocks at least (512 new tokens, 64 heads over 8, one part or two: 27 and 36 us; 300 new ones of two heads behind 5000
// rows, which are few workgroups, 26 and 21 with eight and four blocks).
// Up to 12 blocks a sequence are one part, without a second launch (one token of 32 heads, us in parts and in one: 512 rows 10.7 and 6.9, 701 rows 11.1 and 9.5, 1001 rows 10.5 and 11.1), with
// 128 workgroups and more up to 40 (8 such sequences of 1500 and 2400 rows 22.1 and 19.8, 28.3 and 25.1; 20 of 64 heads over 8 17.7 and 16.0, 21.5 and 21.3).
// 33 .. 64 queries: tiles of one wave each over shared codes (3 x 130000 rows, five tokens of 8 queries, 140 us; three tiles in a wave, one wave a SIMD, 144; two waves a block, two tiles
// each, 161).  Up to 32 queries waves of their own: four tokens 123 and 138 us.  64 queries a workgroup, four of which run at a time, also where the sequences are short: 500 tokens of 32
// heads 19.7 us, 22.7 with 128 queries, 512 of 64 over 8 22.9 and 27.2; 2000 of 64 over 8 100 and 96.
Kv8Plan kv8_plan(int B, int H, int Hkv, int max_new, long max_len, int window, int sinks) {
    const long rows = (long)max_new * (H / Hkv), blocks = kv8_blocks(max_new, max_len, window, sinks);
    Kv8Plan p;
    p.tiles = rows <= 32 ? (int)((rows + 15) / 16) : 0;
    p.rows = rows <= 64 || blocks <= 16 ? 64 : 128;
    p.groups = p.tiles ? 1 : (rows + p.rows - 1) / p.rows;
    const long base = (long)B * Hkv * p.groups, want = (p.tiles || p.rows == 128 ? 512 : 1024) / base, most = blocks / (base < 128 ? 4 : 8);
    long s = want < most ? want : most;
    if (p.tiles && blocks <= (base >= 128 ? 40 : 12)) s = 1;
    p.splits = (int)(s < 1 ? 1 : s > KV8_MAX_SPLITS ? KV8_MAX_SPLITS : s);
    return p;
}
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
}  // namespace

extern "C" size_t smh_kv8_attn_workspace_bytes(int T, int B, int H, int Hkv, int max_new, long max_len, int window, int sinks) {
    if (T < 1 || B < 1 || Hkv < 1 || H < Hkv || H % Hkv != 0 || max_new < 1 || max_len < 1 || window < 0 || sinks < 0) return 0;
    const Kv8Plan p = kv8_plan(B, H, Hkv, max_new < T ? max_new : T, max_len, window, sinks);
    return p.splits == 1 ? 0 : (size_t)p.splits * T * H * (KV8_DIM + 2) * sizeof(float);
}

extern "C" int smh_kv8_attn(const void *q, void *out, int T, int B, int H, int Hkv, int D, long q_stride, const int32_t *lens, const int32_t *cu, int max_new, long max_len, int window,
                            int sinks, const void *codes_k, const void *codes_v, const void *scales, const void *open_k, const void *open_v, const int32_t *pages, long n_pages,
                            long pages_stride, int pages_cols, void *workspace, size_t workspace_bytes, smh_stream_t stream) {
    SMH_REQUIRE(D == KV8_DIM, "smh_kv8_attn: head dim %d (only 128)", D);
    SMH_REQUIRE(B >= 1 && B <= 65535 && Hkv >= 1 && Hkv <= 4096 && H >= Hkv && H % Hkv == 0 && H <= 65535, "smh_kv8_attn: B=%d (1 .. 65535) H=%d Hkv=%d (1 .. 4096)", B, H, Hkv);
    SMH_REQUIRE(T >= 0 && max_new >= 0 && max_new <= KV8_MAX_LEN && max_len >= 1 && window >= 0 && window <= KV8_MAX_LEN && sinks >= 0 && sinks <= KV8_MAX_LEN,
                "smh_kv8_attn: T=%d max_new=%d max_len=%ld window=%d sinks=%d", T, max_new, max_len, window, sinks);
    SMH_REQUIRE(cu || (T == B && max_new == 1), "smh_kv8_attn: without cu every sequence has one row: T=%d B=%d max_new=%d", T, B, max_new);
    SMH_REQUIRE(q_stride >= (long)H * D && q_stride % 8 == 0, "smh_kv8_attn: token stride %ld", q_stride);
    SMH_REQUIRE(codes_k && codes_v && scales && open_k && open_v && pages, "smh_kv8_attn: null pointer in the cache");
    SMH_REQUIRE(aligned16(codes_k) && aligned16(codes_v) && aligned16(open_k) && aligned16(open_v) && ((uintptr_t)scales & 7) == 0,
                "smh_kv8_attn: the cache's tensors are 16-byte aligned, its scales 8");
    SMH_REQUIRE(n_pages >= 1 && pages_cols >= 0 && pages_cols <= KV8_MAX_LEN / KV8_ROWS - 1 && pages_stride >= pages_cols, "smh_kv8_attn: n_pages=%ld pages_cols=%d (at most %d) pages_stride=%ld",
                n_pages, pages_cols, KV8_MAX_LEN / KV8_ROWS - 1, pages_stride);
    if (T == 0 || max_new == 0) return 0;
    SMH_REQUIRE(q && out && lens, "smh_kv8_attn: null pointer");
    SMH_REQUIRE(aligned16(q) && aligned16(out), "smh_kv8_attn: tensors are 16-byte aligned");
    const int most = cu ? (max_new < T ? max_new : T) : 1;
    const Kv8Plan plan = kv8_plan(B, H, Hkv, most, max_len, window, sinks);
    Kv8AttnParams p{(const half_t *)q, (half_t *)out, q_stride, lens, cu,
                    {(uint8_t *)codes_k, (uint8_t *)codes_v, (float *)scales, (half_t *)open_k, (half_t *)open_v, pages, pages_stride, n_pages, pages_cols},
                    T, B, H, Hkv, most, window, sinks, plan.splits, nullptr, nullptr};
    if (plan.splits > 1) {
        const size_t need = (size_t)plan.splits * T * H * (KV8_DIM + 2) * sizeof(float);
        SMH_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need, "smh_kv8_attn: workspace of %zu bytes, %zu needed (16-byte aligned)", workspace_bytes, need);
        p.part_o = (float *)workspace;
        p.part_ml = (float2 *)(p.part_o + (size_t)plan.splits * T * H * KV8_DIM);
    }
    const hipStream_t st = (hipStream_t)stream;
    if (plan.tiles) {
        const dim3 grid(Hkv, plan.splits, B);
        const size_t bytes = 4 * 16 * (KV8_DIM + 4) * 4 + 64 * 8;
        if (plan.tiles == 1) hipLaunchKernelGGL(kv8_attn_few_kernel<1>, grid, dim3(256), bytes, st, p);
        else hipLaunchKernelGGL(kv8_attn_few_kernel<2>, grid, dim3(256), bytes, st, p);
    } else {
        SMH_REQUIRE((long)B * Hkv < (1L << 31) && plan.groups <= 65535, "smh_kv8_attn: max_new=%d with %d queries a kv head (at most 65535 groups of 128)", most, H / Hkv);
        const dim3 grid(B * Hkv, (unsigned)plan.groups, plan.splits);
        if (plan.rows == 64) hipLaunchKernelGGL((kv8_attn_many_kernel<1, 1, 1>), grid, dim3(256), 32768, st, p);
        else hipLaunchKernelGGL((kv8_attn_many_kernel<2, 2, 2>), grid, dim3(256), 65536, st, p);
    }
    if (int rc = launch_status()) return rc;
    if (plan.splits == 1) return 0;
    const long rows = (long)T * H;
    SMH_REQUIRE((rows + 7) / 8 < (1L << 31), "smh_kv8_attn: T=%d", T);
    hipLaunchKernelGGL(kv8_attn_merge_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p);
    return launch_status();
}
