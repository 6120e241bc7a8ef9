// Beam search: the best continuations of each group of beams, and the states that follow them.
//
// Selection.  Candidate (beam r, token t) of a group has the score  scores[r] + x[r][t] - log sum_t' exp(x[r][t']);  the n best leave in descending order,
// equal ones by (beam, token).  A first launch goes over each row once, a workgroup per slice of it: the slice's values stay in registers while its n largest, its maximum and its
// sum of exponentials are found.  A second one has a workgroup per group: it adds the slices' sums up and picks the n best of all lists (one step a bit of the score,
// ended when just n are left above).
//   Order: within a row, and between rows of the same logits, the fp16 values order exactly.  Between other rows the scores are compared in 64 bits, with sums in 64 bits of fp32
//   terms exp(x - m), m the slice's largest value.  With d = m - x a term is off by 2^-23 of itself (the exponential) and d * 2.3 * 2^-24 (difference, product and log2(e)); the mean of d, weighted
//   by the terms, is at most log(vocab) (an entropy is), so a sum is off by less than 2^-18 for up to 2^24 columns (usually 2^-22): candidates of two rows keep their order
//   from 2^-17 apart.  A value's error depends on its slice's maximum: rows of the same values in another order are as close as that, and equal only where they are one slice.
// Bound: 2 bytes a logit from HBM, and short of that because all workgroups of the first launch run at a time and go through loads, bar, candidates and exponentials together, so that the
// phases add up (512 rows of 32016: 17 us, of which HBM needs 5.4; 1600 rows: 36, of which loads 17.5, bar 2, candidates 7, exponentials and sums 10); for few rows by two launches (4 rows: 6.5 and 4.9 us).
//
// Reordering.  Row i of a group takes the contents of row parents[i], in place: a workgroup owns a strip of all rows of a group, has it in LDS and then writes.
// Bound: HBM, each row that another one takes read and each row that changes written once (64 rows of four layers' open blocks, 2 MB each, 17.5 us; 73 with four bytes a thread at a time).
#include "smh_common.hpp"

namespace smh {

constexpr int BEAM_MAX_N = 128, BEAM_MAX_W = 64, BEAM_MAX_LISTS = 4096;

struct SelectParams {
    const half_t *logits;
    long ld;
    const float *scores;
    const uint8_t *ended;                          // may be null
    int rows, W, G, vocab, n, eos, slices, width;  // width: columns of a slice
    float *slice_max;                              // [rows][slices]
    double *slice_sum;                             // [rows][slices], of exp(x - slice_max)
    uint32_t *cand;                                // [rows][slices][n]: keys (below), descending; 0: none
    float *out_scores;                             // [G][n]
    int32_t *out_parents;
    int64_t *out_tokens;
    uint8_t *out_ended;
};

// A value's key: 16 bits that order as the values do (NaN as the least), then 16 bits that are larger for earlier columns of the slice: keys of a slice differ.
__device__ __forceinline__ uint32_t beam_order(half_t x) {
    const uint32_t b = __builtin_bit_cast(uint16_t, x);
    return b & 0x8000u ? 0xFFFFu - b : b | 0x8000u;
}
__device__ __forceinline__ float beam_value(uint32_t order) {
    const uint32_t b = order & 0x8000u ? order & 0x7FFFu : 0xFFFFu - order;
    return fminf((float)__builtin_bit_cast(half_t, (uint16_t)b), 65536.0f);      // (an infinity is the step after 65504: the others of its row stay in order)
}

// 256 threads, CHUNKS * 8 values each, chunk i of thread t being columns (256 i + t) * 8 .. + 7: a slice of 2048 * CHUNKS columns.
template <int CHUNKS>
__global__ __launch_bounds__(256) void beam_slice_kernel(SelectParams p) {
    __shared__ uint32_t top[256];                  // each thread's largest value and the first of its chunks that has it
    extern __shared__ uint32_t found[];            // candidates: at most all values of n threads
    __shared__ double red_sum[4];
    __shared__ int n_found;
    const int slice = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int c0 = slice * p.width, cols = min(p.width, p.vocab - c0), n = p.n;
    uint32_t *cand = p.cand + ((long)row * p.slices + slice) * n;
    // No value of a lost or ended beam counts: its candidates go by their index, which the second launch does by itself
    if (!(p.scores[row] > -INFINITY) || (p.ended != nullptr && p.ended[row] != 0)) return;
    const half_t *x = p.logits + (long)row * p.ld + c0;
    const h8 least = {-(half_t)INFINITY, -(half_t)INFINITY, -(half_t)INFINITY, -(half_t)INFINITY, -(half_t)INFINITY, -(half_t)INFINITY, -(half_t)INFINITY, -(half_t)INFINITY};
    h8 v[CHUNKS];
    const bool aligned = ((uintptr_t)x & 15) == 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int col = (i * 256 + t) * 8;
        if (aligned && col + 8 <= cols) v[i] = *reinterpret_cast<const h8 *>(x + col);
        else {
            v[i] = least;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < cols) v[i][e] = x[col + e];
        }
    }
    auto chunk_key = [](h8 v, uint32_t chunk) {
        const h4 a = __builtin_elementwise_max(__builtin_shufflevector(v, v, 0, 1, 2, 3), __builtin_shufflevector(v, v, 4, 5, 6, 7));
        const h2 b = __builtin_elementwise_max(__builtin_shufflevector(a, a, 0, 1), __builtin_shufflevector(a, a, 2, 3));
        const half_t m = __builtin_elementwise_max(b[0], b[1]) + (half_t)0.0f;      // (+ 0: one zero)
        return beam_order(m) << 16 | (0xFFFFu - chunk);
    };
    // the thread's key: order of its largest value, then the chunks' order (they are in the columns' order), 0 without columns
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        v[i] = __builtin_elementwise_max(v[i], least);                 // (NaN: -infinity)
        if ((i * 256 + t) * 8 < cols) mine = max(mine, chunk_key(v[i], i * 256 + t));
    }
    top[t] = mine;
    if (t == 0) n_found = 0;
    __syncthreads();
    // The n-th largest of these keys, bit by bit.  n threads are not below it; a value that is, by (value, chunk), has n better ones.
    uint32_t mx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) mx[i] = top[i * 64 + lane];
    uint32_t bar = 0;
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t at = bar | 1u << bit;
        int c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c += __popcll(__ballot(mx[i] >= at));
        if (c >= n) bar = at;
        if (c == n) break;                         // (just n are not below it already)
    }
    if (mine >= bar && mine != 0) {
#pragma unroll
        for (int i = 0; i < CHUNKS; ++i) {
            const uint32_t chunk = i * 256 + t;
            if (chunk_key(v[i], chunk) < bar) continue;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t order = beam_order(v[i][e] + (half_t)0.0f);
                if ((order << 16 | (0xFFFFu - chunk)) >= bar && (int)(chunk * 8 + e) < cols) found[atomicAdd(&n_found, 1)] = order << 16 | (0xFFFFu - (chunk * 8 + e));
            }
        }
    }
    uint32_t most = max(max(mx[0], mx[1]), max(mx[2], mx[3]));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    const float m = beam_value(most >> 16);                            // (every slice has a column)
    // exp(x - m): the difference is exact or rounded once, its product with log2(e) is off by 2^-24 of itself, so terms near the largest have 2^-23
    double total = 0.0;
    if (m > -INFINITY) {
        auto add = [&](float x) { total += (double)__builtin_amdgcn_exp2f((x - m) * 1.44269504f); };
        if (m < 65536.0f) {
#pragma unroll
            for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
                for (int e = 0; e < 8; ++e) add((float)v[i][e]);
        } else {                                   // some are infinite
            for (int i = 0; i < CHUNKS; ++i)
                for (int e = 0; e < 8; ++e) add(fminf((float)v[i][e], 65536.0f));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    if (lane == 0) red_sum[wave] = total;
    __syncthreads();
    const int have = n_found;
    if (t == 0) {
        p.slice_max[(long)row * p.slices + slice] = m;
        p.slice_sum[(long)row * p.slices + slice] = red_sum[0] + red_sum[1] + red_sum[2] + red_sum[3];
    }
    // each key's place among them (they differ, so the order they were found in leaves no trace)
    for (int i = t; i < have; i += 256) {
        const uint32_t k = found[i];
        int above = 0;
        for (int j = 0; j < have; ++j) above += found[j] > k;
        if (above < n) cand[above] = k;
    }
    for (int i = have + t; i < n; i += 256) cand[i] = 0;
}

// What the second launch knows of a row
struct BeamRow { double base; float max; int ended; };      // score - log sum (of an ended beam the score); the largest logit, NaN: the row's candidates go by index
__device__ __forceinline__ BeamRow beam_row(const SelectParams &p, long row) {
    // everything is asked for at once: what the first launch left of an ended or lost beam is not used
    const float score = p.scores[row];
    const int ended = p.ended != nullptr && p.ended[row] != 0;
    float m = -INFINITY;
    double s = 0.0;
    for (int i0 = 0; i0 < p.slices; i0 += 4) {
        float mi[4];
        double si[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long at = row * p.slices + min(i0 + i, p.slices - 1);
            mi[i] = p.slice_max[at];
            si[i] = p.slice_sum[at];
        }
        float now = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) now = fmaxf(now, mi[i]);
        if (m != now) s *= m == -INFINITY ? 0.0 : exp((double)m - (double)now);
        m = now;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i0 + i < p.slices) s += si[i] * (mi[i] == m ? 1.0 : exp((double)mi[i] - (double)m));
    }
    if (!(score > -INFINITY) || ended) return BeamRow{(double)score, __builtin_nanf(""), ended};
    // (36 bits of the sum: the order in which one slice's terms were added shows in the last of 53, and here only where a sum is next to a step)
    return BeamRow{(double)score - log(__longlong_as_double((__double_as_longlong(s) + (1 << 15)) & ~0xFFFFll)), m, 0};
}
constexpr uint32_t BEAM_NONE = 0xFFFFFFFFu;        // (beam * vocab + token is below 2^30)
// Candidate i of list (row r, slice) with its key: score and index; BEAM_NONE: there is none
__device__ __forceinline__ void beam_candidate(const SelectParams &p, const BeamRow &row, int r, int slice, int i, uint32_t key, double &value, uint32_t &index) {
    value = -INFINITY;
    index = BEAM_NONE;
    if (row.max != row.max) {                      // one list stands for the whole row
        if (slice != 0 || i >= p.vocab) return;
        int token = i;
        if (row.base > -INFINITY) {                // an ended beam: its end, then the others
            token = i == 0 ? p.eos : i - 1 < p.eos ? i - 1 : i;
            if (i == 0) value = row.base;
        }
        index = (uint32_t)(r * p.vocab + token);
        return;
    }
    if (key == 0) return;
    index = (uint32_t)(r * p.vocab + slice * p.width + (0xFFFFu - (key & 0xFFFFu)));
    const float v = beam_value(key >> 16);
    if (v > -INFINITY) value = row.base + ((double)v - (double)row.max);
}
__device__ __forceinline__ void beam_out(const SelectParams &p, const BeamRow *rows, int g, int k, double value, uint32_t index) {
    const int r = (int)(index / (uint32_t)p.vocab), token = (int)(index - (uint32_t)r * (uint32_t)p.vocab);
    const long o = (long)g * p.n + k;
    p.out_scores[o] = (float)value;
    p.out_parents[o] = r;
    p.out_tokens[o] = token;
    p.out_ended[o] = token == p.eos || rows[r].ended;
}
// 64 bits that order as the numbers do
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v == 0.0 ? 0.0 : v);
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double unordered64(uint64_t o) { return __longlong_as_double((long long)(o >> 63 ? o & ~(1ull << 63) : ~o)); }

// A workgroup per group has all candidates, K of them a thread, and finds the n-th largest score bit by bit; among equal ones at the border the lowest indices stay.
template <int K, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void beam_pick_kernel(SelectParams p) {
    __shared__ BeamRow rows[BEAM_MAX_W];
    __shared__ uint64_t best[BEAM_MAX_N];
    __shared__ uint32_t best_index[BEAM_MAX_N];
    __shared__ int counts[2][WAVES], have;
    const int g = blockIdx.x, t = threadIdx.x, wave = t >> 6, all = p.W * p.slices * p.n, n = p.n;
    const uint32_t *cand = p.cand + (long)g * all;
    uint32_t key[K];
#pragma unroll
    for (int k = 0; k < K; ++k) key[k] = (k * WAVES * 64 + t) < all ? cand[k * WAVES * 64 + t] : 0u;
    if (t < p.W) rows[t] = beam_row(p, (long)g * p.W + t);
    if (t == 0) have = 0;
    __syncthreads();
    uint64_t score[K];                             // 0: no candidate (a number's is larger)
    uint32_t index[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = k * WAVES * 64 + t, list = c / n, r = list / p.slices;
        double v = -INFINITY;
        index[k] = BEAM_NONE;
        if (c < all) beam_candidate(p, rows[r], r, list - r * p.slices, c - list * n, key[k], v, index[k]);
        score[k] = index[k] == BEAM_NONE ? 0 : ordered64(v);
    }
    int turn = 0;
    auto count = [&](auto test) {                  // of all threads' candidates
        int c = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) c += __popcll(__ballot(test(k)));
        if (WAVES > 1) {                           // (two sets: who writes one has passed the barrier behind the last reads of it)
            if ((t & 63) == 0) counts[turn][wave] = c;
            __syncthreads();
            c = 0;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) c += counts[turn][w];
            turn ^= 1;
        }
        return c;
    };
    uint64_t bar = 0;
    bool exact = false;                            // just n scores are not below the bar
    for (int bit = 63; bit >= 0 && !exact; --bit) {
        const uint64_t at = bar | 1ull << bit;
        const int c = count([&](int k) { return score[k] >= at; });
        if (c >= n) bar = at;
        exact = c == n;
    }
    uint32_t last = BEAM_NONE - 1;                 // the last index that stays of the scores that are the bar
    if (!exact) {
        const int left = n - count([&](int k) { return score[k] > bar; });
        last = 0;                                  // the left-th smallest index: the largest with fewer than `left` below it
        for (int bit = 29; bit >= 0; --bit) {
            const uint32_t at = last | 1u << bit;
            if (count([&](int k) { return score[k] == bar && index[k] < at; }) < left) last = at;
        }
    }
    // those n, in any order, and the place of each
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (score[k] != 0 && (exact ? score[k] >= bar : score[k] > bar || (score[k] == bar && index[k] <= last))) {
            const int at = atomicAdd(&have, 1);
            if (at < n) { best[at] = score[k]; best_index[at] = index[k]; }
        }
    __syncthreads();
    const int found = min(have, n);                // (n: a group has at least that many)
    for (int i = t; i < found; i += 64 * WAVES) {
        const uint64_t s = best[i];
        const uint32_t x = best_index[i];
        int above = 0;
        for (int j = 0; j < found; ++j) above += best[j] > s || (best[j] == s && best_index[j] < x);
        beam_out(p, rows, g, above, unordered64(s), x);
    }
}

// The largest of a wave's numbers
__device__ __forceinline__ double wave_max_f64(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmax(v, __shfl_xor(v, o, 64));
    return v;
}

// More candidates than that: a wave per group merges the sorted lists (one for each row and slice); lane l has lists l, l + 64, ..
__global__ __launch_bounds__(64) void beam_merge_kernel(SelectParams p) {
    extern __shared__ int at[];                    // [lists]: entries taken
    __shared__ BeamRow rows[BEAM_MAX_W];
    const int g = blockIdx.x, lane = threadIdx.x, lists = p.W * p.slices;
    const uint32_t *cand = p.cand + (long)g * lists * p.n;
    for (int i = lane; i < lists; i += 64) at[i] = 0;
    if (lane < p.W) rows[lane] = beam_row(p, (long)g * p.W + lane);
    __syncthreads();
    double best = -INFINITY;
    uint32_t index = BEAM_NONE;
    int list = -1;
    auto mine = [&]() {                            // the best of the lane's lists' next candidates
        best = -INFINITY;
        index = BEAM_NONE;
        for (int i = lane; i < lists; i += 64) {
            const int r = i / p.slices, e = at[i];
            double v;
            uint32_t x;
            beam_candidate(p, rows[r], r, i - r * p.slices, e, e < p.n ? cand[(long)i * p.n + e] : 0u, v, x);
            if (x != BEAM_NONE && (index == BEAM_NONE || v > best || (v == best && x < index))) { best = v; index = x; list = i; }
        }
    };
    mine();
    for (int k = 0; k < p.n; ++k) {
        const double v = wave_max_f64(best);
        const uint64_t equal = __ballot(best == v && index != BEAM_NONE);
        if (equal == 0) break;                     // (not reached: a group has at least n candidates)
        int lane_of = __ffsll((unsigned long long)equal) - 1;
        if (equal & (equal - 1)) {                 // equal scores: the lowest index
            uint32_t x = best == v ? index : BEAM_NONE;
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) x = min(x, (uint32_t)__shfl_xor((int)x, o, 64));
            lane_of = __ffsll((unsigned long long)__ballot(index == x)) - 1;
        }
        if (lane == lane_of) {
            beam_out(p, rows, g, k, v, index);
            at[list] += 1;
            mine();
        }
    }
}

// ---- reordering -------------------------------------------------------------------------------------------------------------------
constexpr int REORDER_MAX = 16;
struct ReorderParams {
    char *at[REORDER_MAX];
    long stride[REORDER_MAX], bytes[REORDER_MAX];  // from a row to the next; of a row that move
    int unit[REORDER_MAX];                         // > 0: bytes of an entry, of which the first *upto move
    int piece[REORDER_MAX];                        // bytes that a thread moves at a time: 16 or 4
    int strips[REORDER_MAX];                       // workgroups of the tensors before
    const int32_t *parents, *upto;
    int W, n, pieces_log2;                         // pieces of a strip
};

template <class T>
__device__ __forceinline__ void reorder_strip(char *base, long stride, T *lds, const int32_t *from, const uint8_t *wanted, int W, int pieces_log2, int pieces) {
    const int c = threadIdx.x & ((1 << pieces_log2) - 1), r0 = threadIdx.x >> pieces_log2, by = 256 >> pieces_log2;
    if (c < pieces) {
#pragma unroll 4
        for (int r = r0; r < W; r += by)
            if (wanted[r]) lds[(r << pieces_log2) + c] = *reinterpret_cast<const T *>(base + r * stride + (long)c * sizeof(T));
    }
    __syncthreads();
    if (c < pieces) {
#pragma unroll 4
        for (int r = r0; r < W; r += by)
            if (from[r] != r) *reinterpret_cast<T *>(base + r * stride + (long)c * sizeof(T)) = lds[(from[r] << pieces_log2) + c];
    }
}

__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderParams p) {
    extern __shared__ u32x4 reorder_lds[];
    __shared__ int32_t from[BEAM_MAX_W];
    __shared__ uint8_t wanted[BEAM_MAX_W];         // rows that another one takes
    int k = 0;
    for (int i = 1; i < p.n; ++i)
        if ((int)blockIdx.x >= p.strips[i]) k = i;
    const int g = blockIdx.y, t = threadIdx.x, W = p.W;
    long bytes = p.bytes[k];
    if (p.unit[k] > 0) bytes = min(bytes, max((long)p.upto[0], 0L) * p.unit[k]);
    const long strip = (long)p.piece[k] << p.pieces_log2, b0 = (long)((int)blockIdx.x - p.strips[k]) * strip;
    if (b0 >= bytes) return;
    const int pieces = (int)(min(strip, bytes - b0) / p.piece[k]);     // (a row's bytes are a multiple of them)
    const long stride = p.stride[k];
    if (t < W) {
        from[t] = min(max(p.parents[(long)g * W + t], 0), W - 1);
        wanted[t] = 0;
    }
    __syncthreads();
    if (t < W && from[t] != t) wanted[from[t]] = 1;
    __syncthreads();
    char *base = p.at[k] + (long)g * W * stride + b0;
    if (p.piece[k] == 16) reorder_strip(base, stride, reorder_lds, from, wanted, W, p.pieces_log2, pieces);
    else reorder_strip(base, stride, reinterpret_cast<uint32_t *>(reorder_lds), from, wanted, W, p.pieces_log2, pieces);
}

}  // namespace smh

using namespace smh;

namespace {
struct SelectPlan { int slices, width; size_t sums, maxima, cands, bytes; };
// Slices of 16384 columns where there are 512 of them, of 8192 else (us a call, wide and narrow slices of 32016 columns, 8 beams a group: 64 rows 19.6 and 18.4, 160 20.7 and 20.4, 320 23.8 and
// 28.0, 512 26.7 and 32.3, 1600 48.8 and 62; slices of 32768: 24.9, 26.7 and 50.7 for the last three)
SelectPlan select_plan(long rows, int vocab, int n) {
    SelectPlan p;
    p.width = rows * ((vocab + 16383) / 16384) >= 512 && vocab > 8192 ? 16384 : 8192;
    p.slices = (vocab + p.width - 1) / p.width;
    p.sums = (size_t)rows * p.slices * 8;
    p.maxima = ((size_t)rows * p.slices * 4 + 7) / 8 * 8;
    p.cands = (size_t)rows * p.slices * n * 4;
    p.bytes = p.sums + p.maxima + p.cands;
    return p;
}
bool select_sizes(int G, int W, int vocab, int n) {
    return G >= 1 && W >= 1 && W <= BEAM_MAX_W && vocab >= 1 && vocab <= (1 << 24) && n >= 1 && n <= BEAM_MAX_N && n <= (long)W * vocab && (long)G * W <= (1 << 20);
}
}  // namespace

extern "C" size_t smh_beam_select_workspace_bytes(int G, int W, int vocab, int n) {
    return select_sizes(G, W, vocab, n) ? select_plan((long)G * W, vocab, n).bytes : 0;
}

extern "C" int smh_beam_select(const void *logits, long ld, const float *scores, const uint8_t *ended, int G, int W, int vocab, int n, int64_t eos, float *out_scores,
                               int32_t *out_parents, int64_t *out_tokens, uint8_t *out_ended, void *workspace, size_t workspace_bytes, smh_stream_t stream) {
    SMH_REQUIRE(W >= 1 && W <= BEAM_MAX_W, "smh_beam_select: W=%d (1 .. %d beams a group)", W, BEAM_MAX_W);
    SMH_REQUIRE(n >= 1 && n <= BEAM_MAX_N && n <= (long)W * vocab, "smh_beam_select: n=%d of %d beams x vocab=%d (1 .. %d)", n, W, vocab, BEAM_MAX_N);
    SMH_REQUIRE(select_sizes(G, W, vocab, n), "smh_beam_select: G=%d W=%d vocab=%d", G, W, vocab);
    SMH_REQUIRE(ld >= vocab, "smh_beam_select: ld=%ld below vocab=%d", ld, vocab);
    SMH_REQUIRE(eos >= 0 && eos < vocab, "smh_beam_select: eos=%ld outside the vocabulary of %d", (long)eos, vocab);
    SMH_REQUIRE(logits && scores && out_scores && out_parents && out_tokens && out_ended, "smh_beam_select: null pointer");
    const SelectPlan plan = select_plan((long)G * W, vocab, n);
    SMH_REQUIRE(W * plan.slices <= BEAM_MAX_LISTS, "smh_beam_select: W=%d beams x %d slices of the vocabulary (at most %d)", W, plan.slices, BEAM_MAX_LISTS);
    SMH_REQUIRE(workspace && ((uintptr_t)workspace & 7) == 0 && workspace_bytes >= plan.bytes, "smh_beam_select: workspace of %zu bytes, %zu needed (8-byte aligned)", workspace_bytes, plan.bytes);
    char *ws = (char *)workspace;
    SelectParams p{(const half_t *)logits, ld, scores, ended, G * W, W, G, vocab, n, (int)eos, plan.slices, plan.width,
                   (float *)(ws + plan.sums), (double *)ws, (uint32_t *)(ws + plan.sums + plan.maxima), out_scores, out_parents, out_tokens, out_ended};
    const hipStream_t st = (hipStream_t)stream;
    // (rows along y: at most 65535 a launch)
    for (int r = 0; r < G * W; r += 65535) {
        SelectParams part = p;
        part.logits += (long)r * ld;
        part.scores += r;
        if (ended) part.ended += r;
        part.slice_max += (long)r * plan.slices;
        part.slice_sum += (long)r * plan.slices;
        part.cand += (long)r * plan.slices * n;
        const int rows = min(65535, G * W - r);
        if (plan.width == 16384) hipLaunchKernelGGL(beam_slice_kernel<8>, dim3(plan.slices, rows), dim3(256), n * 256, st, part);
        else hipLaunchKernelGGL(beam_slice_kernel<4>, dim3(plan.slices, rows), dim3(256), n * 128, st, part);
        if (int rc = launch_status()) return rc;
    }
    // (us a call of 32016 columns: 64 beams, 128 kept, 65, by the merge 253; 32 beams, 64 kept, 34 and 87.  32 candidates a thread of 16 waves spill 26 vector registers)
    const long all = (long)W * plan.slices * n;
    if (all <= 256) hipLaunchKernelGGL((beam_pick_kernel<4, 1>), dim3(G), dim3(64), 0, st, p);
    else if (all <= 1024) hipLaunchKernelGGL((beam_pick_kernel<4, 4>), dim3(G), dim3(256), 0, st, p);
    else if (all <= 8192) hipLaunchKernelGGL((beam_pick_kernel<8, 16>), dim3(G), dim3(1024), 0, st, p);
    else if (all <= 32768) hipLaunchKernelGGL((beam_pick_kernel<32, 16>), dim3(G), dim3(1024), 0, st, p);
    else hipLaunchKernelGGL(beam_merge_kernel, dim3(G), dim3(64), (size_t)W * plan.slices * 4, st, p);
    return launch_status();
}

extern "C" int smh_beam_reorder(const int32_t *parents, int G, int W, int n, void *const *tensors, const long *strides, const long *bytes, const int *units, const int32_t *upto,
                                smh_stream_t stream) {
    SMH_REQUIRE(G >= 1 && G <= 65535 && W >= 1 && W <= BEAM_MAX_W, "smh_beam_reorder: G=%d (1 .. 65535) W=%d (1 .. %d)", G, W, BEAM_MAX_W);
    SMH_REQUIRE(n >= 0 && n <= REORDER_MAX, "smh_beam_reorder: %d tensors (at most %d)", n, REORDER_MAX);
    if (n == 0) return 0;
    SMH_REQUIRE(parents && tensors && strides && bytes && units, "smh_beam_reorder: null pointer");
    ReorderParams p{};
    p.parents = parents;
    p.upto = upto;
    p.W = W;
    p.n = n;
    for (int i = 0; i < n; ++i) {
        SMH_REQUIRE(tensors[i] && bytes[i] >= 0 && strides[i] >= bytes[i] && units[i] >= 0, "smh_beam_reorder: tensor %d: rows of %ld bytes %ld apart, entries of %d", i, bytes[i], strides[i],
                    units[i]);
        SMH_REQUIRE(bytes[i] % 4 == 0 && strides[i] % 4 == 0 && ((uintptr_t)tensors[i] & 3) == 0 && units[i] % 4 == 0, "smh_beam_reorder: tensor %d: rows are multiples of 4 bytes, 4-byte aligned", i);
        SMH_REQUIRE(units[i] == 0 || upto, "smh_beam_reorder: tensor %d goes by *upto, which is null", i);
        for (int j = 0; j < i; ++j) SMH_REQUIRE(tensors[i] != tensors[j], "smh_beam_reorder: tensors %d and %d are the same", j, i);
    }
    // a strip of a group is at most 32 KB of LDS: 256 pieces of 16 bytes up to 8 beams, 32 of 64
    p.pieces_log2 = W <= 8 ? 8 : W <= 16 ? 7 : W <= 32 ? 6 : 5;
    long strips = 0;
    for (int i = 0; i < n; ++i) {
        p.at[i] = (char *)tensors[i];
        p.stride[i] = strides[i];
        p.bytes[i] = bytes[i];
        p.unit[i] = units[i];
        p.piece[i] = units[i] == 0 && bytes[i] % 16 == 0 && strides[i] % 16 == 0 && ((uintptr_t)tensors[i] & 15) == 0 ? 16 : 4;
        p.strips[i] = (int)strips;
        const long strip = (long)p.piece[i] << p.pieces_log2;
        strips += (bytes[i] + strip - 1) / strip;
        SMH_REQUIRE(strips < (1L << 31), "smh_beam_reorder: rows too long");
    }
    if (strips == 0) return 0;
    hipLaunchKernelGGL(beam_reorder_kernel, dim3((unsigned)strips, G), dim3(256), ((size_t)W * 16) << p.pieces_log2, (hipStream_t)stream, p);
    return launch_status();
}
